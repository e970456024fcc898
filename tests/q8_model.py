"""A plain model of the 8-bit KV cache in numpy: what the tests of its kernels
are held to. The layout follows include/llmtie_b200.h; nothing here calls the
library."""
from __future__ import annotations

import numpy as np


def sections(kv, hd, cap):
    """{name: (offset, numpy type, shape)} of a cache buffer, and its bytes."""
    nb = cap // 32
    out, at = {}, 0
    for name, dtype, shape in (("k", np.int8, (kv, nb, hd // 64, 32, 64)), ("v", np.int8, (kv, nb, hd, 32)),
                               ("ks", np.float32, (kv, nb)), ("vs", np.float32, (kv, nb)), ("w", np.float32, (kv, nb)),
                               ("kt", np.float16, (kv, 32, hd)), ("vt", np.float16, (kv, 32, hd))):
        out[name] = (at, dtype, shape)
        at += (int(np.prod(shape)) * np.dtype(dtype).itemsize + 127) // 128 * 128
    return out, at


class Q8Model:
    """One sequence's cache as its sections, over a copy of the buffer's bytes."""

    def __init__(self, kv, hd, cap, fill=0):
        self.kv, self.hd, self.cap, self.nb = kv, hd, cap, cap // 32
        self.sec, self.bytes = sections(kv, hd, cap)
        self.buf = np.full(self.bytes, fill, np.uint8)
        for name, (at, dtype, shape) in self.sec.items():
            n = int(np.prod(shape)) * np.dtype(dtype).itemsize
            setattr(self, name, self.buf[at:at + n].view(dtype).reshape(shape))

    def copy(self):
        m = Q8Model(self.kv, self.hd, self.cap)
        m.buf[:] = self.buf
        return m

    # blocks as [32][hd] values
    def block(self, which, h, b):
        if which == "k":
            codes = self.k[h, b].transpose(1, 0, 2).reshape(32, self.hd)
            return codes.astype(np.float64) * np.float64(self.ks[h, b])
        return self.v[h, b].T.astype(np.float64) * np.float64(self.vs[h, b])

    def put(self, which, h, b, x16):
        """Quantises a block of f16 rows [32][hd]."""
        x = x16.astype(np.float32)
        top = np.abs(x).max()
        if np.isfinite(top):
            scale = np.float32(top) / np.float32(127)
            codes = np.rint(x / scale) if scale > 0 else np.zeros_like(x)
        else:
            scale, codes = np.float32(np.nan), np.zeros_like(x)
        codes = codes.astype(np.int8)
        if which == "k":
            self.k[h, b] = codes.reshape(32, self.hd // 64, 64).transpose(1, 0, 2)
            self.ks[h, b] = scale
        else:
            self.v[h, b] = codes.T
            self.vs[h, b] = scale

    def append(self, k, v, past):
        """Rows f32 [n][kv][hd], already rotated."""
        for which, rows in (("k", k), ("v", v)):
            tail = self.kt if which == "k" else self.vt
            with np.errstate(over="ignore"):
                rows16 = rows.astype(np.float16)
            for h in range(self.kv):
                x = np.concatenate([tail[h, :past % 32], rows16[:, h]])
                for i in range(len(x) // 32):
                    self.put(which, h, past // 32 + i, x[32 * i:32 * i + 32])
                    self.w[h, past // 32 + i] = 0
                n = len(x) % 32
                # only rows that are new to the tail are written
                lo = past % 32 if len(x) < 32 else 0
                if n:
                    tail[h, lo:n] = x[len(x) - n + lo:]

    def values(self, which, live):
        """f64 [kv][live][hd]."""
        out = np.zeros((self.kv, live, self.hd))
        tail = self.kt if which == "k" else self.vt
        for h in range(self.kv):
            for b in range(live // 32):
                out[h, 32 * b:32 * b + 32] = self.block(which, h, b)
            out[h, live // 32 * 32:] = tail[h, :live % 32]
        return out

    def evict(self, dst, live, keep, first, recent):
        """The kept blocks' numbers [kv][kept]; dst may be this model."""
        full = live // 32
        src = self.copy()
        picks = []
        for h in range(self.kv):
            if full <= keep:
                pick = list(range(full))
            else:
                w = [float(x) if x > 0 else 0.0 for x in src.w[h]]
                middle = sorted(range(first, full - recent), key=lambda i: (-w[i], i))[:keep - first - recent]
                pick = sorted(list(range(first)) + middle + list(range(full - recent, full)))
            picks.append(pick)
            for name in ("k", "v", "ks", "vs", "w"):
                getattr(dst, name)[h, :len(pick)] = getattr(src, name)[h, pick]
        dst.kt[:, :live % 32] = src.kt[:, :live % 32]
        dst.vt[:, :live % 32] = src.vt[:, :live % 32]
        return np.array(picks, np.int32).reshape(self.kv, -1)


def rotate(x, pos, inv_freq):
    """x [n][heads][hd] f64 turned by (pos + i) * inv_freq, halves layout."""
    half = x.shape[-1] // 2
    a = (pos + np.arange(len(x)))[:, None, None] * inv_freq.astype(np.float64)
    lo, hi = x[..., :half], x[..., half:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)


def attend(q, k, v, scale, last=None):
    """q f64 [n][heads][hd] over k, v f64 [kv][t][hd]; row i sees keys up to last[i].
    Returns (out [n][heads][hd], probabilities [n][heads][t])."""
    n, heads, hd = q.shape
    kv = k.shape[0]
    out, probs = np.zeros_like(q), np.zeros((n, heads, k.shape[1]))
    for h in range(heads):
        s = q[:, h] @ k[h // (heads // kv)].T * scale
        if last is not None:
            s = np.where(np.arange(k.shape[1])[None] > np.asarray(last)[:, None], -np.inf, s)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        probs[:, h] = p
        out[:, h] = p @ v[h // (heads // kv)]
    return out, probs
