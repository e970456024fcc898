"""The 8-bit KV cache: appending, reading back, decode, prefill and eviction,
each against a plain model in 64 bits (tests/q8_model.py)."""
import numpy as np
import pytest
import torch

from tests.helpers import assert_parity, rel_l2
from tests.q8_model import Q8Model, attend, rotate
from ttsxabe_b200 import (CacheOverrun, DecodeScratch, InvalidArgument, KvCacheQ8, Misaligned, OddHeadDim, Prefix,
                          RaggedBlock, SliceOverrun, UnsupportedAttention, decode_plan_q8, evicted_len, kv_q8_bytes)

pytestmark = pytest.mark.gpu

GEOMETRIES = [(32, 8, 128), (20, 20, 64), (8, 1, 128), (12, 4, 64)]


def put(g, model):
    t = torch.from_numpy(model.buf.copy()).to(g.device)
    torch.cuda.synchronize()
    return t


def got(g, t, model):
    g.synchronize()
    m = Q8Model(model.kv, model.hd, model.cap)
    m.buf[:] = t.cpu().numpy()
    return m


def filled(rng, kv, hd, cap, live, scale=1.0):
    """A model that holds `live` random tokens; what lies past them is poison
    (NaN scales and tails, codes of 0x7f, weights of NaN)."""
    m = Q8Model(kv, hd, cap, fill=0x7f)
    m.ks[:], m.vs[:], m.w[:], m.kt[:], m.vt[:] = np.nan, np.nan, np.nan, np.nan, np.nan
    m.append((scale * rng.standard_normal((live, kv, hd))).astype(np.float32),
             rng.standard_normal((live, kv, hd)).astype(np.float32), 0)
    m.w[:, :live // 32] = rng.exponential(size=(kv, live // 32))
    return m


def same_bytes(a, b):
    assert a.bytes == b.bytes
    for name in ("k", "v", "ks", "vs", "w", "kt", "vt"):
        x, y = getattr(a, name), getattr(b, name)
        assert x.tobytes() == y.tobytes(), f"section {name}: {int((x.view(np.uint8) != y.view(np.uint8)).sum())} bytes differ"


def inv_freqs(hd):
    return (10000.0 ** (-2.0 * np.arange(hd // 2) / hd)).astype(np.float32)


# ---- appending ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hd", GEOMETRIES)
@pytest.mark.parametrize("past,n", [(0, 1), (0, 31), (0, 32), (0, 33), (0, 97), (31, 1), (5, 3), (5, 27), (5, 28), (30, 40),
                                    (64, 64), (95, 1), (33, 200)])
def test_append_bits(gpu, heads, kv, hd, past, n):
    # no rotation: f16 rounding, the scale and the codes are single IEEE operations, so bits are equal
    rng = np.random.default_rng(past * 1000 + n)
    cap = (past + n + 31) // 32 * 32 + 32
    m = filled(rng, kv, hd, cap, past)
    k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
    t = put(gpu, m)
    gpu.rope_append_q8(None, gpu.upload(k), gpu.upload(v), [0, n], [t], [cap], [past], [past], None, heads, kv, hd)
    m.append(k, v, past)
    same_bytes(m, got(gpu, t, m))


@pytest.mark.parametrize("pos", [0, 7, 131000, (1 << 31) - 200])
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (12, 4, 64)])
def test_append_rotation(gpu, heads, kv, hd, pos):
    # Rotated elements a c - b s in f32: the angle is reduced in 64 bits and rounded to f32 half turns (2^-25 of a half
    # turn: pi 2^-25 < 2^-23 rad), sine and cosine are within 2 ulp (2^-23), the two products round once each: at most
    # 2^-21 (|a| + |b|). The 64-bit angle itself is rounded twice here and there: 4 x 2^-53 of it. The f16 of the tail
    # adds half a step, 2^-11 relative.
    rng = np.random.default_rng(pos % 1000)
    n, cap = 21, 32
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
    f = inv_freqs(hd)
    m = Q8Model(kv, hd, cap)
    t = put(gpu, m)
    qd, out = gpu.upload(q), gpu.uninit(q.size)
    gpu.rope_append_q8(qd, gpu.upload(k), gpu.upload(v), [0, n], [t], [cap], [0], [pos], gpu.upload(f), heads, kv, hd, q_out=out)
    assert np.array_equal(gpu.download(qd).reshape(q.shape), q)

    def bound(x):
        a = np.abs(x)
        return (2.0 ** -21 + 4 * 2.0 ** -53 * (pos + n)) * (a + np.roll(a, hd // 2, -1))

    w = rotate(q.astype(np.float64), pos, f)
    assert (np.abs(gpu.download(out).reshape(q.shape) - w) <= bound(q)).all()
    w = rotate(k.astype(np.float64), pos, f).transpose(1, 0, 2)
    e = np.abs(got(gpu, t, m).kt[:, :n].astype(np.float64) - w)
    assert (e <= bound(k).transpose(1, 0, 2) * (1 + 2.0 ** -11) + 2.0 ** -11 * np.abs(w) + 2.0 ** -25).all()
    # in place
    gpu.rope_append_q8(qd, gpu.upload(k), gpu.upload(v), [0, n], [t], [cap], [0], [pos], gpu.upload(f), heads, kv, hd)
    assert np.array_equal(gpu.download(qd), gpu.download(out))


def test_rotation_agrees_with_rope_scaled(gpu):
    # rope_scaled multiplies position and frequency in f32: at positions under 64 that is 2^-24 x 64 rad at most,
    # 2^-18; twice that for the frequency's own rounding being shared covers the rest
    rng = np.random.default_rng(4)
    heads, kv, hd, n = 8, 2, 128, 40
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
    div = gpu.upload(np.linspace(1.0, 4.0, hd // 2).astype(np.float32))
    f = gpu.rope_inv_freq(500000.0, hd, div)
    want = gpu.upload(q)
    gpu.rope_scaled(want, 0, div, n, heads, hd, 500000.0, 20)
    t = put(gpu, Q8Model(kv, hd, 64))
    mine = gpu.upload(q)
    gpu.rope_append_q8(mine, gpu.upload(k), gpu.upload(v), [0, n], [t], [64], [0], [20], f, heads, kv, hd)
    assert np.abs(gpu.download(want) - gpu.download(mine)).max() <= 2.0 ** -17 * 2 * np.abs(q).max()


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (20, 20, 64)])
def test_append_does_not_depend_on_how_rows_arrive(gpu, heads, kv, hd):
    rng = np.random.default_rng(9)
    n, cap = 150, 160
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
    f = gpu.upload(inv_freqs(hd))
    m = Q8Model(kv, hd, cap)
    buffers, queries = [], []
    for cuts in ([0, n], [0, 31, 32, 33, 100, n], list(range(n + 1))):
        t, qo = put(gpu, m), []
        for a, b in zip(cuts, cuts[1:]):
            x = gpu.upload(q[a:b])
            gpu.rope_append_q8(x, gpu.upload(k[a:b]), gpu.upload(v[a:b]), [0, b - a], [t], [cap], [a], [a], f, heads, kv, hd)
            qo.append(gpu.download(x))
        r = got(gpu, t, m)
        r.kt[:, n % 32:] = 0     # (rows of the tail past the live ones are what earlier blocks left)
        r.vt[:, n % 32:] = 0
        buffers.append(r)
        queries.append(np.concatenate(qo))
    for b, x in zip(buffers[1:], queries[1:]):
        same_bytes(buffers[0], b)
        assert np.array_equal(queries[0], x)


def test_append_ragged_batch(gpu):
    """37 sequences (more than one launch takes), some without rows, capacities
    of their own, rows packed from a row that is not the first; nothing beside
    the new tokens changes."""
    rng = np.random.default_rng(5)
    heads, kv, hd = 4, 2, 64
    past = [int(x) for x in rng.integers(0, 80, 37)]
    new = [int(x) for x in rng.choice([0, 1, 2, 31, 32, 33, 70], 37)]
    cap = [(p + n + 32) // 32 * 32 + 32 * int(rng.integers(0, 3)) for p, n in zip(past, new)]
    cu = np.concatenate([[3], 3 + np.cumsum(new)]).astype(int).tolist()
    ms = [filled(rng, kv, hd, c, p) for c, p in zip(cap, past)]
    k, v = rng.standard_normal((2, cu[-1], kv, hd)).astype(np.float32)
    q = rng.standard_normal((cu[-1], heads, hd)).astype(np.float32)
    ts = [put(gpu, m) for m in ms]
    f = gpu.upload(inv_freqs(hd))
    kd, vd, qd = gpu.upload(k), gpu.upload(v), gpu.upload(q)
    gpu.rope_append_q8(qd, kd, vd, cu, ts, cap, past, past, f, heads, kv, hd)
    out = gpu.download(qd).reshape(q.shape)
    assert np.array_equal(out[:3], q[:3])
    for b, m in enumerate(ms):
        alone = put(gpu, m)
        rows = slice(cu[b], cu[b + 1])
        if new[b]:
            x = gpu.upload(q[rows])
            gpu.rope_append_q8(x, gpu.upload(k[rows]), gpu.upload(v[rows]), [0, new[b]], [alone], [cap[b]], [past[b]], [past[b]],
                               f, heads, kv, hd)
            assert np.array_equal(gpu.download(x).reshape(-1, heads, hd), out[rows])
        same_bytes(got(gpu, alone, m), got(gpu, ts[b], m))


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 1e30])
def test_a_block_with_a_non_finite_value_reads_as_nan(gpu, bad):
    rng = np.random.default_rng(2)
    kv, hd, cap = 2, 64, 96
    k, v = rng.standard_normal((2, 64, kv, hd)).astype(np.float32)
    k[40, 1, 3] = bad
    m = Q8Model(kv, hd, cap)
    t = put(gpu, m)
    gpu.rope_append_q8(None, gpu.upload(k), gpu.upload(v), [0, 64], [t], [cap], [0], [0], None, 2, kv, hd)
    m.append(k, v, 0)
    r = got(gpu, t, m)
    assert np.isnan(r.ks[1, 1]) and not r.k[1, 1].any()
    keys, _ = gpu.cache_read_q8([t], [cap], [64], [0], [0, 64], kv, hd)
    gpu.synchronize()
    keys = keys.float().cpu().numpy().reshape(64, kv, hd)
    assert np.isnan(keys[32:, 1]).all() and np.isfinite(keys[:32]).all() and np.isfinite(keys[:, 0]).all()
    # and the rows that see it are NaN, the other head's are not
    q = rng.standard_normal(2 * hd).astype(np.float32)
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [t], [64], [cap], 2, kv, hd, 0.125, DecodeScratch()))
    assert np.isfinite(out[:hd]).all() and np.isnan(out[hd:]).all()


def test_blocks_of_zeros_and_of_the_smallest_values(gpu):
    kv, hd, cap = 1, 64, 64
    k = np.zeros((64, kv, hd), np.float32)
    k[32:] = 6e-8 * np.sign(np.random.default_rng(0).standard_normal((32, kv, hd)))
    v = np.full((64, kv, hd), 65504.0, np.float32)
    m = Q8Model(kv, hd, cap)
    t = put(gpu, m)
    gpu.rope_append_q8(None, gpu.upload(k), gpu.upload(v), [0, 64], [t], [cap], [0], [0], None, 1, kv, hd)
    m.append(k, v, 0)
    same_bytes(m, got(gpu, t, m))


# ---- reading back, cutting, growing ----------------------------------------------------------------------------

@pytest.mark.parametrize("kv,hd", [(8, 128), (3, 64)])
@pytest.mark.parametrize("live,first,n", [(100, 0, 100), (100, 3, 1), (100, 31, 2), (100, 96, 4), (64, 32, 32), (20, 5, 15),
                                          (130, 17, 110)])
def test_read(gpu, kv, hd, live, first, n):
    rng = np.random.default_rng(live + first)
    m = filled(rng, kv, hd, 160, live)
    t = put(gpu, m)
    pad = 2
    ko, vo = (torch.full(((n + pad + 1) * kv * hd,), 7.0, dtype=torch.float16, device=gpu.device) for _ in "kv")
    torch.cuda.synchronize()
    gpu.cache_read_q8([t], [160], [live], [first], [pad, pad + n], kv, hd, k_out=ko, v_out=vo)
    gpu.synchronize()
    for which, x in (("k", ko), ("v", vo)):
        x = x.cpu().numpy().reshape(-1, kv, hd)
        # the value is the f32 product of code and scale, rounded to f16 once
        want = m.values(which, live).astype(np.float32).astype(np.float16)[:, first:first + n].transpose(1, 0, 2)
        assert np.array_equal(x[pad:pad + n], want)
        assert (x[:pad] == 7).all() and (x[pad + n:] == 7).all()


@pytest.mark.parametrize("live,to", [(100, 100), (100, 97), (100, 96), (100, 70), (100, 64), (100, 1), (100, 0), (96, 95), (64, 40)])
@pytest.mark.parametrize("kv,hd", [(8, 128), (2, 64)])
def test_rewind(gpu, kv, hd, live, to):
    rng = np.random.default_rng(live + to)
    m = filled(rng, kv, hd, 128, live)
    t = put(gpu, m)
    gpu.cache_rewind_q8([t], [128], [live], [to], kv, hd)
    w = m.copy()
    if to % 32 and to // 32 != live // 32:
        for h in range(kv):
            w.kt[h, :to % 32] = m.block("k", h, to // 32)[:to % 32].astype(np.float32).astype(np.float16)
            w.vt[h, :to % 32] = m.block("v", h, to // 32)[:to % 32].astype(np.float32).astype(np.float16)
    same_bytes(w, got(gpu, t, m))


def test_grow(gpu):
    rng = np.random.default_rng(1)
    kv, hd = 4, 128
    for live in (0, 5, 64, 101):
        m = filled(rng, kv, hd, 128, live)
        w = Q8Model(kv, hd, 256)
        t, u = put(gpu, m), put(gpu, w)
        gpu.cache_grow_q8(t, u, kv, hd, 128, 256, live)
        m.evict(w, live, live // 32, 0, 0)
        same_bytes(w, got(gpu, u, w))


# ---- decode ----------------------------------------------------------------------------------------------------

def decode_want(q, m, live, heads, scale):
    o, p = attend(q.astype(np.float64)[None], m.values("k", live), m.values("v", live), scale)
    share = p[0].reshape(m.kv, heads // m.kv, live).sum(1)[:, :live // 32 * 32].reshape(m.kv, -1, 32).sum(-1)
    return o[0], share


# Decode's roundings: q to 16 bits of its row's largest value (3.3 sigma over 128 normal values: an error of 1e-4 / 3.46
# sigma an element), so scores err by 3e-5 (scale |k| = 1); the probabilities by 2^-16 / 3.46 of the block's largest, some
# ten times the typical one: 4e-5. An output's relative error is about that of the probabilities, 5e-5 of its norm;
# four times that, with room for rows of few keys, is the bound. An f16 output adds 2^-12 rms at most.
DECODE_REL = 3e-4


@pytest.mark.parametrize("heads,kv,hd", GEOMETRIES + [(3, 3, 128), (16, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("live", [1, 2, 31, 32, 33, 64, 255, 256, 257, 1000])
def test_decode(gpu, heads, kv, hd, live):
    rng = np.random.default_rng(live * 7 + heads)
    cap = (live + 31) // 32 * 32 + 64
    m = filled(rng, kv, hd, cap, live)
    q = rng.standard_normal((heads, hd)).astype(np.float32)
    scale = hd ** -0.5
    t = put(gpu, m)
    scratch = DecodeScratch()
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [t], [live], [cap], heads, kv, hd, scale, scratch))
    want, share = decode_want(q, m, live, heads, scale)
    assert np.isfinite(out).all()
    assert rel_l2(want, out.reshape(heads, hd)) <= DECODE_REL
    same_bytes(m, got(gpu, t, m))
    # f16 out, and the weights
    half = torch.empty(heads * hd, dtype=torch.float16, device=gpu.device)
    gpu.decode_batched_q8(gpu.upload(q), [t], [live], [cap], heads, kv, hd, scale, scratch, out=half, weigh=True)
    gpu.synchronize()
    assert np.array_equal(half.cpu().numpy(), out.astype(np.float16))
    r = got(gpu, t, m)
    # a weight is a sum of probabilities: their errors (scores within 3e-5 rms, 2e-4 at most) and f32 sums
    w = m.w[:, :live // 32] + share
    assert np.abs(r.w[:, :live // 32] - w).max(initial=0) <= 2e-4 * (1 + np.abs(w).max(initial=0))
    assert r.w[:, live // 32:].tobytes() == m.w[:, live // 32:].tobytes()


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (20, 20, 64), (8, 1, 128)])
def test_decode_ragged_batch(gpu, heads, kv, hd):
    """More sequences than a launch takes, of any length, some empty."""
    rng = np.random.default_rng(3)
    live = [0, 1, 40, 700, 32, 64, 33] + [int(x) for x in rng.integers(0, 300, 28)] + [0]
    cap = [max(32, (n + 31) // 32 * 32) for n in live]
    ms = [filled(rng, kv, hd, c, n) for c, n in zip(cap, live)]
    q = rng.standard_normal((len(live), heads, hd)).astype(np.float32)
    ts = [put(gpu, m) for m in ms]
    scratch = DecodeScratch()
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), ts, live, cap, heads, kv, hd, hd ** -0.5, scratch, weigh=True))
    out = out.reshape(q.shape)
    for b, n in enumerate(live):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        want, share = decode_want(q[b], ms[b], n, heads, hd ** -0.5)
        assert rel_l2(want, out[b]) <= DECODE_REL, f"sequence {b} of {n}"
        w = ms[b].w[:, :n // 32] + share
        assert np.abs(got(gpu, ts[b], ms[b]).w[:, :n // 32] - w).max(initial=0) <= 2e-4 * (1 + np.abs(w).max(initial=0))
    # the same call again gives the same bits, whatever the order of the grid's blocks
    for _ in range(5):
        again = gpu.download(gpu.decode_batched_q8(gpu.upload(q), ts, live, cap, heads, kv, hd, hd ** -0.5, scratch))
        assert np.array_equal(again.reshape(q.shape), out)


@pytest.mark.parametrize("heads,kv,hd,batch,live,cluster", [
    (8, 8, 128, 1, 30, 1), (32, 8, 128, 16, 600, 2), (32, 8, 128, 8, 1800, 4), (32, 8, 128, 1, 1999, 8), (4, 1, 128, 1, 7000, 16),
    (32, 8, 128, 1, 33000, 0), (20, 20, 64, 8, 1500, 2), (20, 20, 64, 1, 1500, 8), (8, 1, 64, 1, 9000, 16), (4, 1, 64, 40, 5, 1),
    (8, 8, 64, 2, 20000, 0)])
def test_decode_by_every_way_over_the_device(gpu, heads, kv, hd, batch, live, cluster):
    """A cluster of each size a pair, and the cut by work; lengths that differ by
    a block or two, and weights."""
    rng = np.random.default_rng(live)
    lives = [live - int(x) for x in rng.integers(0, min(live, 70), batch)]
    assert decode_plan_q8(lives[:32], kv, hd)[1] == cluster
    cap = [(n + 31) // 32 * 32 for n in lives]
    ms = []
    for c, n in zip(cap, lives):
        m = Q8Model(kv, hd, c, fill=0x7f)
        full = n // 32
        m.k[:, :full], m.v[:, :full] = (rng.integers(-127, 128, x.shape) for x in (m.k[:, :full], m.v[:, :full]))
        m.ks[:], m.vs[:] = np.nan, np.nan
        m.ks[:, :full], m.vs[:, :full] = rng.uniform(0.005, 0.02, (2, kv, full))
        m.kt[:, :n % 32], m.vt[:, :n % 32] = rng.standard_normal((2, kv, n % 32, hd))
        m.w[:] = 0.5
        ms.append(m)
    ts = [put(gpu, m) for m in ms]
    q = rng.standard_normal((batch, heads, hd)).astype(np.float32)
    scratch = DecodeScratch()
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), ts, lives, cap, heads, kv, hd, hd ** -0.5, scratch, weigh=True)).reshape(q.shape)
    for b, n in enumerate(lives):
        want, share = decode_want(q[b], ms[b], n, heads, hd ** -0.5)
        assert rel_l2(want, out[b]) <= DECODE_REL, f"sequence {b} of {n}"
        w = got(gpu, ts[b], ms[b]).w
        assert np.abs(w[:, :n // 32] - (0.5 + share)).max(initial=0) <= 2e-4 * (1.5 + share.max(initial=0))
        assert (w[:, n // 32:] == 0.5).all()


@pytest.mark.parametrize("heads,kv,hd,lives", [
    (8, 1, 128, (20001,)), (4, 1, 128, (40000, 30)), (8, 2, 128, (31, 0, 33333)), (12, 4, 128, (12345,)),
    (8, 1, 64, (25000, 7, 64, 1)), (3, 3, 64, (30007, 40000))])
def test_decode_of_pairs_that_several_clusters_share(gpu, heads, kv, hd, lives):
    """Long contexts of few KV heads, shorter ones among them that leave clusters
    without a block; the same bits every time."""
    rng = np.random.default_rng(sum(lives))
    grid, cluster, _ = decode_plan_q8(lives, kv, hd)
    assert cluster == 8 and grid > 8 * kv * len(lives)
    cap = [(n + 31) // 32 * 32 or 32 for n in lives]
    ms = []
    for c, n in zip(cap, lives):
        m = Q8Model(kv, hd, c, fill=0x7f)
        full = n // 32
        m.k[:, :full], m.v[:, :full] = (rng.integers(-127, 128, x.shape) for x in (m.k[:, :full], m.v[:, :full]))
        m.ks[:], m.vs[:] = np.nan, np.nan
        m.ks[:, :full], m.vs[:, :full] = rng.uniform(0.005, 0.02, (2, kv, full))
        m.kt[:, :n % 32], m.vt[:, :n % 32] = rng.standard_normal((2, kv, n % 32, hd))
        m.w[:] = 0
        ms.append(m)
    ts = [put(gpu, m) for m in ms]
    q = rng.standard_normal((len(lives), heads, hd)).astype(np.float32)
    scratch = DecodeScratch()
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), ts, lives, cap, heads, kv, hd, hd ** -0.5, scratch, weigh=True)).reshape(q.shape)
    for b, n in enumerate(lives):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        want, share = decode_want(q[b], ms[b], n, heads, hd ** -0.5)
        assert rel_l2(want, out[b]) <= DECODE_REL, f"sequence {b} of {n}"
        w = got(gpu, ts[b], ms[b]).w
        assert np.abs(w[:, :n // 32] - share).max(initial=0) <= 2e-4 * (1 + share.max(initial=0))
    for _ in range(5):
        again = gpu.download(gpu.decode_batched_q8(gpu.upload(q), ts, lives, cap, heads, kv, hd, hd ** -0.5, scratch))
        assert np.array_equal(again.reshape(q.shape), out)


def test_decode_sink_and_long_faint_context(gpu):
    """One key far above all others, whose sum is as large as its own: no key's
    probability may be lost below it."""
    kv, hd, live = 1, 64, 4096
    m = Q8Model(kv, hd, live)
    m.ks[:], m.vs[:] = 1.0 / 127, 1.0
    m.v[:] = 1                                    # every value 1 ...
    m.k[0, 5, 0, 7, 0] = 127                      # ... and one key that q points at
    m.v[0, 5, :, 7] = 3
    q = np.zeros(hd, np.float32)
    q[0] = 8.3 * 8                                # e^8.3 = 4024 times any other key
    want, _ = decode_want(q[None], m, live, 1, 0.125)
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [put(gpu, m)], [live], [live], 1, kv, hd, 0.125, DecodeScratch()))
    assert rel_l2(want, out) <= DECODE_REL
    assert 1.9 < want.mean() < 2.1


@pytest.mark.parametrize("where", ["first", "last"])
def test_decode_with_a_score_spread_beyond_f32_exponents(gpu, where):
    """Scores 300 apart: what is negligible vanishes, nothing overflows."""
    rng = np.random.default_rng(0)
    kv, hd, live = 1, 64, 2000
    m = filled(rng, kv, hd, 2016, live, scale=60.0)
    if where == "last":
        m.k[:] = m.k[:, ::-1].copy()
        m.ks[:, :live // 32] = m.ks[:, :live // 32][:, ::-1].copy()
        m.k[:, :live // 32] = rng.integers(-127, 128, m.k[:, :live // 32].shape)
    q = (20 * rng.standard_normal((1, hd))).astype(np.float32)
    want, _ = decode_want(q, m, live, 1, 0.125)
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [put(gpu, m)], [live], [2016], 1, kv, hd, 0.125, DecodeScratch()))
    # (scores of +-1000 err by 2^-16 of themselves and more: the winner takes all but some 1e-2)
    assert np.isfinite(out).all() and rel_l2(want, out) <= 5e-2


def test_decode_query_of_zeros_and_non_finite_queries(gpu):
    rng = np.random.default_rng(0)
    heads, kv, hd, live = 4, 1, 128, 100
    m = filled(rng, kv, hd, 128, live)
    q = rng.standard_normal((heads, hd)).astype(np.float32)
    q[1] = 0
    q[2, 5] = np.inf
    q[3, 9] = np.nan
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [put(gpu, m)], [live], [128], heads, kv, hd, 0.09, DecodeScratch()))
    out = out.reshape(heads, hd)
    want, _ = decode_want(q[:2], m, live, 2, 0.09)
    assert rel_l2(want, out[:2]) <= DECODE_REL
    assert np.isnan(out[2:]).all()


def test_decode_offsets_past_32_bits(gpu):
    """A cache whose value codes start beyond 2^31 bytes, and whose last blocks
    are the ones that count."""
    kv, hd = 1, 128
    live = (1 << 24) + (1 << 20) + 9           # 2.3 GB of codes each for keys and values
    cap = (live + 31) // 32 * 32
    t = torch.zeros(kv_q8_bytes(kv, hd, cap), dtype=torch.uint8, device=gpu.device)
    rng = np.random.default_rng(8)
    k, v = rng.standard_normal((2, 200, kv, hd)).astype(np.float32)
    k *= 4
    torch.cuda.synchronize()
    at = live - 200
    # rows of zeros lead up to a block's start
    lead = at % 32
    rows = lambda x: gpu.upload(np.concatenate([np.zeros((lead, kv, hd), np.float32), x]))  # noqa: E731
    gpu.rope_append_q8(None, rows(k), rows(v), [0, lead + 200], [t], [cap], [at - lead], [0], None, 1, kv, hd)
    ko, vo = gpu.cache_read_q8([t], [cap], [live], [at], [0, 200], kv, hd)
    gpu.synchronize()
    kk, vv = (x.double().cpu().numpy().reshape(200, hd) for x in (ko, vo))
    assert rel_l2(v[:, 0], vv) < 0.02
    q = (3 * k[150, 0] / np.linalg.norm(k[150, 0])).astype(np.float32)
    s = np.concatenate([kk @ q.astype(np.float64), [0.0]])
    p = np.exp(s - s.max())
    p[-1] *= live - 200                        # every other key scores 0, its value is 0
    want = (p[:-1] @ vv) / p.sum()
    out = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [t], [live], [cap], 1, kv, hd, 1.0, DecodeScratch()))
    # (the values compared are rounded to f16, 2^-12 rms, and the scores to 2^-16 of |q| |k|)
    assert rel_l2(want, out) <= 2e-3


# ---- prefill ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (20, 20, 64), (12, 4, 128), (8, 1, 64), (16, 1, 128), (5, 1, 64)])
@pytest.mark.parametrize("past,n", [(0, 1), (0, 5), (0, 32), (0, 129), (63, 1), (40, 90), (700, 33), (62, 4), (31, 2), (1000, 8), (300, 17)])
def test_flash(gpu, heads, kv, hd, past, n):
    rng = np.random.default_rng(past + n)
    live = past + n
    cap = (live + 31) // 32 * 32 + 32
    m = filled(rng, kv, hd, cap, live)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    t = put(gpu, m)
    for causal in (True, False):
        out = gpu.download(gpu.flash_attn_q8(gpu.upload(q), [0, n], [t], [cap], [past], heads, kv, hd, hd ** -0.5, causal))
        last = past + np.arange(n) if causal else None
        want, _ = attend(q.astype(np.float64), m.values("k", live), m.values("v", live), hd ** -0.5, last)
        assert_parity(f"{past} + {n}", want, out.reshape(q.shape))
    same_bytes(m, got(gpu, t, m))


def test_flash_ragged_batch(gpu):
    """Nineteen sequences, some without rows, f16 out; rows around them are left
    as they were."""
    rng = np.random.default_rng(6)
    heads, kv, hd = 8, 2, 128
    past = [int(x) for x in rng.integers(0, 200, 19)]
    new = [int(x) for x in rng.choice([0, 1, 17, 128, 150], 19)]
    cu = np.concatenate([[2], 2 + np.cumsum(new)]).astype(int).tolist()
    live = [p + n for p, n in zip(past, new)]
    cap = [max(32, (n + 31) // 32 * 32) for n in live]
    ms = [filled(rng, kv, hd, c, n) for c, n in zip(cap, live)]
    q = rng.standard_normal((cu[-1] + 1, heads, hd)).astype(np.float32)
    out = torch.full((q.size,), 9.0, dtype=torch.float16, device=gpu.device)
    torch.cuda.synchronize()
    gpu.flash_attn_q8(gpu.upload(q), cu, [put(gpu, m) for m in ms], cap, past, heads, kv, hd, hd ** -0.5, True, out=out)
    gpu.synchronize()
    out = out.float().cpu().numpy().reshape(q.shape)
    assert (out[:2] == 9).all() and (out[cu[-1]:] == 9).all()
    for b, m in enumerate(ms):
        rows = slice(cu[b], cu[b + 1])
        if new[b]:
            want, _ = attend(q[rows].astype(np.float64), m.values("k", live[b]), m.values("v", live[b]), hd ** -0.5,
                             past[b] + np.arange(new[b]))
            assert_parity(f"sequence {b}", want, out[rows])


@pytest.mark.parametrize("heads,kv,hd,batch", [(8, 1, 128, 33), (4, 4, 64, 70), (6, 2, 128, 32)])
def test_flash_of_more_sequences_than_a_launch_takes(gpu, heads, kv, hd, batch):
    rng = np.random.default_rng(batch)
    past = [int(x) for x in rng.integers(0, 90, batch)]
    new = [int(x) for x in rng.choice([0, 33, 66, 129, 140], batch)]
    cu = np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()
    live = [p + n for p, n in zip(past, new)]
    cap = [max(32, (n + 31) // 32 * 32) for n in live]
    ms = [filled(rng, kv, hd, c, n) for c, n in zip(cap, live)]
    q = rng.standard_normal((cu[-1], heads, hd)).astype(np.float32)
    out = gpu.download(gpu.flash_attn_q8(gpu.upload(q), cu, [put(gpu, m) for m in ms], cap, past, heads, kv, hd, hd ** -0.5, True))
    out = out.reshape(q.shape)
    for b, m in enumerate(ms):
        rows = slice(cu[b], cu[b + 1])
        if new[b]:
            want, _ = attend(q[rows].astype(np.float64), m.values("k", live[b]), m.values("v", live[b]), hd ** -0.5,
                             past[b] + np.arange(new[b]))
            assert_parity(f"sequence {b}", want, out[rows])


@pytest.mark.parametrize("heads,kv,hd,batch", [(16, 4, 128, 20), (32, 8, 64, 11)])
def test_flash_of_a_few_more_blocks_than_the_device_holds(gpu, heads, kv, hd, batch):
    """Rows whose keys are cut because the last round of blocks would leave most of
    the device idle; sequences of different lengths over one cache."""
    rng = np.random.default_rng(batch)
    new, longest = 40, 2500
    m = filled(rng, kv, hd, 2560, longest + new)
    t = put(gpu, m)
    past = [longest - int(x) for x in rng.integers(0, 300, batch)]
    past[0] = longest
    cu = [new * b for b in range(batch + 1)]
    q = rng.standard_normal((cu[-1], heads, hd)).astype(np.float32)
    # (a shorter sequence's last tokens lie in complete blocks: it ends with one)
    past = [p if p == longest else (p + new) // 32 * 32 - new for p in past]
    out = gpu.download(gpu.flash_attn_q8(gpu.upload(q), cu, [t] * batch, [2560] * batch, past, heads, kv, hd, hd ** -0.5, True))
    out = out.reshape(q.shape)
    k, v = m.values("k", longest + new), m.values("v", longest + new)
    for b in range(batch):
        rows = slice(cu[b], cu[b + 1])
        want, _ = attend(q[rows].astype(np.float64), k[:, :past[b] + new], v[:, :past[b] + new], hd ** -0.5, past[b] + np.arange(new))
        assert_parity(f"sequence {b}", want, out[rows])


def test_flash_of_sequences_that_unpack_to_more_than_a_gigabyte(gpu):
    """Twelve of them over one cache, 134 MB each: a launch ends with the eighth. The
    rows are the same, so the results are, but for how a launch cuts its rows' keys."""
    rng = np.random.default_rng(3)
    heads, kv, hd, past, new, batch = 8, 4, 128, 65400, 40, 12
    n = past + new
    k, v = (gpu.upload(rng.standard_normal((n, kv * hd)).astype(np.float32)) for _ in range(2))
    cap = (n + 31) // 32 * 32
    t = gpu.kv_alloc_q8(kv, hd, cap)
    gpu.rope_append_q8(None, k, v, [0, n], [t], [cap], [0], [0], None, heads, kv, hd)
    q = rng.standard_normal((new, heads, hd)).astype(np.float32)
    cu = [new * b for b in range(batch + 1)]
    out = gpu.download(gpu.flash_attn_q8(gpu.upload(np.tile(q, (batch, 1, 1))), cu, [t] * batch, [cap] * batch, [past] * batch, heads, kv,
                                         hd, hd ** -0.5, True)).reshape(batch, -1)
    ko, vo = gpu.cache_read_q8([t], [cap], [n], [0], [0, n], kv, hd)
    gpu.synchronize()
    kk, vv = (x.double().cpu().numpy().reshape(n, kv, hd).transpose(1, 0, 2) for x in (ko, vo))
    at = np.array([0, new - 1])
    want, _ = attend(q[at].astype(np.float64), kk, vv, hd ** -0.5, past + at)
    for b in (0, 7, 8, 11):
        assert_parity(f"sequence {b}", want, out[b].reshape(q.shape)[at])


def test_flash_of_a_prompt_longer_than_a_launch_takes(gpu):
    """Rows past 16384 go as another sequence over the same keys; checked on the
    rows around the seam and at the end."""
    rng = np.random.default_rng(6)
    heads, kv, hd, n = 2, 1, 64, 16384 + 70
    cap = (n + 31) // 32 * 32
    k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    t = gpu.kv_alloc_q8(kv, hd, cap)
    gpu.rope_append_q8(None, gpu.upload(k), gpu.upload(v), [0, n], [t], [cap], [0], [0], None, heads, kv, hd)
    out = gpu.download(gpu.flash_attn_q8(gpu.upload(q), [0, n], [t], [cap], [0], heads, kv, hd, 0.125, True)).reshape(q.shape)
    ko, vo = gpu.cache_read_q8([t], [cap], [n], [0], [0, n], kv, hd)
    gpu.synchronize()
    kk, vv = (x.double().cpu().numpy().reshape(n, kv, hd).transpose(1, 0, 2) for x in (ko, vo))
    at = np.array([0, 1, 130, 16382, 16383, 16384, 16385, n - 1])
    want, _ = attend(q[at].astype(np.float64), kk, vv, 0.125, at)
    assert_parity("rows at the seam", want, out[at])


# ---- eviction --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv,hd", [(8, 128), (3, 64)])
@pytest.mark.parametrize("live,keep,first,recent", [(1000, 10, 1, 2), (1000, 3, 1, 2), (1000, 31, 0, 0), (1000, 40, 1, 1), (1000, 0, 0, 0),
                                                    (992, 12, 0, 5), (40, 0, 0, 0), (31, 4, 1, 1), (0, 1, 1, 0), (20000, 100, 4, 8)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(gpu, kv, hd, live, keep, first, recent, in_place):
    rng = np.random.default_rng(live + keep)
    cap = max(32, (live + 31) // 32 * 32) + 32
    m = Q8Model(kv, hd, cap)
    m.buf[:] = rng.integers(0, 256, m.bytes)
    m.ks[:], m.vs[:] = rng.random(m.ks.shape), rng.random(m.vs.shape)
    # few different weights: ties are the rule; some negative, NaN or infinite
    m.w[:] = rng.choice([0.0, 0.5, 1.0, 2.5, 1e-30, -1.0, np.nan, np.inf], m.w.shape)
    want = m.copy() if in_place else Q8Model(kv, hd, max(32, (evicted_len(live, keep) + 31) // 32 * 32), fill=0x55)
    t = put(gpu, m)
    d = t if in_place else put(gpu, want)
    kept = min(live // 32, keep)
    index = torch.full((kv * kept + 1,), -5, dtype=torch.int32, device=gpu.device)
    torch.cuda.synchronize()
    gpu.cache_evict_q8([t], [cap], [d], [want.cap], [live], [keep], first, recent, kv, hd, index=index)
    picks = m.evict(want, live, keep, first, recent)
    same_bytes(want, got(gpu, d, want))
    index = index.cpu().numpy()
    assert np.array_equal(index[:-1].reshape(kv, -1), picks) and index[-1] == -5
    if not in_place:
        same_bytes(m, got(gpu, t, m))


def test_evict_ragged_batch(gpu):
    rng = np.random.default_rng(12)
    kv, hd = 2, 64
    live = [int(x) for x in rng.integers(0, 900, 34)]
    keep = [int(x) for x in rng.integers(3, 20, 34)]
    cap = [max(32, (n + 31) // 32 * 32) for n in live]
    ms = [filled(rng, kv, hd, c, n) for c, n in zip(cap, live)]
    ts = [put(gpu, m) for m in ms]
    most = max(min(n // 32, k) for n, k in zip(live, keep))
    index = torch.full((34 * kv * most,), -1, dtype=torch.int32, device=gpu.device)
    torch.cuda.synchronize()
    gpu.cache_evict_q8(ts, cap, ts, cap, live, keep, 1, 2, kv, hd, index=index)
    index = index.cpu().numpy().reshape(34, kv, most)
    for b, m in enumerate(ms):
        picks = m.evict(m, live[b], keep[b], 1, 2)
        same_bytes(m, got(gpu, ts[b], m))
        assert np.array_equal(index[b, :, :picks.shape[1]], picks) and (index[b, :, picks.shape[1]:] == -1).all()


# ---- together --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (8, 8, 64)])
def test_a_conversation(gpu, heads, kv, hd):
    """A prompt, decoded tokens with their weights, an eviction, more tokens, a
    cut into the last block and another prompt, against the model in 64 bits."""
    rng = np.random.default_rng(21)
    f = inv_freqs(hd)
    fd = gpu.upload(f)
    c = KvCacheQ8(gpu, kv, hd, 4096)
    m, scratch, scale = Q8Model(kv, hd, 4096), DecodeScratch(), hd ** -0.5
    held = 0

    def rows(n):
        q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
        qd = gpu.upload(q)
        c.append(qd, gpu.upload(k), gpu.upload(v), n, fd, heads)
        # what the cache holds is taken from the device: its codes are tested above
        w = got(gpu, c.data, Q8Model(kv, hd, c.cap))
        return rotate(q.astype(np.float64), c.pos - n, f), qd, w

    q, qd, m = rows(300)
    out = gpu.download(gpu.flash_attn_q8(qd, [0, 300], [c.data], [c.cap], [0], heads, kv, hd, scale, True))
    want, _ = attend(q, m.values("k", 300), m.values("v", 300), scale, np.arange(300))
    assert_parity("prompt", want, out.reshape(want.shape))
    total = np.zeros((kv, 300 // 32))
    for _ in range(40):
        q, qd, m = rows(1)
        out = gpu.download(gpu.decode_batched_q8(qd, [c.data], [c.len], [c.cap], heads, kv, hd, scale, scratch, weigh=True))
        want, share = decode_want(q[0], m, c.len, heads, scale)
        assert rel_l2(want, out.reshape(want.shape)) <= DECODE_REL
        total += share[:, :300 // 32]
    m = got(gpu, c.data, m)
    assert np.abs(m.w[:, :300 // 32] - total).max() <= 2e-4 * (1 + total.max())
    assert (c.len, c.pos) == (340, 340)
    c.evict(6, keep_first=1, keep_recent=2)
    m.evict(m, 340, 6, 1, 2)
    held = evicted_len(340, 6)
    assert (c.len, c.pos) == (held, 340)
    same_bytes(m, got(gpu, c.data, m))
    for _ in range(30):
        q, qd, m = rows(1)
        out = gpu.download(gpu.decode_batched_q8(qd, [c.data], [c.len], [c.cap], heads, kv, hd, scale, scratch))
        want, _ = decode_want(q[0], m, c.len, heads, scale)
        assert rel_l2(want, out.reshape(want.shape)) <= DECODE_REL
    with pytest.raises(InvalidArgument):
        c.truncate(100)
    c.truncate(350)
    assert (c.len, c.pos) == (held + 10, 350)
    q, qd, m = rows(50)
    out = gpu.download(gpu.flash_attn_q8(qd, [0, 50], [c.data], [c.cap], [c.len - 50], heads, kv, hd, scale, True))
    want, _ = attend(q, m.values("k", c.len), m.values("v", c.len), scale, c.len - 50 + np.arange(50))
    assert_parity("second prompt", want, out.reshape(want.shape))


def test_prefix_over_8_bit_caches(gpu):
    """`Prefix` cuts 8-bit caches as it cuts f16 ones; they grow by whole blocks."""
    rng = np.random.default_rng(1)
    heads, kv, hd = 4, 2, 64
    layers = [KvCacheQ8(gpu, kv, hd, 1000) for _ in range(2)]
    p = Prefix(layers)
    first = [int(x) for x in rng.integers(0, 99, 400)]
    for start, ids in ((0, first), (250, first[:250] + [100] * 700)):
        assert p.keep(ids) == start
        n = len(ids) - start
        for c in layers:
            k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
            c.append(None, gpu.upload(k), gpu.upload(v), n, None, heads)
            assert c.len == len(ids) and c.cap % 32 == 0 and c.data.numel() == kv_q8_bytes(kv, hd, c.cap)
        p.extend(ids[start:])
    p.reset()
    assert layers[0].len == 0


def test_one_head_is_what_the_f16_path_gives(gpu):
    """Over the values that the 8-bit cache stands for, held in f16, the f16
    decode agrees to what both round."""
    rng = np.random.default_rng(3)
    heads, kv, hd, live, cap = 32, 8, 128, 1000, 1024
    m = filled(rng, kv, hd, cap, live)
    q = rng.standard_normal((heads, hd)).astype(np.float32)
    t = put(gpu, m)
    kc = np.zeros((kv, cap, hd), np.float16)
    vc = np.zeros((kv, hd, cap), np.float16)
    kc[:, :live] = m.values("k", live)
    vc[:, :, :live] = m.values("v", live).transpose(0, 2, 1)
    a = gpu.download(gpu.decode_batched_q8(gpu.upload(q), [t], [live], [cap], heads, kv, hd, hd ** -0.5, DecodeScratch()))
    b = gpu.download(gpu.attn_decode_f16(gpu.upload(q), gpu.upload_u16(kc.view(np.uint16)), gpu.upload_u16(vc.view(np.uint16)),
                                         heads, kv, hd, live, cap, hd ** -0.5, False, DecodeScratch()))
    assert_parity("f16 cache", b, a)


# ---- graphs, streams, workspaces -----------------------------------------------------------------------------------

def test_a_step_replayed_from_a_graph(gpu):
    """Append, decode with weights and eviction captured after one call, then
    replayed after a larger call has outgrown the workspaces: the same bits."""
    rng = np.random.default_rng(17)
    heads, kv, hd, live, cap = 32, 8, 128, 600, 640
    m = filled(rng, kv, hd, cap, live)
    q = rng.standard_normal((heads, hd)).astype(np.float32)
    k, v = rng.standard_normal((2, 1, kv, hd)).astype(np.float32)
    f, qd, kd, vd = gpu.upload(inv_freqs(hd)), gpu.upload(q), gpu.upload(k), gpu.upload(v)
    qo, out = gpu.uninit(q.size), gpu.uninit(q.size)
    flash = gpu.uninit(q.size)
    t, d = put(gpu, m), put(gpu, Q8Model(kv, hd, 320))
    scratch = DecodeScratch()

    def step():
        gpu.rope_append_q8(qd, kd, vd, [0, 1], [t], [cap], [live], [live], f, heads, kv, hd, q_out=qo)
        gpu.decode_batched_q8(qo, [t], [live + 1], [cap], heads, kv, hd, hd ** -0.5, scratch, out=out, weigh=True)
        gpu.flash_attn_q8(qo, [0, 1], [t], [cap], [live], heads, kv, hd, hd ** -0.5, True, out=flash)
        gpu.cache_evict_q8([t], [cap], [d], [320], [live + 1], [8], 1, 2, kv, hd)

    step()
    first = got(gpu, t, m), got(gpu, d, Q8Model(kv, hd, 320)), gpu.download(out), gpu.download(flash)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(gpu.stream):
        with torch.cuda.graph(graph, stream=gpu.stream):
            step()
    # a call that needs more of every workspace
    big = filled(rng, kv, hd, 4096, 4000)
    tb = [put(gpu, big) for _ in range(6)]
    qb = gpu.upload(rng.standard_normal(6 * heads * hd).astype(np.float32))
    gpu.decode_batched_q8(qb, tb, [4000] * 6, [4096] * 6, heads, kv, hd, 0.1, scratch, weigh=True)
    gpu.flash_attn_q8(qb, [0, 1, 2, 3, 4, 5, 6], tb, [4096] * 6, [3999] * 6, heads, kv, hd, 0.1, True)
    gpu.cache_evict_q8(tb, [4096] * 6, tb, [4096] * 6, [4000] * 6, [100] * 6, 1, 1, kv, hd)
    gpu.synchronize()
    t.copy_(torch.from_numpy(m.buf))
    torch.cuda.synchronize()
    for _ in range(2):
        t.copy_(torch.from_numpy(m.buf))
        out.zero_()
        flash.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(gpu.stream):
            graph.replay()
        same_bytes(first[0], got(gpu, t, m))
        same_bytes(first[1], got(gpu, d, first[1]))
        assert np.array_equal(first[2], gpu.download(out))
        assert np.array_equal(first[3], gpu.download(flash))


def test_growing_under_a_capture_is_refused(gpu):
    rng = np.random.default_rng(1)
    heads, kv, hd = 4, 2, 64
    m = filled(rng, kv, hd, 64, 40)
    t, q, out = put(gpu, m), gpu.upload(rng.standard_normal((heads, hd))), gpu.uninit(heads * hd)
    scratch = DecodeScratch()
    scratch._bind(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(gpu.stream):
        with torch.cuda.graph(graph, stream=gpu.stream):
            with pytest.raises(Exception, match="allocating"):
                gpu.decode_batched_q8(q, [t], [40], [64], heads, kv, hd, 0.1, scratch, out=out)
    want, _ = decode_want(gpu.download(q).reshape(heads, hd), m, 40, heads, 0.1)
    assert rel_l2(want, gpu.download(gpu.decode_batched_q8(q, [t], [40], [64], heads, kv, hd, 0.1, scratch)).reshape(heads, hd)) <= DECODE_REL


def test_two_handles_at_once(gpu):
    """Two handles, their streams and scratches side by side."""
    from ttsxabe_b200 import Gpu

    rng = np.random.default_rng(5)
    heads, kv, hd, live, cap = 32, 8, 128, 5000, 5024
    other = Gpu.open(gpu.ordinal)
    m = Q8Model(kv, hd, cap)
    m.k[:], m.v[:] = rng.integers(-127, 128, m.k.shape), rng.integers(-127, 128, m.v.shape)
    m.ks[:], m.vs[:] = 0.01, 0.01
    t = put(gpu, m)
    q = rng.standard_normal((2, heads, hd)).astype(np.float32)
    sides = [(g, DecodeScratch(), g.upload(q[i])) for i, g in enumerate((gpu, other))]
    want = [g.download(g.decode_batched_q8(x, [t], [live], [cap], heads, kv, hd, 0.09, s)) for g, s, x in sides]
    outs = [[], []]
    for _ in range(20):
        for i, (g, s, x) in enumerate(sides):
            outs[i].append(g.decode_batched_q8(x, [t], [live], [cap], heads, kv, hd, 0.09, s))
    for i, (g, s, x) in enumerate(sides):
        assert all(np.array_equal(g.download(o), want[i]) for o in outs[i])
    sides[1][1].close()
    other.close()


# ---- refusals --------------------------------------------------------------------------------------------------

def test_refusals(gpu):
    heads, kv, hd, cap = 8, 2, 64, 64
    t, u = gpu.kv_alloc_q8(kv, hd, cap), gpu.kv_alloc_q8(kv, hd, cap)
    q, k = gpu.zeros(2 * heads * hd), gpu.zeros(2 * kv * hd)
    f = gpu.rope_inv_freq(10000.0, hd)
    s = DecodeScratch()
    before = gpu.launch_count()

    def append(q=q, k=k, v=k, cu=(0, 1, 2), caches=(t, u), caps=(cap, cap), past=(0, 0), pos=(0, 0), inv=f, heads=heads, kv=kv, hd=hd, q_out=None):
        gpu.rope_append_q8(q, k, v, list(cu), list(caches), list(caps), list(past), list(pos), inv, heads, kv, hd, q_out=q_out)

    for error, args in [
        (CacheOverrun, dict(past=(0, 64))), (CacheOverrun, dict(past=(-1, 0))), (InvalidArgument, dict(caches=(t, t))),
        (InvalidArgument, dict(cu=(0, 2, 1))), (InvalidArgument, dict(cu=(-1, 1, 2))), (SliceOverrun, dict(cu=(0, 1, 3))),
        (InvalidArgument, dict(pos=(0, -1))), (InvalidArgument, dict(pos=((1 << 31) - 1, 0))), (RaggedBlock, dict(caps=(48, 64))),
        (UnsupportedAttention, dict(hd=96)), (UnsupportedAttention, dict(kv=0)), (SliceOverrun, dict(caps=(64, 96))),
        (SliceOverrun, dict(inv=f[:hd // 2 - 1])), (Misaligned, dict(k=gpu.zeros(2 * kv * hd + 1)[1:])),
        (SliceOverrun, dict(q_out=q[:heads * hd])), (InvalidArgument, dict(q_out=q[4:], cu=(0, 0, 1))), (InvalidArgument, dict(q=gpu.zeros(2 * heads * hd), q_out=k.new_zeros(1), cu=(0, 0, 0), past=(0,))),
        (InvalidArgument, dict(caches=(t, torch.zeros(t.numel(), dtype=torch.uint8)))), (SliceOverrun, dict(caches=(t, u[:-1]))),
        (InvalidArgument, dict(k=k.half())), (InvalidArgument, dict(v=gpu.zeros(4 * kv * hd)[::2])), (InvalidArgument, dict(q=q.half())),
        (InvalidArgument, dict(inv=f.double())), (InvalidArgument, dict(q_out=q.double())), (InvalidArgument, dict(cu=(0, 1))),
    ]:
        with pytest.raises(error):
            append(**args)

    def decode(q=q, caches=(t, u), live=(1, 1), caps=(cap, cap), heads=heads, kv=kv, hd=hd, **kw):
        gpu.decode_batched_q8(q, list(caches), list(live), list(caps), heads, kv, hd, 0.1, s, **kw)

    for error, args in [
        (CacheOverrun, dict(live=(65, 1))), (CacheOverrun, dict(live=(-1, 1))), (UnsupportedAttention, dict(heads=7)),
        (UnsupportedAttention, dict(heads=18, q=gpu.zeros(4 * 18 * hd))), (SliceOverrun, dict(q=q[:-4])), (SliceOverrun, dict(out=q[:-4])),
        (InvalidArgument, dict(caches=(t, t), weigh=True)), (InvalidArgument, dict(out=q.double())), (InvalidArgument, dict(live=(1,))),
        (InvalidArgument, dict(q=q.half())), (InvalidArgument, dict(out=gpu.zeros(4 * heads * hd)[::2])),
        (InvalidArgument, dict(out=q)), (InvalidArgument, dict(out=q.view(torch.float16)[heads * hd:])),
        (Misaligned, dict(out=gpu.zeros(2 * heads * hd + 1)[1:])), (RaggedBlock, dict(caps=(40, 64))),
    ]:
        with pytest.raises(error):
            decode(**args)

    def flash(q=q, cu=(0, 1, 2), caches=(t, u), caps=(cap, cap), past=(0, 0), heads=heads, kv=kv, hd=hd, **kw):
        gpu.flash_attn_q8(q, list(cu), list(caches), list(caps), list(past), heads, kv, hd, 0.1, True, **kw)

    for error, args in [(CacheOverrun, dict(past=(64, 0))), (CacheOverrun, dict(past=(-1, 0))), (UnsupportedAttention, dict(heads=7)),
                        (SliceOverrun, dict(cu=(0, 1, 3))), (InvalidArgument, dict(cu=(0, 2, 1))), (Misaligned, dict(q=gpu.zeros(2 * heads * hd + 1)[1:])),
                        (InvalidArgument, dict(out=q)), (InvalidArgument, dict(q=q.half()))]:
        with pytest.raises(error):
            flash(**args)

    def evict(src=(t,), sc=(cap,), dst=(u,), dc=(cap,), live=(64,), keep=(1,), first=0, recent=0, **kw):
        gpu.cache_evict_q8(list(src), list(sc), list(dst), list(dc), list(live), list(keep), first, recent, kv, hd, **kw)

    for error, args in [(InvalidArgument, dict(first=1, recent=1)), (InvalidArgument, dict(keep=(-1,))),
                        (InvalidArgument, dict(first=-1, recent=2)), (InvalidArgument, dict(recent=-1)),
                        (InvalidArgument, dict(first=(1 << 63) + 1, recent=1 << 63)), (CacheOverrun, dict(live=(65,))),
                        (InvalidArgument, dict(dst=(t,), dc=(32,))), (CacheOverrun, dict(dc=(32,), live=(63,), sc=(64,))),
                        (InvalidArgument, dict(src=(t, t), sc=(cap,) * 2, dst=(u, u), dc=(cap,) * 2, live=(64,) * 2, keep=(1,) * 2)),
                        (SliceOverrun, dict(index=torch.zeros(1, dtype=torch.int32, device=gpu.device))),
                        (InvalidArgument, dict(index=torch.zeros(9, device=gpu.device)))]:
        with pytest.raises(error):
            evict(**args)
    with pytest.raises(CacheOverrun):
        gpu.cache_rewind_q8([t], [cap], [10], [11], kv, hd)
    with pytest.raises(InvalidArgument):
        gpu.cache_rewind_q8([t, t], [cap] * 2, [40] * 2, [33] * 2, kv, hd)
    with pytest.raises(CacheOverrun):
        gpu.cache_read_q8([t], [cap], [10], [5], [0, 6], kv, hd)
    rows = torch.empty(5 * kv * hd, dtype=torch.float16, device=gpu.device)
    with pytest.raises(InvalidArgument):
        gpu.cache_read_q8([t], [cap], [10], [5], [0, 5], kv, hd, k_out=rows, v_out=rows)
    with pytest.raises(InvalidArgument):
        gpu.cache_read_q8([t], [cap], [10], [5], [0, 5], kv, hd, k_out=rows.float(), v_out=rows)
    with pytest.raises(SliceOverrun):
        gpu.cache_read_q8([t], [cap], [10], [5], [0, 5], kv, hd, k_out=torch.empty(4, dtype=torch.float16, device=gpu.device))
    with pytest.raises(CacheOverrun):
        gpu.cache_grow_q8(t, u, kv, hd, 64, 32, 10)
    with pytest.raises(InvalidArgument):
        gpu.cache_grow_q8(t, t, kv, hd, 64, 64, 10)
    with pytest.raises(RaggedBlock):
        gpu.kv_alloc_q8(kv, hd, 50)
    with pytest.raises(OddHeadDim):
        gpu.rope_inv_freq(10000.0, 65)
    assert gpu.launch_count() == before


def test_calls_with_nothing_to_do_launch_nothing(gpu):
    heads, kv, hd, cap = 8, 2, 64, 64
    t = gpu.kv_alloc_q8(kv, hd, cap)
    q, k = gpu.zeros(heads * hd), gpu.zeros(kv * hd)
    before = gpu.launch_count()
    gpu.rope_append_q8(q, k, k, [0, 0], [t], [cap], [0], [0], None, heads, kv, hd)
    gpu.rope_append_q8(q, k, k, [0], [], [], [], [], None, heads, kv, hd)
    gpu.flash_attn_q8(q, [0, 0], [t], [cap], [0], heads, kv, hd, 0.1, True)
    gpu.cache_read_q8([t], [cap], [10], [5], [0, 0], kv, hd)
    gpu.cache_rewind_q8([t], [cap], [40], [32], kv, hd)
    gpu.decode_batched_q8(q, [], [], [], heads, kv, hd, 0.1, DecodeScratch())
    assert gpu.launch_count() == before
