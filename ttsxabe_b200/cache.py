"""The f16 KV cache of one layer and its growth policy.

`KvCache` is what `Cache`/`LayerCache` are in the model crates
(crates/llmtie-chat/src/model.rs:200-262, :714-747;
crates/llmtie-translate/src/model.rs:662-694): keys `[kv_heads][cap][hd]`,
values transposed `[kv_heads][hd][cap]`, both zeroed at allocation, capacity
a power of two of at least 256 that doubles by re-striding, `truncate` only
lowering the live length.
"""
from __future__ import annotations

from . import _lib
from .gpu import Gpu, InvalidArgument, evicted_len


def want_capacity(cap: int, past: int, n: int, max_positions: int) -> int:
    """Capacity to allocate so a cache of `cap` holds past + n positions; 0 if
    it already does (chat/model.rs:714-721)."""
    return int(_lib.load().llmtie_kv_want_capacity(cap, past, n, max_positions))


class KvCache:
    def __init__(self, gpu: Gpu, kv_heads: int, head_dim: int, max_positions: int) -> None:
        self.gpu = gpu
        self.kv_heads = kv_heads
        self.head_dim = head_dim
        self.max_positions = max_positions
        self.cap = 0
        self.len = 0
        self.k = None
        self.v = None

    def reserve(self, n: int) -> None:
        """Makes room for n more positions, growing by re-stride when needed."""
        want = want_capacity(self.cap, self.len, n, self.max_positions)
        if want == 0:
            return
        g = self.gpu
        kv_dim = self.kv_heads * self.head_dim
        k = g.zeros_f16(want * kv_dim)
        v = g.zeros_f16(want * kv_dim)
        if self.len > 0:
            g.cache_grow_f16(self.k, k, self.kv_heads, self.head_dim, self.cap, want, self.len,
                             False)
            g.cache_grow_f16(self.v, v, self.kv_heads, self.head_dim, self.cap, want, self.len,
                             True)
        self.k, self.v, self.cap = k, v, want

    def append(self, k_src, v_src, src_off_k: int, src_off_v: int, n: int) -> None:
        """Appends n positions of projected (already rotated) k and v."""
        self.reserve(n)
        g = self.gpu
        g.cache_append_f16(k_src, src_off_k, self.k, n, self.kv_heads, self.head_dim, self.cap,
                           self.len, False)
        g.cache_append_f16(v_src, src_off_v, self.v, n, self.kv_heads, self.head_dim, self.cap,
                           self.len, True)
        self.len += n

    def truncate(self, length: int) -> None:
        """Forgets every position from `length` on. Nothing is zeroed: attention
        reads only the live positions, and the next prefill writes its own keys
        and values from `length` before any attention reads them."""
        self.len = min(self.len, length)

    def clear(self) -> None:
        self.len = 0


class KvCacheQ8:
    """The 8-bit KV cache of one layer, with the growth policy of `KvCache`
    (capacities rounded up to whole blocks of 32 tokens). `len` counts the tokens
    it holds, `pos` those of the conversation: an eviction makes it the shorter
    of the two, and new tokens go on at `pos`."""

    def __init__(self, gpu: Gpu, kv_heads: int, head_dim: int, max_positions: int) -> None:
        self.gpu = gpu
        self.kv_heads = kv_heads
        self.head_dim = head_dim
        self.max_positions = max_positions
        self.cap = 0
        self.len = 0
        self.pos = 0
        self.newest = 0     # this many of the last tokens lie as they came, no block gone among them
        self.data = None

    def reserve(self, n: int) -> None:
        """Makes room for n more positions."""
        want = want_capacity(self.cap, self.len, n, self.max_positions)
        if want == 0:
            return
        want = (want + 31) // 32 * 32
        g = self.gpu
        data = g.kv_alloc_q8(self.kv_heads, self.head_dim, want)
        if self.len > 0:
            g.cache_grow_q8(self.data, data, self.kv_heads, self.head_dim, self.cap, want,
                            self.len)
        self.data, self.cap = data, want

    def append(self, q, k, v, n: int, inv_freq, heads: int, q_out=None) -> None:
        """Rotates n projected rows of q, k and v and appends those of k and v."""
        self.reserve(n)
        self.gpu.rope_append_q8(q, k, v, [0, n], [self.data], [self.cap], [self.len], [self.pos],
                                inv_freq, heads, self.kv_heads, self.head_dim, q_out=q_out)
        self.len += n
        self.pos += n
        self.newest += n

    def evict(self, keep: int, keep_first: int = 1, keep_recent: int = 1) -> None:
        """Keeps `keep` complete blocks, in place: the first, the most recent, and
        those that decode steps with `weigh` gave the most weight."""
        if self.len // 32 <= keep:
            return
        self.gpu.cache_evict_q8([self.data], [self.cap], [self.data], [self.cap], [self.len],
                                [keep], keep_first, keep_recent, self.kv_heads, self.head_dim)
        self.newest = min(self.newest, 32 * keep_recent + self.len % 32)
        self.len = evicted_len(self.len, keep)

    def can_truncate(self, length: int) -> bool:
        """Whether the conversation can be cut to `length` positions: not where blocks
        have been evicted among what would stay or go."""
        return length == 0 or self.pos - length <= self.newest

    def truncate(self, length: int) -> None:
        """Forgets every position of the conversation from `length` on."""
        gone = self.pos - length
        if gone <= 0:
            return
        if length == 0:
            self.clear()
            return
        if not self.can_truncate(length):
            raise InvalidArgument(f"cutting a conversation of {self.pos} positions to {length}: "
                                  f"blocks before the last {self.newest} have been evicted")
        self.gpu.cache_rewind_q8([self.data], [self.cap], [self.len], [self.len - gone],
                                 self.kv_heads, self.head_dim)
        self.len -= gone
        self.newest -= gone
        self.pos = length

    def clear(self) -> None:
        self.len = self.pos = self.newest = 0


def shared_prefix(held, ids) -> int:
    """Leading tokens of `ids` that a cache holding `held` can keep (never all
    of `ids`: the last token is always run)."""
    import ctypes as C

    h = (C.c_uint32 * len(held))(*held)
    i = (C.c_uint32 * len(ids))(*ids)
    return int(_lib.load().llmtie_kv_shared_prefix(h, len(held), i, len(ids)))


class Prefix:
    """`Prefix` (crates/llmtie-chat/src/generate.rs:258-283): the caches of one
    conversation kept from one completion to the next, with exactly the tokens
    they hold. A turn's prompt shares its opening with the last one, so only
    the tokens from the first that differs are prefilled."""

    def __init__(self, caches) -> None:
        self.caches = list(caches)          # one KvCache or KvCacheQ8 a layer
        self.held: list[int] = []

    def __len__(self) -> int:
        return len(self.held)

    def shared_with(self, ids) -> int:
        n = 0
        for a, b in zip(self.held, ids):
            if a != b:
                break
            n += 1
        return n

    def keep(self, ids) -> int:
        """Cuts the caches back to what they share with the prompt `ids`
        (generate.rs:139-141) and returns that length: the prompt is run from
        there on, at the rotary positions from there on, behind what each cache
        holds (`past`: the returned value, but for 8-bit caches that have evicted
        blocks). Where the cut would fall among evicted blocks nothing is kept."""
        reused = shared_prefix(self.held, ids)
        if any(isinstance(c, KvCacheQ8) and not c.can_truncate(reused) for c in self.caches):
            reused = 0
        for c in self.caches:
            c.truncate(reused)
        del self.held[reused:]
        return reused

    @property
    def past(self) -> list[int]:
        """How many tokens each layer's cache holds: what a call that appends to it or
        attends over it is given as `past`."""
        return [c.len for c in self.caches]

    def extend(self, ids) -> None:
        """Records tokens the caches now hold (after a prefill or a decoded step)."""
        self.held.extend(int(x) for x in ids)

    def reset(self) -> None:
        """What complete_after does when a completion failed half way."""
        for c in self.caches:
            c.clear()
        self.held.clear()
