"""Keeping a conversation whose 8-bit caches have evicted blocks: what a cut leaves, and
where none is possible."""
import numpy as np
import pytest
import torch

from ttsxabe_b200 import InvalidArgument, KvCacheQ8, Prefix, evicted_len


class NoDevice:
    """The calls that a KvCacheQ8 makes, remembered."""

    def __init__(self):
        self.cuts = []

    def kv_alloc_q8(self, kv, hd, cap):
        return cap

    def rope_append_q8(self, *args, **kw):
        pass

    def cache_grow_q8(self, *args):
        pass

    def cache_evict_q8(self, *args):
        pass

    def cache_rewind_q8(self, caches, cap, live, to, kv, hd):
        self.cuts.append((live, to))


def conversation(n, layers=2, keep=6, recent=2):
    g = NoDevice()
    caches = [KvCacheQ8(g, 2, 64, 4096) for _ in range(layers)]
    p = Prefix(caches)
    ids = list(range(n))
    assert p.keep(ids) == 0
    for c in caches:
        c.append(None, None, None, n, None, 2)
        c.evict(keep, 1, recent)
    p.extend(ids)
    return g, p


def test_a_cut_among_the_most_recent_tokens_leaves_the_caches_shorter_than_the_conversation():
    g, p = conversation(340)
    held = evicted_len(340, 6)
    assert p.past == [held, held] and len(p) == 340
    # 64 tokens of recent blocks and the 20 of the tail may be cut
    assert p.keep(list(range(300)) + [-1]) == 300
    assert p.past == [held - 40] * 2 and [c.pos for c in p.caches] == [300, 300] and len(p) == 300
    assert g.cuts == [([held], [held - 40])] * 2


def test_a_cut_among_evicted_blocks_keeps_nothing():
    g, p = conversation(340)
    assert not p.caches[0].can_truncate(255) and p.caches[0].can_truncate(256) and p.caches[0].can_truncate(0)
    assert p.keep(list(range(255)) + [-1]) == 0
    assert p.past == [0, 0] and [c.pos for c in p.caches] == [0, 0] and len(p) == 0 and not g.cuts


def test_layers_are_cut_together_or_not_at_all():
    g, p = conversation(340)
    p.caches[1].evict(2, 1, 1)
    assert p.keep(list(range(280)) + [-1]) == 0           # (the second layer kept one recent block)
    assert p.past == [0, 0] and not g.cuts


def test_a_cache_by_itself_still_refuses():
    g, p = conversation(340, layers=1)
    with pytest.raises(InvalidArgument, match="evicted"):
        p.caches[0].truncate(100)
    assert p.past == [evicted_len(340, 6)]


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [330, 290])
def test_a_prompt_behind_what_an_eviction_left(gpu, shared):
    from tests.helpers import assert_parity
    from tests.q8_model import attend

    heads, kv, hd, n, new = 8, 2, 64, 340, 40
    scale = hd ** -0.5
    torch.manual_seed(shared)
    c = KvCacheQ8(gpu, kv, hd, 4096)
    p = Prefix([c])
    f = gpu.rope_inv_freq(10000.0, hd)

    def append(rows):
        q, k, v = (torch.randn(rows, w * hd, device=gpu.device) for w in (heads, kv, kv))
        torch.cuda.synchronize()
        c.append(q, k, v, rows, f, heads)
        return q

    assert p.keep(list(range(n))) == 0
    append(n)
    p.extend(range(n))
    c.evict(6, 1, 2)
    assert p.keep(list(range(shared)) + [-1] * new) == shared
    past = p.past
    assert past == [evicted_len(n, 6) - (n - shared)]
    q = append(new)
    out = gpu.download(gpu.flash_attn_q8(q, [0, new], [c.data], [c.cap], past, heads, kv, hd, scale, True))
    ko, vo = gpu.cache_read_q8([c.data], [c.cap], [c.len], [0], [0, c.len], kv, hd)
    gpu.synchronize()
    kk, vv = (x.double().cpu().numpy().reshape(-1, kv, hd).transpose(1, 0, 2) for x in (ko, vo))
    qq = q.double().cpu().numpy().reshape(new, heads, hd)
    want, _ = attend(qq, kk, vv, scale, past[0] + np.arange(new))
    assert_parity("behind an eviction", want, out.reshape(want.shape))
