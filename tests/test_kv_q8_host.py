"""The 8-bit cache's host side: sizes, refusals that need no device, and the
model the GPU tests are held to."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests.q8_model import Q8Model, attend, rotate, sections
from ttsxabe_b200 import Gpu, InvalidArgument, UnsupportedAttention, _lib, decode_plan_q8, evicted_len, kv_q8_bytes


@pytest.mark.parametrize("kv,hd,cap", [(8, 128, 4096), (20, 64, 1504), (1, 64, 32), (3, 128, 96)])
def test_size_is_that_of_the_documented_layout(kv, hd, cap):
    assert kv_q8_bytes(kv, hd, cap) == sections(kv, hd, cap)[1]


def test_shapes_without_a_cache():
    assert kv_q8_bytes(8, 96, 64) == 0
    assert kv_q8_bytes(0, 64, 64) == 0
    assert kv_q8_bytes(8, 64, 65) == 0


def test_half_the_bytes_of_an_f16_cache():
    # codes are half of it; scales, weights and the tail add little to a long cache
    kv, hd, cap = 8, 128, 131072
    assert kv_q8_bytes(kv, hd, cap) < 0.505 * (2 * kv * hd * cap * 2)


def test_null_handle_is_refused():
    lib = _lib.load()
    z, i = C.c_void_p(), (C.c_int32 * 2)(0, 0)
    p = (C.c_void_p * 1)()
    assert lib.llmtie_rope_append_q8(None, z, 0, z, 0, z, 0, z, 0, i, 1, p, i, i, i, z, 0, 8, 8, 64) == 12
    assert lib.llmtie_decode_batched_q8(None, z, 0, p, i, i, 1, 8, 8, 64, 1.0, 0, z, z, 0, 0) == 12
    assert lib.llmtie_flash_attn_q8(None, z, 0, i, 1, p, i, i, 8, 8, 64, 1.0, 1, z, 0, 0) == 12
    assert lib.llmtie_cache_evict_q8(None, p, i, p, i, i, i, 1, 0, 0, 8, 64, z, 0) == 12
    assert lib.llmtie_cache_read_q8(None, p, i, i, i, i, 1, 8, 64, z, 0, z, 0) == 12
    assert lib.llmtie_cache_rewind_q8(None, p, i, i, i, 1, 8, 64) == 12
    assert lib.llmtie_cache_grow_q8(None, z, 0, z, 0, 8, 64, 64, 64, 1) == 12
    assert lib.llmtie_rope_inv_freq(None, z, 64, 10000.0, z, 0) == 12


def test_evicted_len():
    assert evicted_len(100, 2) == 68
    assert evicted_len(100, 3) == evicted_len(100, 9) == 100
    assert evicted_len(96, 0) == 0


def test_model_codes_are_within_half_a_step():
    rng = np.random.default_rng(0)
    m = Q8Model(2, 64, 96)
    k, v = rng.standard_normal((2, 70, 2, 64)).astype(np.float32)
    m.append(k[:5], v[:5], 0)
    m.append(k[5:], v[5:], 5)
    for which, x in (("k", k), ("v", v)):
        e = np.abs(m.values(which, 70) - x.transpose(1, 0, 2))
        step = (m.ks if which == "k" else m.vs)[:, :2].repeat(32, 1)[..., None]
        # half a step of the codes, and half a step of f16 before it
        assert (e[:, :64] <= 0.5 * step * (1 + 1e-6) + 2.0 ** -11 * np.abs(x.transpose(1, 0, 2)[:, :64])).all()
        assert (e[:, 64:] <= 2.0 ** -11 * np.abs(x.transpose(1, 0, 2)[:, 64:])).all()


def test_model_attention_and_rotation():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((3, 4, 8)), rng.standard_normal((1, 6, 8)), rng.standard_normal((1, 6, 8))
    o, p = attend(q, k, v, 0.5, [0, 3, 5])
    assert np.allclose(p.sum(-1), 1) and np.allclose(o[0], v[0, 0]) and (p[1, :, 4:] == 0).all()
    f = np.array([1.0, 0.5, 0.1, 0.01])
    assert np.allclose(np.linalg.norm(rotate(q, 9, f), axis=-1), np.linalg.norm(q, axis=-1))
    # a score depends on the distance alone
    a, b = rotate(q[:1], 3, f), rotate(q[1:2], 10, f)
    c, d = rotate(q[:1], 103, f), rotate(q[1:2], 110, f)
    assert np.allclose((a * b).sum(-1), (c * d).sum(-1))


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_plan(hd):
    most = 148 * (2 if hd == 128 else 3)
    rng = np.random.default_rng(hd)
    seen = set()
    for _ in range(400):
        kv = int(rng.choice([1, 2, 8, 20]))
        n = int(rng.integers(1, 33))
        live = [int(x) for x in np.exp(rng.uniform(0, np.log(40000), n))]
        grid, cluster, ns = decode_plan_q8(live, kv, hd)
        pairs, units = n * kv, kv * sum((t + 31) // 32 for t in live)
        seen.add(cluster)
        assert ns > 0
        if cluster:
            parts, rest = divmod(grid, pairs * cluster)
            assert rest == 0 and parts >= 1 and cluster in (1, 2, 4, 8, 16)
            assert parts == 1 or (cluster == 8 and parts <= 32 and pairs * parts <= 36)
            assert cluster == 1 or grid <= most
            assert cluster < 8 or pairs <= (36 if cluster == 8 else 16)
        else:
            assert 1 <= grid <= min(most, (units + 3) // 4)
    assert {0, 1, 2, 4} <= seen
    assert decode_plan_q8([2048], 8, hd)[1] in (8, 16)
    assert decode_plan_q8([131072] * 8, 8, hd)[0] <= most
    # few pairs of many blocks: several clusters each
    grid, cluster, _ = decode_plan_q8([40000, 30000], 1, hd)
    assert cluster == 8 and grid >= 10 * 16
    # no clusters where the device holds none; nothing for no tokens
    assert decode_plan_q8([2048], 8, hd, resident=(0, 0))[1] <= 4
    assert decode_plan_q8([0, 0], 8, hd)[:2] == (0, 0)


def test_decode_plan_refusals():
    with pytest.raises(UnsupportedAttention):
        decode_plan_q8([5], 8, 96)
    with pytest.raises(InvalidArgument):
        decode_plan_q8([5] * 33, 8, 64)
    with pytest.raises(InvalidArgument):
        decode_plan_q8([5], 8, 64, sm_count=0)


def test_a_cache_of_another_device_is_refused():
    """A list of caches is checked before the table of their addresses is made."""
    class Cache:
        is_cuda, device = True, torch.device("cuda", 1)

        def numel(self):
            return 1 << 20

        def element_size(self):
            return 1

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 1 << 20

    def table(ordinal, caches, cap):
        gpu = Gpu.__new__(Gpu)
        gpu._h, gpu.ordinal = None, ordinal
        return gpu._q8_table(caches, cap, 2, 64)

    assert table(1, [Cache()], [64])[0] == 1 << 20
    for args in [(0, [Cache()], [64]), (1, [torch.zeros(1 << 20)], [64])]:
        with pytest.raises(InvalidArgument, match="not cuda"):
            table(*args)
