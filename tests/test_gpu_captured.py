"""Captured calls: what the handle does meanwhile leaves them alone."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def prefill(gpu, rows, past, heads, kv, hd, seed):
    torch.manual_seed(seed)
    n = past + rows
    cap = (n + 7) // 8 * 8
    q = torch.randn(rows, heads * hd, device=gpu.device)
    k = torch.randn(kv, cap, hd, device=gpu.device).half()
    v = torch.randn(kv, hd, cap, device=gpu.device).half()
    torch.cuda.synchronize()
    return lambda: gpu.flash_attn_f16(q, k, v, rows, past, heads, kv, hd, cap, hd ** -0.5, True)


def captured(gpu, run, times=1):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu.stream):
        outs = [run() for _ in range(times)]
    return graph, outs


def test_a_timeout_reported_while_a_graph_runs_on_another_stream(gpu):
    """The wait that runs out is one for a flag that nothing raises (the merge of a
    sharded step); the graph's blocks are taking items off their launches' counters."""
    from tests.test_gpu_aux import _exchange_of_one_device
    from ttsxabe_b200 import DeviceTimeout

    run = prefill(gpu, 2048, 0, 32, 8, 128, seed=3)
    want = run()
    gpu.synchronize()
    graph, outs = captured(gpu, run, times=24)              # some 24 x 45 us
    xch, gather, flags, step = _exchange_of_one_device(gpu, 2, 32, 128, step_value=1)
    gpu.synchronize()
    other = torch.cuda.Stream()
    try:
        for limit in (20_000, 100_000, 200_000, 400_000, 800_000, 1_200_000, 50_000, 300_000):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            gpu.set_wait_limit_cycles(limit)
            with torch.cuda.stream(other):
                graph.replay()
            gpu.lse_merge_wait(xch, 32, 128)
            with pytest.raises(DeviceTimeout):
                gpu.synchronize()
            torch.cuda.synchronize()
            for o in outs:
                assert torch.equal(o, want)
    finally:
        gpu.set_wait_limit_cycles(0)
    with torch.cuda.stream(other):
        graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    gpu.synchronize()


def other_forms(gpu, hd=128):
    """Calls that use each workspace of a handle: {name: make(own handle, size)}, where
    a call of a larger size needs more of it."""
    heads, kv = 8, 2

    def cut(own, size):                       # keys cut into pieces, merged by a second kernel
        return prefill(own, 200, 4000 * size, heads, kv, hd, seed=size)

    def ragged(own, size):                    # a table of cosines and sines
        n = 9000 * size
        torch.manual_seed(size)
        q, k, v = (torch.randn(n, w * hd, device=gpu.device) for w in (heads, kv, kv))
        kc, vc = (torch.zeros(kv * n * hd, dtype=torch.float16, device=gpu.device) for _ in range(2))
        torch.cuda.synchronize()
        return lambda: own.prefill_varlen(q, k, v, [0, n], [kc], [vc], [0], [n], None, heads, kv, hd, 10000.0, hd ** -0.5)

    def staged(own, size):                    # an f16 copy of f32 caches
        n = 3000 * size
        torch.manual_seed(size)
        q = torch.randn(300, heads * hd, device=gpu.device)
        k, v = torch.randn(2, kv * n * hd, device=gpu.device)
        torch.cuda.synchronize()
        return lambda: own.flash_attn(q, k, v, 300, n - 300, heads, kv, hd, n, hd ** -0.5, True)

    def decode(own, size):                    # partial results and counters
        from ttsxabe_b200 import DecodeScratch
        scratch = own.__dict__.setdefault("scratch_of_this_test", DecodeScratch())
        b = 30 * size - 20
        torch.manual_seed(size)
        q = torch.randn(b, heads * hd, device=gpu.device)
        k, v = (torch.randn(kv * 4096 * hd, device=gpu.device).half() for _ in range(2))
        torch.cuda.synchronize()
        return lambda: own.decode_batched(q, [k] * b, [v] * b, [4000] * b, [4096] * b, heads, kv, hd, hd ** -0.5, False, scratch)

    return {"cut": cut, "ragged": ragged, "staged": staged, "decode": decode}


@pytest.mark.parametrize("form", ["cut", "ragged", "staged", "decode"])
def test_a_graph_keeps_what_its_calls_were_given(gpu, form):
    """Captured after one call, replayed after a larger call outgrew the workspace."""
    from ttsxabe_b200 import Gpu

    own = Gpu.open(gpu.ordinal)
    small, large = (other_forms(gpu)[form](own, size) for size in (1, 4))
    want = small()
    own.synchronize()
    graph, outs = captured(own, small)
    more = large()
    own.synchronize()
    first = more.clone()
    for _ in range(3):
        outs[0].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(own.stream):
            graph.replay()
        again = large()
        own.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(again, first)
    graph.reset()
    own.synchronize()
    own.close()


@pytest.mark.parametrize("form", ["cut", "ragged", "staged", "decode"])
def test_growing_under_a_capture_is_refused_and_the_handle_stays_usable(gpu, form):
    from ttsxabe_b200 import Gpu

    own = Gpu.open(gpu.ordinal)
    run = other_forms(gpu)[form](own, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=own.stream):
        with pytest.raises(Exception, match="captur"):
            run()
    out = run()
    own.synchronize()
    want = other_forms(gpu)[form](gpu, 1)()
    gpu.synchronize()
    assert torch.equal(out, want)
    gpu.__dict__.pop("scratch_of_this_test", None)
    graph.reset()
    own.close()
