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
