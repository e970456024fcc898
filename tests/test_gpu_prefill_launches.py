"""Captured prefills: two graphs of one handle that run beside each other, and more
launches in a graph than the handle has counters for; and few rows over a long context."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, HD, ROWS = 32, 8, 128, 2048      # 256 pairs of query tiles: more than the device has SMs


def prefill(gpu, seed):
    r = np.random.default_rng(seed)
    q = gpu.upload(r.standard_normal((ROWS, HEADS * HD), dtype=np.float32))
    k = gpu.upload_f16(r.standard_normal((KV, ROWS, HD), dtype=np.float32))
    v = gpu.upload_f16(r.standard_normal((KV, HD, ROWS), dtype=np.float32))

    def run():
        return gpu.flash_attn_f16(q, k, v, ROWS, 0, HEADS, KV, HD, ROWS, HD ** -0.5, True)
    return run


def captured(gpu, run, times=1):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=gpu.stream):
        outs = [run() for _ in range(times)]
    return graph, outs


def test_graphs_replayed_beside_each_other_and_beside_a_call(gpu):
    runs = [prefill(gpu, s) for s in range(3)]
    want = [f() for f in runs]
    gpu.synchronize()
    graphs = [captured(gpu, f, times=4) for f in runs[:2]]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for _, outs in graphs:
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = runs[2]()
        torch.cuda.synchronize()
        for (_, outs), w in zip(graphs, want):
            for o in outs:
                assert torch.equal(o, w)
        assert torch.equal(eager, want[2])
    gpu.synchronize()


def test_captured_after_the_counters_are_used_up(gpu):
    from ttsxabe_b200 import Gpu
    own = Gpu.open(0)
    run = prefill(own, 7)
    want = run()
    own.synchronize()
    out = own.uninit(ROWS * HEADS * HD)
    for _ in range(9):                       # 9 x 1024 launches of one small item each
        captured(own, small(own, out), times=1024)
    graph, outs = captured(own, run)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    own.synchronize()
    graph.reset()
    own.close()


def small(gpu, out):
    q, k, v = gpu.zeros(128 * 2 * HD), gpu.zeros_f16(128 * HD), gpu.zeros_f16(128 * HD)

    def run():
        gpu._lib.llmtie_flash_attn_f16(gpu._h, q.data_ptr(), q.numel(), k.data_ptr(), k.numel(), v.data_ptr(), v.numel(),
                                       out.data_ptr(), out.numel(), 128, 0, 2, 1, HD, 128, 0.1, 1)
    return run


@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 128), (2, 1, 128)])
def test_few_rows_of_one_pair_of_heads_over_a_long_context(gpu, heads, kv, hd):
    """The keys are cut into as many pieces as there are SMs for a pair of heads."""
    past, rows = 131072 - 100, 100
    n = past + rows
    torch.manual_seed(5)
    q = torch.randn(rows, heads, hd, device=gpu.device)
    k = torch.randn(kv, n + 4, hd, device=gpu.device).half()
    v = torch.randn(kv, hd, n + 4, device=gpu.device).half()
    v[:, :, :past] += torch.linspace(-1, 1, past, device=gpu.device).half()     # (a piece left out or taken twice shows)
    torch.cuda.synchronize()
    out = gpu.flash_attn_f16(q, k, v, rows, past, heads, kv, hd, n + 4, hd ** -0.5, True)
    gpu.synchronize()
    out = out.view(rows, heads, hd)
    for h in range(heads):
        kh, vh = k[h // (heads // kv), :n].double(), v[h // (heads // kv), :, :n].double()
        s = q[:, h].double() @ kh.T * hd ** -0.5
        s.masked_fill_(torch.arange(n, device=gpu.device)[None] > past + torch.arange(rows, device=gpu.device)[:, None], float("-inf"))
        want = torch.softmax(s, -1) @ vh.T
        # scores off by 2^-11 of q and the probabilities and the sum by as much, each in
        # proportion to a mean of |v| of about one: against values of either sign
        assert (out[:, h].double() - want).abs().max().item() <= 4 * 2.0 ** -11
