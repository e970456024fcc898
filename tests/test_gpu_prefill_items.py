"""Prefill launches of more items than the device has SMs, whose blocks take one item
after another: items of a single key tile, and tiles that have no rows."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def attention(q, k, v, scale, first):
    """q f64 [n][heads][hd] over k, v f64 [kv][t][hd], row i over keys up to first + i.
    Returns the result and what the kernel may be off by: its probabilities are
    rounded to f16, half a step of 2^-10 each, or of 2^-24 where they are subnormal (in
    units of a row's largest or more), against values of either sign."""
    n, heads, hd = q.shape
    out, tol = torch.empty_like(q), torch.empty_like(q)
    hidden = torch.arange(k.shape[1], device=q.device)[None] > first + torch.arange(n, device=q.device)[:, None]
    for h in range(heads):
        kh, vh = k[h // (heads // k.shape[0])], v[h // (heads // k.shape[0])]
        e = (q[:, h] @ kh.T * scale).masked_fill(hidden, float("-inf"))
        e = torch.exp(e - e.max(-1, keepdim=True).values)
        l = e.sum(-1, keepdim=True)
        out[:, h] = e / l @ vh
        seen = (~hidden).double() @ vh.abs()
        # (a twentieth more, and 2^-18, for the 32-bit sums and exponentials)
        tol[:, h] = 1.05 * (2.0 ** -11 * (e / l @ vh.abs()) + 2.0 ** -25 * seen / l) + 2.0 ** -18
    return out, tol


class Batch:
    """Prompts of new[b] rows behind past[b] tokens, over 8-bit caches."""

    def __init__(self, gpu, heads, kv, hd, past, new, seed):
        self.gpu, self.shape, self.past, self.new = gpu, (heads, kv, hd), past, new
        torch.manual_seed(seed)
        self.cu = np.concatenate([[0], np.cumsum(new)]).tolist()
        live = [p + n for p, n in zip(past, new)]
        self.cap = [(n + 31) // 32 * 32 for n in live]
        rows = np.concatenate([[0], np.cumsum(live)]).tolist()
        self.caches = [gpu.kv_alloc_q8(kv, hd, c) for c in self.cap]
        self.q = torch.randn(self.cu[-1], heads, hd, device=gpu.device).half().float()
        k, v = torch.randn(2, rows[-1], kv, hd, device=gpu.device)
        torch.cuda.synchronize()
        zeros = [0] * len(new)
        gpu.rope_append_q8(None, k, v, rows, self.caches, self.cap, zeros, zeros, None, heads, kv, hd)
        ko, vo = gpu.cache_read_q8(self.caches, self.cap, live, zeros, rows, kv, hd)
        gpu.synchronize()
        self.kv16 = [[x.view(-1, kv, hd)[a:b].double().transpose(0, 1) for x in (ko, vo)] for a, b in zip(rows, rows[1:])]

    def run(self):
        heads, kv, hd = self.shape
        out = self.gpu.flash_attn_q8(self.q, self.cu, self.caches, self.cap, self.past, heads, kv, hd, hd ** -0.5, True)
        return out.view(-1, heads, hd)

    def check(self, out):
        for b, (k, v) in enumerate(self.kv16):
            rows = slice(self.cu[b], self.cu[b + 1])
            if self.new[b]:
                want, tol = attention(self.q[rows].double(), k, v, self.shape[2] ** -0.5, self.past[b])
                assert ((out[rows].double() - want).abs() <= tol).all(), f"sequence {b}"


# heads to a KV head: odd, so that an item is two row blocks of one head
@pytest.mark.parametrize("heads,kv,hd", [(36, 4, 64), (27, 3, 128)])
@pytest.mark.parametrize("rows", [(1, 128), (1, 300)])
def test_items_of_a_tile_or_two_whose_second_tile_is_often_empty(gpu, heads, kv, hd, rows):
    """32 sequences of up to 128 rows are items of one key tile whose second row block
    has no rows; with up to 300 rows they alternate with items of both."""
    rng = np.random.default_rng(rows[1])
    new = [int(x) for x in rng.integers(*rows, 32)]
    b = Batch(gpu, heads, kv, hd, [0] * 32, new, seed=hd)
    first = b.run()
    gpu.synchronize()
    b.check(first)
    for _ in range(30):
        again = b.run()
        gpu.synchronize()
        assert torch.equal(again, first)


def test_long_items_among_many_short_ones(gpu):
    """A few items of 40 key tiles and both row blocks, many of one tile and one."""
    past = [5000, 0, 4900] + [0] * 29
    new = [200, 256, 130] + [1 + 4 * i for i in range(29)]
    b = Batch(gpu, 27, 3, 128, past, new, seed=1)
    first = b.run()
    gpu.synchronize()
    b.check(first)
    for _ in range(10):
        again = b.run()
        gpu.synchronize()
        assert torch.equal(again, first)


@pytest.mark.parametrize("heads,kv,hd", [(36, 4, 64), (27, 3, 128), (32, 8, 128)])
def test_a_launch_whose_waits_run_out_ends_and_leaves_the_next_one_right(gpu, heads, kv, hd):
    """With a limit of a cycle or a few thousand, waits give up anywhere in an item.
    The launch ends, says so once, and what comes after it is whole."""
    from ttsxabe_b200 import DeviceTimeout

    past, new = [700] + [0] * 31, [300] + [1 + 9 * i for i in range(31)]
    b = Batch(gpu, heads, kv, hd, past, new, seed=2)
    want = b.run()
    gpu.synchronize()
    b.check(want)
    for limit in (1, 500, 3000, 10000, 30000):
        gpu.set_wait_limit_cycles(limit)
        try:
            b.run()
            try:
                gpu.synchronize()
                reported = False
            except DeviceTimeout:
                reported = True
            gpu.synchronize()
        finally:
            gpu.set_wait_limit_cycles(0)
        assert reported or limit > 1
        again = b.run()
        gpu.synchronize()
        assert torch.equal(again, want)


def test_the_wait_limit_is_one_for_a_step_however_long_an_item_is(gpu):
    """Items of 512 key tiles without a second row block: the warps that sit an item out
    wait much longer than 200000 cycles (0.1 ms), none waits as long for a step."""
    heads, kv, hd, rows, n = 156, 52, 128, 100, 65536
    torch.manual_seed(4)
    q = torch.randn(rows, heads, hd, device=gpu.device).half().float()
    k = torch.randn(kv, n, hd, device=gpu.device, dtype=torch.float16)
    v = torch.randn(kv, hd, n, device=gpu.device, dtype=torch.float16)
    torch.cuda.synchronize()
    gpu.set_wait_limit_cycles(200_000)
    try:
        out = gpu.flash_attn_f16(q, k, v, rows, n - rows, heads, kv, hd, n, hd ** -0.5, True).view(rows, heads, hd)
        gpu.synchronize()
    finally:
        gpu.set_wait_limit_cycles(0)
    for j in (0, 25, 51):
        group = slice(3 * j, 3 * j + 3)
        want, tol = attention(q[:, group].double(), k[j:j + 1].double(), v[j:j + 1].double().transpose(1, 2), hd ** -0.5, n - rows)
        assert ((out[:, group].double() - want).abs() <= tol).all(), f"KV head {j}"
