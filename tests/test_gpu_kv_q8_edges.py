"""The 8-bit KV cache where it could go wrong: waits that run out, values that are not
finite, caches that are forked, buffers in the wrong place."""
import numpy as np
import pytest
import torch

from ttsxabe_b200 import DecodeScratch, DeviceTimeout, decode_plan_q8

pytestmark = pytest.mark.gpu


def caches_of(gpu, kv, hd, lives, seed, cap=None):
    """Caches of random tokens, and their capacities."""
    torch.manual_seed(seed)
    caps = [max(32, (n + 31) // 32 * 32) if cap is None else cap for n in lives]
    ts = [gpu.kv_alloc_q8(kv, hd, c) for c in caps]
    rows = np.concatenate([[0], np.cumsum(lives)]).tolist()
    k, v = torch.randn(2, rows[-1], kv * hd, device=gpu.device)
    torch.cuda.synchronize()
    zeros = [0] * len(lives)
    gpu.rope_append_q8(None, k, v, rows, ts, caps, zeros, zeros, None, kv, kv, hd)
    gpu.synchronize()
    return ts, caps


# ---- waits that run out ----------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hd,batch,live,cluster", [
    (32, 8, 128, 16, 600, 2), (32, 8, 128, 1, 1999, 8), (4, 1, 128, 1, 7000, 16), (32, 8, 128, 1, 33000, 0), (20, 20, 64, 8, 1500, 2),
    (8, 1, 128, 1, 40000, 8)])
def test_decode_under_a_limit_of_a_cycle_ends_and_leaves_the_next_one_right(gpu, heads, kv, hd, batch, live, cluster):
    """A wait may give up or find its copy there in time; either way the launch ends,
    and its counters are at zero for the next."""
    lives = [live - 3 * b for b in range(batch)]
    assert decode_plan_q8(lives, kv, hd)[1] == cluster
    ts, caps = caches_of(gpu, kv, hd, lives, seed=live)
    q = torch.randn(batch, heads * hd, device=gpu.device)
    torch.cuda.synchronize()
    scratch = DecodeScratch()

    def run():
        return gpu.decode_batched_q8(q, ts, lives, caps, heads, kv, hd, hd ** -0.5, scratch)

    want = run()
    gpu.synchronize()
    for _ in range(5):
        gpu.set_wait_limit_cycles(1)
        try:
            out = run()
            try:
                gpu.synchronize()
                assert torch.equal(out, want)
            except DeviceTimeout:
                pass
        finally:
            gpu.set_wait_limit_cycles(0)
        gpu.synchronize()
        out = run()
        gpu.synchronize()
        assert torch.equal(out, want)


# ---- values that are not finite ------------------------------------------------------------

@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("heads,kv,hd,past,n", [
    (8, 2, 128, 500, 8), (8, 1, 64, 61, 9), (4, 4, 64, 3, 20),           # few rows: the decode kernel
    (32, 8, 128, 90, 200), (27, 3, 128, 500, 150), (36, 4, 64, 0, 140),  # the prefill kernel
    (8, 2, 128, 4000, 250)])                                              # its keys cut into pieces
def test_rows_before_a_value_that_is_not_finite(gpu, heads, kv, hd, past, n, which, bad):
    """It lies in the tail or in a complete block of the first KV head, among the
    prompt's own rows. Rows that may not see it are what they are without it, bit
    for bit, and those that see it are not finite."""
    live = past + n
    cap = (live + 31) // 32 * 32
    torch.manual_seed(live)
    k, v = torch.randn(2, live, kv, hd, device=gpu.device)
    q = torch.randn(n, heads, hd, device=gpu.device)
    torch.cuda.synchronize()

    def run(k, v):
        t = gpu.kv_alloc_q8(kv, hd, cap)
        gpu.rope_append_q8(None, k, v, [0, live], [t], [cap], [0], [0], None, heads, kv, hd)
        out = gpu.flash_attn_q8(q, [0, n], [t], [cap], [past], heads, kv, hd, hd ** -0.5, True)
        gpu.synchronize()
        return out.view(n, heads, hd)

    clean = run(k, v)
    assert clean.isfinite().all()
    spots = [live - 1, live - n // 3] + ([live // 32 * 32 - 7] if live // 32 * 32 - 7 > past else [])
    for spot in spots:
        rows = {"k": k, "v": v}
        x = rows[which] = rows[which].clone()
        x[spot, 0, 5] = bad
        torch.cuda.synchronize()
        out = run(rows["k"], rows["v"])
        group = heads // kv
        assert torch.equal(out[:, group:], clean[:, group:])
        # a complete block is of NaN throughout
        first = spot // 32 * 32 if spot < live // 32 * 32 else spot
        before = max(first - past, 0)
        assert torch.equal(out[:before, :group], clean[:before, :group])
        seen = out[before:, :group]
        if which == "k" and first == spot:
            # (where the infinite key's score is minus infinity, nothing is added)
            counts = torch.isnan(x[spot, 0, 5]) | (q[before:, :group, 5] > 0)
            assert seen[counts].isnan().all()
        elif first != spot:
            assert seen.isnan().all()
        else:
            assert (~seen.isfinite()).any(-1).all()


# ---- caches that are forked --------------------------------------------------------------

@pytest.mark.parametrize("kv,hd", [(8, 128), (3, 64)])
def test_a_cache_evicted_into_several_others(gpu, kv, hd):
    """One call that forks a cache gives what a call for each gives; so does growing it
    behind them. The source is left as it was."""
    live, cap = 900, 928
    (src,), _ = caches_of(gpu, kv, hd, [live], seed=hd, cap=cap)
    q = torch.randn(kv * hd, device=gpu.device)
    torch.cuda.synchronize()
    gpu.decode_batched_q8(q, [src], [live], [cap], kv, kv, hd, hd ** -0.5, DecodeScratch(), weigh=True)
    gpu.synchronize()
    before = src.clone()
    caps, keep = [320, 608, 928, 64], [9, 18, 28, 0]
    alone, forked = ([gpu.kv_alloc_q8(kv, hd, c) for c in caps] for _ in range(2))
    for d, c, k in zip(alone, caps, keep):
        gpu.cache_evict_q8([src], [cap], [d], [c], [live], [k], 0, 0, kv, hd)
    gpu.cache_evict_q8([src] * 4, [cap] * 4, forked, caps, [live] * 4, keep, 0, 0, kv, hd)
    gpu.synchronize()
    assert torch.equal(src, before)
    for a, b in zip(alone, forked):
        assert torch.equal(a, b)


def test_evictions_that_would_race_are_refused(gpu):
    from ttsxabe_b200 import InvalidArgument

    kv, hd, cap, live = 2, 64, 128, 100
    (a, b, c), _ = caches_of(gpu, kv, hd, [live] * 3, seed=1, cap=cap)
    both = gpu.kv_alloc_q8(kv, hd, 2 * cap)
    size = a.numel()
    before = gpu.launch_count()
    for src, dst in [((a, a), (b, b)),          # one destination twice
                     ((a, b), (b, c)),          # a destination that is another's source
                     ((a, a), (a, c)),          # cut in place and read
                     ((a, a), (c, a)),
                     ((both[:size],), (both[16:size + 16],)),
                     ((both[256:size + 256],), (both[:size],))]:
        n = len(src)
        with pytest.raises(InvalidArgument, match="share memory"):
            gpu.cache_evict_q8(list(src), [cap] * n, list(dst), [cap] * n, [live] * n, [2] * n, 0, 0, kv, hd)
    assert gpu.launch_count() == before
    # in place beside a copy of another
    gpu.cache_evict_q8([a, b], [cap] * 2, [a, c], [cap] * 2, [live] * 2, [2] * 2, 0, 0, kv, hd)
    gpu.synchronize()


# ---- what a call launches ------------------------------------------------------------------

def test_decode_counts_every_kernel(gpu):
    """One, another for the weights of complete blocks, another for the zeros of
    sequences without a token."""
    kv, hd = 2, 64
    ts, caps = caches_of(gpu, kv, hd, [70, 5], seed=1)
    q = torch.randn(2, kv * hd, device=gpu.device)
    torch.cuda.synchronize()
    for lives, weigh, want in [([70, 5], False, 1), ([70, 5], True, 2), ([0, 5], False, 2), ([0, 5], True, 2), ([70, 0], True, 3), ([0, 0], True, 1)]:
        before = gpu.launch_count()
        out = gpu.decode_batched_q8(q, ts, lives, caps, kv, kv, hd, 0.1, DecodeScratch(), weigh=weigh).view(2, -1)
        gpu.synchronize()
        assert gpu.launch_count() - before == want, (lives, weigh)
        for b in range(2):
            assert (out[b] == 0).all() == (lives[b] == 0)


# ---- buffers in the wrong place -----------------------------------------------------------

def test_buffers_in_a_caches_memory_are_refused(gpu):
    from ttsxabe_b200 import InvalidArgument

    heads, kv, hd, cap, live = 4, 2, 64, 64, 40
    (t, u), _ = caches_of(gpu, kv, hd, [live] * 2, seed=1, cap=cap)
    f32, f16, i32 = (t.view(x) for x in (torch.float32, torch.float16, torch.int32))
    q, k = gpu.zeros(heads * hd), gpu.zeros(kv * hd)
    f = gpu.rope_inv_freq(10000.0, hd)
    rows = torch.empty(live * kv * hd, dtype=torch.float16, device=gpu.device)
    torch.cuda.synchronize()
    before, held = gpu.launch_count(), t.clone()
    a, w = [t], [cap]

    def append(q=q, k=k, v=k, f=f, q_out=None):
        gpu.rope_append_q8(q, k, v, [0, 1], a, w, [live], [live], f, heads, kv, hd, q_out=q_out)

    wide, narrow = heads * hd, kv * hd
    for call in [lambda: append(q=f32[:wide]), lambda: append(q_out=f32[16:wide + 16]), lambda: append(k=f32[:narrow]),
                 lambda: append(v=f32[-narrow:]), lambda: append(f=f32[:hd // 2]), lambda: append(k=f32[4:narrow + 4]),
                 lambda: gpu.decode_batched_q8(q, a, [live], w, heads, kv, hd, 0.1, DecodeScratch(), out=f32[:wide]),
                 lambda: gpu.decode_batched_q8(q, a, [live], w, heads, kv, hd, 0.1, DecodeScratch(), out=f16[-wide:]),
                 lambda: gpu.decode_batched_q8(f32[:wide], a, [live], w, heads, kv, hd, 0.1, DecodeScratch(), weigh=True),
                 lambda: gpu.flash_attn_q8(q, [0, 1], a, w, [live - 1], heads, kv, hd, 0.1, True, out=f32[:wide]),
                 lambda: gpu.cache_read_q8(a, w, [live], [0], [0, live], kv, hd, k_out=f16[:rows.numel()], v_out=rows),
                 lambda: gpu.cache_read_q8(a, w, [live], [0], [0, live], kv, hd, k_out=rows, v_out=f16[:rows.numel()]),
                 lambda: gpu.cache_evict_q8(a, w, [u], w, [live], [1], 0, 0, kv, hd, index=i32[:8]),
                 lambda: gpu.cache_evict_q8([u], w, a, w, [live], [1], 0, 0, kv, hd, index=i32[:8])]:
        with pytest.raises(InvalidArgument, match="memory of an 8-bit cache"):
            call()
    assert gpu.launch_count() == before
    # a query that is only read may lie anywhere
    gpu.decode_batched_q8(f32[:wide], a, [live], w, heads, kv, hd, 0.1, DecodeScratch())
    gpu.synchronize()
    assert torch.equal(t, held)


def test_rotated_queries_over_the_frequencies_are_refused(gpu):
    from ttsxabe_b200 import InvalidArgument

    heads, kv, hd, cap = 4, 2, 64, 64
    t = gpu.kv_alloc_q8(kv, hd, cap)
    k, both = gpu.zeros(kv * hd), gpu.zeros(heads * hd + hd)
    torch.cuda.synchronize()
    with pytest.raises(InvalidArgument, match="overlaps"):
        gpu.rope_append_q8(gpu.zeros(heads * hd), k, k, [0, 1], [t], [cap], [0], [0], both[heads * hd - 8:heads * hd + hd // 2 - 8],
                           heads, kv, hd, q_out=both[:heads * hd])


# ---- a kernel set up while the one that writes its input still runs ---------------------------

@pytest.mark.parametrize("heads,kv,hd,n,past", [(32, 8, 128, 512, 3000), (32, 8, 128, 64, 200), (20, 20, 64, 300, 0)])
def test_a_prompt_right_behind_the_kernel_that_rotates_its_queries(gpu, heads, kv, hd, n, past):
    """The queries are rotated in place; the same bits as with a pause in between, over
    buffers that hold other queries from one round to the next."""
    live = past + n
    cap = (live + 31) // 32 * 32
    (t,), _ = caches_of(gpu, kv, hd, [past], seed=n, cap=cap) if past else ([gpu.kv_alloc_q8(kv, hd, cap)], None)
    f = gpu.rope_inv_freq(10000.0, hd)
    rows = [torch.randn(n, w * hd, device=gpu.device) for w in (heads, heads, kv, kv)]
    x, held = torch.empty_like(rows[0]), t.clone()
    torch.cuda.synchronize()

    def step(source, pause):
        with torch.cuda.stream(gpu.stream):
            x.copy_(source)
            t.copy_(held)                  # (the rows of its tail gave way to the prompt's)
        gpu.rope_append_q8(x, rows[2], rows[3], [0, n], [t], [cap], [past], [past], f, heads, kv, hd)
        if pause:
            gpu.synchronize()
        out = gpu.flash_attn_q8(x, [0, n], [t], [cap], [past], heads, kv, hd, hd ** -0.5, True)
        gpu.synchronize()
        return out

    want = [step(q, True) for q in rows[:2]]
    for i in range(60):
        assert torch.equal(step(rows[i % 2], False), want[i % 2])


# ---- scales --------------------------------------------------------------------------------

@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5])
@pytest.mark.parametrize("heads,kv,hd,past,n", [(8, 2, 128, 300, 1), (8, 2, 128, 300, 6), (32, 8, 128, 90, 200), (27, 3, 64, 70, 140),
                                                (8, 2, 128, 4000, 250)])
def test_any_scale(gpu, heads, kv, hd, past, n, scale):
    """Of either sign and none, in the decode kernel and in the prefill kernel. A query
    rounded to f16, half a step of 2^-10 a channel, moves a score by no more than d =
    |scale| sum |q k| 2^-11, so the probabilities by a factor within e^(2 d) either way
    and the result by (e^(2 d) - 1) sum p |v|; the rest is what the prefill of such
    queries may be off by."""
    from tests.test_gpu_prefill_items import attention

    live = past + n
    (t,), (cap,) = caches_of(gpu, kv, hd, [live], seed=live)
    q = 0.1 * torch.randn(n, heads, hd, device=gpu.device)
    torch.cuda.synchronize()
    out = gpu.flash_attn_q8(q, [0, n], [t], [cap], [past], heads, kv, hd, scale, True)
    ko, vo = gpu.cache_read_q8([t], [cap], [live], [0], [0, live], kv, hd)
    gpu.synchronize()
    k, v = (x.view(-1, kv, hd).double().transpose(0, 1) for x in (ko, vo))
    want, tol = attention(q.double(), k, v, scale, past)
    most, _ = attention(q.double(), k, v.abs(), scale, past)                 # sum p |v|
    for h in range(heads):
        d = abs(scale) * (q[:, h].double().abs() @ k[h // (heads // kv)].abs().T).max(-1, keepdim=True).values * 2.0 ** -11
        tol[:, h] += torch.expm1(2 * d) * most[:, h]
    assert ((out.view_as(want).double() - want).abs() <= tol).all()
    if n == 1:
        one = gpu.decode_batched_q8(q, [t], [live], [cap], heads, kv, hd, scale, DecodeScratch())
        gpu.synchronize()
        assert ((one.view_as(want).double() - want).abs() <= tol).all()


# ---- the longest caches ----------------------------------------------------------------------

def test_weights_past_the_rows_of_a_grid(gpu):
    """More than 2^28 tokens (34 GB of codes): 2^23 + 1 complete blocks, each of which
    gets its share of an even attention."""
    from ttsxabe_b200 import kv_q8_bytes

    kv, hd = 1, 64
    at = (1 << 28) + 32
    live, cap = at + 8, at + 32
    t = torch.zeros(kv_q8_bytes(kv, hd, cap), dtype=torch.uint8, device=gpu.device)
    k, v = torch.zeros(8, hd, device=gpu.device), torch.ones(8, hd, device=gpu.device)
    q = torch.randn(hd, device=gpu.device)
    torch.cuda.synchronize()
    gpu.rope_append_q8(None, k, v, [0, 8], [t], [cap], [at], [0], None, 1, kv, hd)
    out = gpu.decode_batched_q8(q, [t], [live], [cap], 1, kv, hd, 0.125, DecodeScratch(), weigh=True)
    gpu.synchronize()
    nb = cap // 32
    first = 2 * cap * hd + 2 * ((4 * nb + 127) // 128 * 128)      # behind the codes and two sections of scales
    w = t[first:first + 4 * nb].view(torch.float32)[:at // 32].double()
    # (sums in f32: two roundings for each doubling of the number of terms, and the exponentials')
    off = 64 * 2.0 ** -24
    assert ((w * live / 32 - 1).abs() <= off).all()
    assert ((out.double() * live / 8 - 1).abs() <= off).all()
