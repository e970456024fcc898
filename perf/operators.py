"""The cases by which the operators over an 8-bit KV cache are measured.

A cache is one buffer. Its tokens lie in blocks of 32; a complete block of one KV head is int8 codes with one f32
scale for its keys and one for its values (code = rint(x / scale), scale = max|x| / 127, x rounded to f16 first); the
tokens of the last, incomplete block are f16 rows (the tail). With nb = capacity / 32 the buffer holds, each section
starting at a multiple of 128 bytes:

  key codes [kv][nb][hd / 64][32][64], value codes [kv][nb][hd][32], key scales f32 [kv][nb], value scales f32
  [kv][nb], accumulated attention weights f32 [kv][nb], key tail f16 [kv][32][hd], value tail f16 [kv][32][hd].

Four operators: rows of new tokens rotated and appended ("append"), attention of one query a sequence ("decode"),
causal attention of the appended rows ("prefill"), and eviction of the blocks that attention cares least for ("evict").
"""
import math
import random

import torch

own = False

DEV = "cuda"


# ---- cases ---------------------------------------------------------------------------------------------------

def _case(name, op, heads, kv, hd, batch, lo, hi, new=1, mix=1, keep=0, weigh=False, rotate=True):
    """`lo`..`hi`: tokens already in each sequence's cache, drawn from `mix` (evict and decode: all its tokens);
    `new`: up to how many rows each sequence brings."""
    return {"name": name, "op": op, "heads": heads, "kv": kv, "hd": hd, "batch": batch, "lo": lo, "hi": hi, "new": new,
            "mix": mix, "keep": keep, "weigh": weigh, "rotate": rotate}


def listed():
    return [
        # one decoded token of each of sixteen chats: every projection row rotated and put away, a launch of microseconds
        _case("append step b16", "append", 32, 8, 128, 16, 2048, 4096, new=1, mix=3),
        # ragged prompts that go on from kept prefixes of any length
        _case("append ragged b8", "append", 32, 8, 128, 8, 0, 700, new=512, mix=5),
        # a long prompt into an empty cache
        _case("append prompt 8192", "append", 32, 8, 128, 1, 0, 0, new=8192),
        # one short chat's token: latency
        _case("decode b1 ctx2048", "decode", 32, 8, 128, 1, 2048, 2048),
        # a batch of chats of unequal length, accumulating the weights that eviction goes by
        _case("decode b16 ragged weigh", "decode", 32, 8, 128, 16, 2048, 4096, mix=7, weigh=True),
        # a speech decoder's own or cross attention, a head each to itself, over 30 s of frames
        _case("decode b8 1500 h64", "decode", 20, 20, 64, 8, 1500, 1500),
        # long contexts, the whole memory bandwidth
        _case("decode b8 ctx131072", "decode", 32, 8, 128, 8, 131072, 131072),
        # a batch of ragged prompts over kept prefixes
        _case("prefill ragged b8", "prefill", 32, 8, 128, 8, 0, 512, new=512, mix=11),
        # a long prompt's next piece
        _case("prefill 512 on 16384", "prefill", 32, 8, 128, 1, 16384, 16384, new=512),
        # a long prompt at once
        _case("prefill 8192", "prefill", 32, 8, 128, 1, 0, 0, new=8192),
        # a batch of chats cut back to half of their cache
        _case("evict b16 4096 to 2048", "evict", 32, 8, 128, 16, 3900, 4096, keep=64, mix=13),
        # a long context cut back to an eighth
        _case("evict b4 131072 to 16384", "evict", 32, 8, 128, 4, 131072, 131072, keep=512),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "evict"])
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 4, 128), (12, 4, 128), (8, 1, 128), (16, 16, 128), (20, 20, 64), (16, 4, 64), (8, 1, 64)])
    batch = _log(rng, 1, 32)
    mix = rng.randrange(1, 1 << 30)
    width = kv * hd
    if op == "append":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(8192, 8192 * 40 * 128 // ((heads + kv) * hd * batch))))
        past = _log(rng, 1, 4096) - 1
        return _nameless(op, heads, kv, hd, batch, past // 2, past, new=new, mix=mix, rotate=rng.random() < 0.75)
    if op == "decode":
        most = max(64, 8 * 131072 * 1024 // (batch * width))
        hi = _log(rng, 1, min(131072, most))
        return _nameless(op, heads, kv, hd, batch, max(1, int(hi * rng.choice([0.3, 0.8, 1.0]))), hi, mix=mix, weigh=rng.random() < 0.4)
    if op == "prefill":
        new = _log(rng, 1, 4096)
        room = 8192 * 8192 * 32 // 2 // (batch * heads * new)
        past = _log(rng, 1, max(1, min(32768, room - new))) - 1
        while batch > 1 and batch * heads * new * (past + new) > 8192 * 8192 * 32 // 2:
            batch //= 2
        return _nameless(op, heads, kv, hd, batch, past // 2, past, new=new, mix=mix)
    hi = _log(rng, 64, min(131072, 4 * 131072 * 1024 // (batch * width)))
    keep = max(2, int(hi // 32 * rng.uniform(0.1, 0.95)))
    return _nameless(op, heads, kv, hd, batch, max(1, int(hi * rng.choice([0.5, 0.9, 1.0]))), hi, keep=keep, mix=mix)


def _nameless(*a, **k):
    c = _case("", *a, **k)
    del c["name"]
    return c


# ---- what a case means ---------------------------------------------------------------------------------------

def _lengths(case):
    """Tokens held by each sequence, and the rows that each brings."""
    r = random.Random(case["mix"])
    held = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    new = [r.randint(max(1, case["new"] // 2), case["new"]) if case["batch"] > 1 else case["new"] for _ in held]
    if case["op"] in ("decode", "evict"):
        new = [0] * len(held)
    return held, new


def _blocks(n):
    return (n + 31) // 32


def _sections(kv, hd, cap):
    """(offset, bytes) of each section, and the buffer's bytes."""
    nb = cap // 32
    got, at = {}, 0
    for name, size in (("k", kv * nb * 32 * hd), ("v", kv * nb * 32 * hd), ("ks", kv * nb * 4), ("vs", kv * nb * 4), ("w", kv * nb * 4),
                       ("kt", kv * 32 * hd * 2), ("vt", kv * 32 * hd * 2)):
        got[name] = (at, size)
        at += (size + 127) // 128 * 128
    return got, at


def _views(buf, kv, hd, cap):
    """A batch of caches uint8 [B][bytes] as its sections."""
    b, nb = buf.shape[0], cap // 32
    sec, _ = _sections(kv, hd, cap)

    def part(name, dtype, *shape):
        at, size = sec[name]
        return buf[:, at:at + size].view(dtype).view(b, kv, *shape)

    return {"k": part("k", torch.int8, nb, hd // 64, 32, 64), "v": part("v", torch.int8, nb, hd, 32),
            "ks": part("ks", torch.float32, nb), "vs": part("vs", torch.float32, nb), "w": part("w", torch.float32, nb),
            "kt": part("kt", torch.float16, 32, hd), "vt": part("vt", torch.float16, 32, hd)}


def _quantise(x):
    """Blocks f32 [..., 32, hd] of values that f16 holds: (codes as f32, scale [...])."""
    s = x.abs().amax((-2, -1)) / 127
    c = torch.where(s[..., None, None] > 0, torch.round(x / s[..., None, None]), torch.zeros((), device=x.device))
    return c, s


def _fill(v, x, which):
    """Writes blocks f16-valued x [B, kv, nb, 32, hd] as codes and scales."""
    b, kv, nb, _, hd = x.shape
    c, s = _quantise(x)
    c = c.to(torch.int8)
    if which == "k":
        v["k"].copy_(c.view(b, kv, nb, 32, hd // 64, 64).transpose(3, 4))
    else:
        v["v"].copy_(c.transpose(3, 4))
    v[which + "s"].copy_(s)


def _plan(case):
    """What follows from the lengths alone, as host lists and device index tensors."""
    held, new = _lengths(case)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    live = [h + n for h, n in zip(held, new)]
    cap = max(1, max(_blocks(n) for n in live)) * 32
    t = lambda v, d=torch.int64: torch.tensor(v, dtype=d, device=DEV)  # noqa: E731
    p = {"held": held, "new": new, "cu": cu, "live": live, "cap": cap, "held_t": t(held), "new_t": t(new), "cu_t": t(cu), "live_t": t(live)}
    if case["op"] == "append":
        # the blocks that the new rows touch, and the rows of them
        first = [h // 32 for h in held]
        touched = [n - 32 * f for n, f in zip(live, first)]
        most = max(_blocks(n) for n in touched)
        full = [(b, j, first[b] + j) for b, n in enumerate(touched) for j in range(n // 32)]
        p["blocks"], p["first"] = most, [32 * f for f in first]
        p["full_b"], p["full_j"], p["full_at"] = t([x[0] for x in full]), t([x[1] for x in full]), t([x[2] for x in full])
        p["rest_b"] = t([b for b, n in enumerate(touched) if n % 32])
        p["rest_j"] = t([n // 32 for n in touched if n % 32])
        p["touched"] = touched
        # row i of what is read back is row back_t of sequence back_b's touched blocks
        p["back_cu"] = [sum(touched[:b]) for b in range(len(touched) + 1)]
        seq = torch.repeat_interleave(torch.arange(len(touched)), torch.tensor(touched))
        p["back_b"] = seq.to(DEV)
        p["back_t"] = (torch.arange(len(seq)) - torch.tensor(p["back_cu"])[seq]).to(DEV)
        # row i of the packed rows is at this position
        rows = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
        p["pos_t"] = (torch.arange(len(rows)) - torch.tensor(cu)[rows] + torch.tensor(held)[rows]).to(DEV)
    if case["op"] == "prefill":
        p["row_b"] = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(DEV)
        p["row_t"] = (torch.arange(cu[-1], device=DEV) - p["cu_t"][p["row_b"]])
    if case["op"] == "evict":
        full = [n // 32 for n in live]
        p["kept"] = [min(f, case["keep"]) for f in full]
        p["keep_first"], p["keep_recent"] = _protected(case)
        p["dst_cap"] = max(1, max(_blocks(32 * k + n % 32) for k, n in zip(p["kept"], live))) * 32
        p["full_t"], p["kept_t"] = t(full), t(p["kept"])
    return p


def _protected(case):
    """Blocks at either end that eviction leaves alone: a first one, and an eighth of what is kept."""
    return 1, max(1, case["keep"] // 8)


# ---- inputs --------------------------------------------------------------------------------------------------

def prepare(case, seed):
    heads, kv, hd, batch = case["heads"], case["kv"], case["hd"], case["batch"]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    p = _plan(case)
    cap, nb = p["cap"], p["cap"] // 32
    state = {"case": case, "plan": p}
    buf = torch.zeros(batch, _sections(kv, hd, cap)[1], dtype=torch.uint8, device=DEV)
    v = _views(buf, kv, hd, cap)
    channel = torch.exp(0.5 * normal(kv, 1, 1, hd))   # keys have some strong channels
    for b in range(batch):
        one = {n: x[b:b + 1] for n, x in v.items()}
        _fill(one, (normal(1, kv, nb, 32, hd) * channel).half().float(), "k")
        _fill(one, normal(1, kv, nb, 32, hd).half().float(), "v")
    v["kt"].copy_(normal(batch, kv, 32, hd) * channel[:, 0])
    v["vt"].copy_(normal(batch, kv, 32, hd))
    # weights that a few hundred decoded tokens leave: most blocks little, some much
    v["w"].copy_(torch.exp(1.5 * normal(batch, kv, nb)))
    state["cache"], state["view"] = buf, v
    total = p["cu"][-1]
    if case["op"] == "append":
        state["k"], state["v"] = normal(total * kv * hd), normal(total * kv * hd)
        state["q"] = state["q_out"] = state["inv_freq"] = None   # rows that come rotated already bring no queries
        if case["rotate"]:
            state["q"] = normal(total * heads * hd)
            state["q_out"] = torch.empty_like(state["q"])
            state["inv_freq"] = (10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)).float().to(DEV)
        n = p["back_cu"][-1] * kv * hd
        state["k_back"], state["v_back"] = (torch.empty(n, dtype=torch.float16, device=DEV) for _ in "kv")
    elif case["op"] == "evict":
        state["dst"] = torch.zeros(batch, _sections(kv, hd, p["dst_cap"])[1], dtype=torch.uint8, device=DEV)
        state["dst_view"] = _views(state["dst"], kv, hd, p["dst_cap"])
        state["index"] = torch.full((batch * kv * max(p["kept"] + [1]),), -1, dtype=torch.int32, device=DEV)
    else:
        rows = batch if case["op"] == "decode" else total
        state["q"] = normal(rows * heads * hd)
        state["out"] = torch.empty(rows * heads * hd, dtype=torch.float16, device=DEV)
    if own:
        _handles(state)
    return state


def _handles(state):
    """What a program keeps next to its data: the device handle, the decode scratch and the tables of sequences."""
    from ttsxabe_b200 import DecodeScratch

    g, p, case = _gpu(), state["plan"], state["case"]
    state["gpu"], state["scratch"] = g, DecodeScratch()
    batch = case["batch"]
    state["caches"] = g.ptr_table(list(state["cache"]))
    state["caps"] = g.i32_table([p["cap"]] * batch)
    for name in ("held", "live", "cu"):
        state[name] = g.i32_table(p[name])
    if case["op"] == "append":
        state["back_cu"], state["first"] = g.i32_table(p["back_cu"]), g.i32_table(p["first"])
    if case["op"] == "evict":
        state["dsts"], state["dst_caps"] = g.ptr_table(list(state["dst"])), g.i32_table([p["dst_cap"]] * batch)
        state["keeps"] = g.i32_table([case["keep"]] * batch)


_GPU = []


def _gpu():
    if not _GPU:
        from ttsxabe_b200 import Gpu

        _GPU.append(Gpu.open(0))
    return _GPU[0]


# ---- one pass ------------------------------------------------------------------------------------------------

def run(state):
    return _RUN[state["case"]["op"]](state)


def _append(s):
    c, p = s["case"], s["plan"]
    heads, kv, hd, batch = c["heads"], c["kv"], c["hd"], c["batch"]
    if own:
        g = s["gpu"]
        g.rope_append_q8(s["q"], s["k"], s["v"], s["cu"], s["caches"], s["caps"], s["held"], s["held"], s["inv_freq"], heads, kv, hd,
                         q_out=s["q_out"])
        g.cache_read_q8(s["caches"], s["caps"], s["live"], s["first"], s["back_cu"], kv, hd, k_out=s["k_back"], v_out=s["v_back"])
        out = {"k": s["k_back"], "v": s["v_back"]}
        return {"q": s["q_out"], **out} if c["rotate"] else out
    k, v, out = s["k"].view(-1, kv, hd), s["v"].view(-1, kv, hd), {}
    if c["rotate"]:
        q, angle = s["q"].view(-1, heads, hd), p["pos_t"].double()[:, None, None] * s["inv_freq"].double()
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        q, k = (torch.cat((x[..., :hd // 2] * cos - x[..., hd // 2:] * sin, x[..., hd // 2:] * cos + x[..., :hd // 2] * sin), -1) for x in (q, k))
        out["q"] = q.reshape(-1)
    # the touched blocks: rows of the tail, then the new ones
    at = torch.arange(32 * p["blocks"], device=DEV)[None] - (p["held_t"] % 32)[:, None]
    src = (at.clamp(min=0).minimum(p["new_t"][:, None] - 1) + p["cu_t"][:-1, None]).reshape(-1)
    for name, rows in (("k", k), ("v", v)):
        tail = s["view"][name + "t"]
        x = rows.half()[src].view(batch, -1, kv, hd)
        old = torch.cat((tail, tail.new_zeros(batch, kv, 32 * p["blocks"] - 32, hd)), 2).transpose(1, 2)
        x = torch.where((at < 0)[..., None, None], old, x).float().view(batch, p["blocks"], 32, kv, hd).permute(0, 3, 1, 2, 4)
        codes, scale = _quantise(x)
        full = codes[p["full_b"], :, p["full_j"]]
        laid = full.view(-1, kv, 32, hd // 64, 64).transpose(2, 3) if name == "k" else full.transpose(2, 3)
        s["view"][name][p["full_b"], :, p["full_at"]] = laid.to(torch.int8)
        s["view"][name + "s"][p["full_b"], :, p["full_at"]] = scale[p["full_b"], :, p["full_j"]]
        s["view"]["w"][p["full_b"], :, p["full_at"]] = 0
        rest = (torch.arange(32, device=DEV)[None] < (p["live_t"][p["rest_b"]] % 32)[:, None])[:, None, :, None]
        tail[p["rest_b"]] = torch.where(rest, x[p["rest_b"], :, p["rest_j"]].half(), tail[p["rest_b"]])
        x[p["full_b"], :, p["full_j"]] = full * scale[p["full_b"], :, p["full_j"]][..., None, None]
        x = x.permute(0, 2, 3, 1, 4).reshape(batch, -1, kv, hd)
        out[name] = x[p["back_b"], p["back_t"]].half().reshape(-1)
    return out


def _values(s, name):
    """The cache's keys or values f32 [B, kv, cap, hd], the tail in its place."""
    c, p, v = s["case"], s["plan"], s["view"]
    batch, kv, hd, nb = c["batch"], c["kv"], c["hd"], p["cap"] // 32
    x = v[name].transpose(-2, -3) if name == "k" else v[name].transpose(-1, -2)
    x = x.reshape(batch, kv, nb, 32, hd).float() * v[name + "s"][..., None, None]
    every, at = torch.arange(batch, device=DEV), (p["live_t"] // 32).clamp(max=nb - 1)
    there = (torch.arange(32, device=DEV)[None] < (p["live_t"] - 32 * at)[:, None]) & (p["live_t"] % 32 > 0)[:, None]
    x[every, :, at] = torch.where(there[:, None, :, None], v[name + "t"].float(), x[every, :, at])
    return x.reshape(batch, kv, nb * 32, hd)


def _decode(s):
    c, p = s["case"], s["plan"]
    heads, kv, hd, batch = c["heads"], c["kv"], c["hd"], c["batch"]
    if own:
        s["gpu"].decode_batched_q8(s["q"], s["caches"], s["live"], s["caps"], heads, kv, hd, hd ** -0.5, s["scratch"], out=s["out"],
                                   weigh=c["weigh"])
        return (s["out"], s["view"]["w"]) if c["weigh"] else s["out"]
    q = s["q"].view(batch, kv, heads // kv, hd)
    score = (q @ _values(s, "k").transpose(2, 3)) * hd ** -0.5
    score = score.masked_fill((torch.arange(p["cap"], device=DEV)[None] >= p["live_t"][:, None])[:, None, None], -math.inf)
    prob = torch.exp(score - score.amax(-1, keepdim=True))
    prob = prob / prob.sum(-1, keepdim=True)
    out = (prob @ _values(s, "v")).half().reshape(-1)
    if not c["weigh"]:
        return out
    share = prob.sum(2).view(batch, kv, -1, 32).sum(-1)
    full = torch.arange(p["cap"] // 32, device=DEV)[None] < (p["live_t"] // 32)[:, None]
    s["view"]["w"].add_(torch.where(full[:, None], share, torch.zeros((), device=DEV)))
    return out, s["view"]["w"]


def _prefill(s):
    c, p = s["case"], s["plan"]
    heads, kv, hd, batch = c["heads"], c["kv"], c["hd"], c["batch"]
    if own:
        s["gpu"].flash_attn_q8(s["q"], s["cu"], s["caches"], s["caps"], s["held"], heads, kv, hd, hd ** -0.5, True, out=s["out"])
        return s["out"]
    most = max(p["new"])
    q = s["q"].new_zeros(batch, most, heads * hd)
    q[p["row_b"], p["row_t"]] = s["q"].view(-1, heads * hd)
    q = q.view(batch, most, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, hd)
    score = ((q @ _values(s, "k").transpose(2, 3)) * hd ** -0.5).view(batch, kv, heads // kv, most, -1)
    last = p["held_t"][:, None] + torch.arange(most, device=DEV)
    score.masked_fill_((torch.arange(p["cap"], device=DEV) > last[..., None])[:, None, None], -math.inf)
    prob = torch.exp_(score.sub_(score.amax(-1, keepdim=True)))
    out = (prob.view(batch, kv, -1, p["cap"]) @ _values(s, "v")).view(batch, kv, heads // kv, most, hd)
    out = (out / prob.sum(-1, keepdim=True)).permute(0, 3, 1, 2, 4).reshape(batch, most, heads * hd)
    return out[p["row_b"], p["row_t"]].half().reshape(-1)


def _evict(s):
    c, p = s["case"], s["plan"]
    kv, hd, batch = c["kv"], c["hd"], c["batch"]
    if own:
        s["gpu"].cache_evict_q8(s["caches"], s["caps"], s["dsts"], s["dst_caps"], s["live"], s["keeps"], p["keep_first"], p["keep_recent"], kv, hd,
                                index=s["index"])
        return _evicted(s)
    v, d = s["view"], s["dst_view"]
    nb, out_nb = p["cap"] // 32, p["dst_cap"] // 32
    at = torch.arange(nb, device=DEV)
    full = p["full_t"][:, None]
    safe = ((at < p["keep_first"]) | (at >= full - p["keep_recent"]))[:, None]
    weight = torch.where(v["w"] > 0, v["w"], torch.zeros((), device=DEV))
    weight = torch.where(safe, math.inf, weight).masked_fill((at >= full)[:, None], -1.0)
    order = torch.argsort(weight, dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    gone = rank >= p["kept_t"][:, None, None]
    most = max(p["kept"] + [1])
    source = torch.argsort(gone.to(torch.int8), dim=-1, stable=True)[..., :most]
    there = (torch.arange(most, device=DEV) < p["kept_t"][:, None])[:, None].expand_as(source)
    s["index"].copy_(torch.where(there, source, -1).reshape(-1))
    for name in ("k", "v", "ks", "vs", "w"):
        x = v[name]
        pick = source.view(*source.shape, *[1] * (x.dim() - 3)).expand(*source.shape, *x.shape[3:])
        mask = there.view(*source.shape, *[1] * (x.dim() - 3))
        to = d[name][:, :, :min(most, out_nb)]
        to.copy_(torch.where(mask, torch.gather(x, 2, pick), to) if out_nb >= most else to)
    rows = (torch.arange(32, device=DEV)[None] < (p["live_t"] % 32)[:, None])[:, None, :, None]
    for name in ("kt", "vt"):
        d[name].copy_(torch.where(rows, v[name], d[name]))
    return _evicted(s)


def _evicted(s):
    # codes move and are never computed: they come back as they are held, next to their scales
    d = s["dst_view"]
    return {"index": s["index"], **{n: d[n] for n in ("k", "v", "ks", "vs", "w", "kt", "vt")}}


_RUN = {"append": _append, "decode": _decode, "prefill": _prefill, "evict": _evict}


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    heads, kv, hd, op = case["heads"], case["kv"], case["hd"], case["op"]
    held, new = _lengths(case)
    live = [h + n for h, n in zip(held, new)]
    total = sum(new)
    cache = sum(2 * kv * ((n // 32) * (32 * hd + 4) + (n % 32) * hd * 2) for n in live)
    if op == "append":
        back = sum(n - h // 32 * 32 for n, h in zip(live, held))
        done = sum(n // 32 - h // 32 for n, h in zip(live, held))
        old = sum(h % 32 for h in held)
        turned = heads if case["rotate"] else 0
        rows = total * (2 * turned + 2 * kv) * hd * 4 + old * 2 * kv * hd * 2
        return {"bytes": rows + done * kv * (2 * (32 * hd + 4) + 4) + sum(n % 32 for n in live) * 2 * kv * hd * 2 + back * 2 * kv * hd * 2,
                "flops": total * 3 * (turned + kv) * hd}
    if op == "decode":
        extra = sum(n // 32 for n in live) * kv * 8 if case["weigh"] else 0
        return {"bytes": cache + len(live) * heads * hd * 6 + extra, "flops": 4 * heads * hd * sum(live)}
    if op == "prefill":
        pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
        return {"bytes": cache + total * heads * hd * 6, "flops": 4 * heads * hd * pairs}
    kept = [min(n // 32, case["keep"]) for n in live]
    move = sum(kv * (k * (2 * (32 * hd + 4) + 4) + (n % 32) * 2 * hd * 2) for k, n in zip(kept, live))
    return {"bytes": 2 * move + sum(n // 32 for n in live) * kv * 4 + sum(kept) * kv * 4, "flops": sum(n // 32 for n in live) * kv}


# ---- the definition, in 64 bits, sequence by sequence --------------------------------------------------------

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"append": _exact_append, "decode": _exact_decode, "prefill": _exact_prefill, "evict": _exact_evict}[case["op"]](s)


def _held64(s, b, name, tokens):
    """The first `tokens` keys or values of sequence b, f64 [kv, tokens, hd]."""
    c, v = s["case"], s["view"]
    kv, hd, full = c["kv"], c["hd"], tokens // 32
    code = v[name][b, :, :full].double()
    if name == "k":
        code = torch.cat([code[:, :, j] for j in range(hd // 64)], -1)
    else:
        code = code.swapaxes(-1, -2)
    x = (code * v[name + "s"][b, :, :full, None, None].double()).reshape(kv, 32 * full, hd)
    return torch.cat((x, v[name + "t"][b, :, :tokens % 32].double()), 1)


def _exact_append(s):
    c, p = s["case"], s["plan"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    qs, ks, vs = [], [], []
    for b, (past, n) in enumerate(zip(p["held"], p["new"])):
        at = slice(p["cu"][b], p["cu"][b + 1])
        k, v = (s[m].view(-1, kv, hd)[at].double() for m in "kv")
        if c["rotate"]:
            q = s["q"].view(-1, heads, hd)[at].double()
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                               torch.arange(past, past + n, device=DEV).double()[:, None] * s["inv_freq"].double())[:, None]
            q, k = (torch.view_as_real(torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn).movedim(-1, -2).flatten(-2) for x in (q, k))
            qs.append(q.reshape(-1))
        for rows, name, to in ((k, "k", ks), (v, "v", vs)):
            # the cache holds what f16 holds of the f32 row
            x = torch.cat((s["view"][name + "t"][b, :, :past % 32].double().swapaxes(0, 1), rows.float().half().double()))
            full = len(x) // 32
            y = x[:32 * full].view(full, 32, kv, hd)
            step = y.abs().amax((1, 3), keepdim=True) / 127
            y = torch.where(step > 0, torch.round(y / step) * step, 0.0).view(-1, kv, hd)
            to.append(torch.cat((y, x[32 * full:])).reshape(-1))
    out = {"k": torch.cat(ks), "v": torch.cat(vs)}
    return {"q": torch.cat(qs), **out} if c["rotate"] else out


def _exact_decode(s):
    c, p = s["case"], s["plan"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    outs, weights = [], s["view"]["w"].double()
    for b, n in enumerate(p["live"]):
        q = s["q"].view(-1, kv, heads // kv, hd)[b].double()
        z = torch.einsum("kgd,ktd->kgt", q, _held64(s, b, "k", n)) / math.sqrt(hd)
        w = torch.softmax(z, -1)
        outs.append(torch.einsum("kgt,ktd->kgd", w, _held64(s, b, "v", n)).reshape(-1))
        weights[b, :, :n // 32] += w[..., :n // 32 * 32].sum(1).view(kv, -1, 32).sum(-1)
    return (torch.cat(outs), weights) if c["weigh"] else torch.cat(outs)


def _exact_prefill(s):
    c, p = s["case"], s["plan"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    outs = []
    for b, (past, n) in enumerate(zip(p["held"], p["new"])):
        q = s["q"].view(-1, kv, heads // kv, hd)[p["cu"][b]:p["cu"][b + 1]].double()
        k, v = _held64(s, b, "k", past + n), _held64(s, b, "v", past + n)
        out = torch.empty_like(q)
        for i in range(0, n, 1024):
            z = torch.einsum("ikgd,ktd->kgit", q[i:i + 1024], k) / math.sqrt(hd)
            row = torch.arange(i, min(n, i + 1024), device=DEV)
            z[..., torch.arange(past + n, device=DEV)[None] > past + row[:, None]] = -math.inf
            out[i:i + 1024] = torch.einsum("kgit,ktd->ikgd", torch.softmax(z, -1), v)
        outs.append(out.reshape(-1))
    return torch.cat(outs)


def _exact_evict(s):
    c, p = s["case"], s["plan"]
    d, v = {n: x.clone() for n, x in s["dst_view"].items()}, s["view"]
    index = s["index"].view(c["batch"], c["kv"], -1).clone()
    for b, n in enumerate(p["live"]):
        full, keep = n // 32, p["kept"][b]
        first, recent = p["keep_first"], p["keep_recent"]
        for h in range(c["kv"]):
            if full <= keep:
                chosen = list(range(full))
            else:
                w = [x if x > 0 else 0.0 for x in v["w"][b, h].tolist()]
                middle = sorted(range(first, full - recent), key=lambda i: (-w[i], i))[:keep - first - recent]
                chosen = list(range(first)) + sorted(middle) + list(range(full - recent, full))
            index[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32, device=DEV)
            for m in ("k", "v", "ks", "vs", "w"):
                d[m][b, h, :len(chosen)] = v[m][b, h, chosen]
        for m in ("kt", "vt"):
            d[m][b, :, :n % 32] = v[m][b, :, :n % 32]
    return {"index": index.reshape(-1), "k": d["k"], "v": d["v"], **{m: d[m].double() for m in ("ks", "vs", "w", "kt", "vt")}}
