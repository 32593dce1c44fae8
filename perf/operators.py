"""Rotary positions, appending to a paged KV cache, and attention over it: cases, inputs and plain forms.

The three operators are what a host with a paged cache runs per layer: the
rotation of q and k by position (whole or part of the head, NeoX or interleaved
pairs), the append of a ragged batch's new keys and values to their pages with
QK-RMSNorm and the rotation on the way, and the causal attention of the new
tokens over the pages.  Cache pools are [n_pages][n_kv_heads][page_size][head_dim]
(one layer here); a page table row lists a sequence's pages in order.
"""
import math
import random

import torch

own = False

# (q heads, KV heads, head_dim) of the models whose shapes the repository's benchmark and tests use
SHAPES = [(32, 4, 64), (14, 2, 64), (28, 4, 128), (32, 8, 128), (40, 8, 128)]
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BASE = 1e6
EPS = 1e-6


def listed():
    return [
        # one decoded token's q and k, the smallest call: its latency is what counts
        dict(name="rope_token", op="rope", tokens=1, hq=14, hkv=2, hd=64, rot=64, mode="neox", dtype="f16",
             fused=False, inverse=False, rows=4096),
        # a long prompt's q and k taken out of a fused q|k|v projection, far positions
        dict(name="rope_prompt", op="rope", tokens=8192, hq=32, hkv=8, hd=128, rot=128, mode="neox", dtype="bf16",
             fused=True, inverse=False, rows=131072),
        # gradients going back through a rotation of half of each head, an odd number of tokens
        dict(name="rope_partial_grad", op="rope", tokens=2047, hq=28, hkv=4, hd=128, rot=64, mode="interleaved",
             dtype="f32", fused=False, inverse=True, rows=8192),
        # one new token of each of 64 sequences, straight from fp32 projections
        dict(name="append_tokens", op="append", ones=64, chunks=0, new_lo=1, new_hi=1, past_lo=1024, past_hi=2048,
             hq=28, hkv=4, hd=128, rot=128, mode="neox", norm=False, dtype="f32", cache="f16", page=16, lens=1),
        # a whole prompt with QK-norm
        dict(name="append_prompt", op="append", ones=0, chunks=1, new_lo=2048, new_hi=2048, past_lo=0, past_hi=0,
             hq=32, hkv=8, hd=128, rot=128, mode="neox", norm=True, dtype="f16", cache="f16", page=64, lens=2),
        # ragged chunks beside single tokens, half of the head rotated, bf16 throughout
        dict(name="append_ragged", op="append", ones=13, chunks=7, new_lo=33, new_hi=701, past_lo=0, past_hi=1500,
             hq=32, hkv=4, hd=64, rot=32, mode="interleaved", norm=False, dtype="bf16", cache="bf16", page=32, lens=3),
        # one sequence, one token, short context: latency
        dict(name="attn_token", op="attn", ones=1, chunks=0, new_lo=1, new_hi=1, past_lo=511, past_hi=511,
             hq=32, hkv=4, hd=64, cache="f16", page=16, lens=4),
        # the serving batch: 64 ragged sequences, one token each
        dict(name="attn_batch", op="attn", ones=64, chunks=0, new_lo=1, new_hi=1, past_lo=1024, past_hi=8192,
             hq=28, hkv=4, hd=128, cache="f16", page=16, lens=5),
        # one sequence over a long context, and a few drafted tokens to check
        dict(name="attn_long_draft", op="attn", ones=0, chunks=1, new_lo=3, new_hi=3, past_lo=131069, past_hi=131069,
             hq=40, hkv=8, hd=128, cache="f16", page=64, lens=6),
        # a whole prompt
        dict(name="attn_prompt", op="attn", ones=0, chunks=1, new_lo=2048, new_hi=2048, past_lo=0, past_hi=0,
             hq=32, hkv=8, hd=128, cache="f16", page=64, lens=7),
        # the largest: a chunk of a long prompt whose beginning is cached
        dict(name="attn_chunk", op="attn", ones=0, chunks=2, new_lo=1024, new_hi=1024, past_lo=16384, past_hi=30000,
             hq=32, hkv=8, hd=128, cache="bf16", page=128, lens=8),
        # prompts' chunks and decoding sequences in one step, odd lengths
        dict(name="attn_mixed", op="attn", ones=24, chunks=3, new_lo=100, new_hi=513, past_lo=17, past_hi=4096,
             hq=28, hkv=4, hd=128, cache="bf16", page=32, lens=9),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    hq, hkv, hd = rng.choice(SHAPES)
    mode = rng.choice(["neox", "interleaved"])
    op = rng.choice(["rope", "append", "attn", "attn"])
    if op == "rope":
        rot = rng.choice([hd, hd // 2, hd // 4])
        return dict(op="rope", tokens=_log(rng, 1, 8191), hq=hq, hkv=hkv, hd=hd, rot=rot, mode=mode,
                    dtype=rng.choice(["f16", "bf16", "f32"]), fused=rng.random() < 0.5, inverse=rng.random() < 0.3,
                    rows=_log(rng, 512, 131072))
    cache = rng.choice(["f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1 << 30)
    if op == "append":
        rot = rng.choice([hd, hd, hd // 2])
        ones, chunks = rng.choice([(_log(rng, 1, 128), 0), (rng.randrange(0, 17), rng.randrange(1, 9))])
        hi = _log(rng, 2, 512) if chunks else 1
        return dict(op="append", ones=ones, chunks=chunks, new_lo=max(1, hi // 3), new_hi=hi, past_lo=0,
                    past_hi=_log(rng, 1, 1500), hq=hq, hkv=hkv, hd=hd, rot=rot, mode=mode, norm=rng.random() < 0.5,
                    dtype=rng.choice([cache, "f32"]), cache=cache, page=page, lens=lens)
    kind = rng.choice(["ones", "draft", "chunk", "mixed"])
    if kind == "ones":
        ones, chunks, hi, past = _log(rng, 1, 64), 0, 1, _log(rng, 16, 8192)
    elif kind == "draft":
        ones, chunks, hi, past = rng.randrange(0, 5), _log(rng, 1, 16), rng.randrange(2, 9), _log(rng, 16, 16384)
    elif kind == "chunk":
        ones, chunks, hi, past = 0, rng.randrange(1, 4), _log(rng, 16, 1024), _log(rng, 1, 8192)
    else:
        ones, chunks, hi, past = rng.randrange(1, 25), rng.randrange(1, 4), _log(rng, 16, 512), _log(rng, 16, 4096)
    return dict(op="attn", ones=ones, chunks=chunks, new_lo=max(1, hi // 2), new_hi=hi, past_lo=past // 3,
                past_hi=past, hq=hq, hkv=hkv, hd=hd, cache=cache, page=page, lens=lens)


def _lengths(case):
    """(new tokens, cached rows) of every sequence, the chunks spread among the single tokens."""
    rng = random.Random(case["lens"])
    new = [1] * case["ones"] + [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["chunks"])]
    rng.shuffle(new)
    return new, [rng.randint(case["past_lo"], case["past_hi"]) for _ in new]


def _table(rows, rot, device):
    """cos and sin of every position, angles in 64 bits, held in 32: what a program builds once."""
    freq = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _paged(case, gen, dev):
    """The pools of one layer with their pages dealt at random, and the batch's lengths."""
    new, past = _lengths(case)
    page, hkv, hd = case["page"], case["hkv"], case["hd"]
    total = [n + p for n, p in zip(new, past)]
    need = [-(-t // page) for t in total]
    width = max(need)
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=gen, device=dev)[:sum(need)].to(torch.int32).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [0] * (width - n))
        at += n
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    i32 = dict(dtype=torch.int32, device=dev)
    dt = DTYPES[case["cache"]]
    pools = [(0.5 * torch.randn((1, n_pages, hkv, page, hd), generator=gen, device=dev)).to(dt) for _ in range(2)]
    return dict(k_pool=pools[0], v_pool=pools[1], pages=torch.tensor(rows, **i32), start=torch.tensor(start, **i32),
                kv_len=torch.tensor(total, **i32), tokens=start[-1], max_new=max(new), max_len=max(total))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    s = dict(case=case)
    if case["op"] == "rope":
        n, dt = case["tokens"], DTYPES[case["dtype"]]
        s["cos"], s["sin"] = _table(case["rows"], case["rot"], dev)
        s["pos"] = torch.randint(0, case["rows"], (n,), generator=gen, device=dev, dtype=torch.int32)
        if case["fused"]:  # rows of one projection's output: q heads, k heads, v heads
            qkv = torch.randn((n, hq + 2 * hkv, hd), generator=gen, device=dev).to(dt)
            s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        else:
            s["q"] = torch.randn((n, hq, hd), generator=gen, device=dev).to(dt)
            s["k"] = torch.randn((n, hkv, hd), generator=gen, device=dev).to(dt)
        s["q_out"] = torch.empty((n, hq, hd), dtype=dt, device=dev)
        s["k_out"] = torch.empty((n, hkv, hd), dtype=dt, device=dev)
    else:
        s.update(_paged(case, gen, dev))
        n = s["tokens"]
        if case["op"] == "append":
            dt = DTYPES[case["dtype"]]
            s["q"] = torch.randn((n, hq, hd), generator=gen, device=dev).to(dt)
            s["k"] = torch.randn((n, hkv, hd), generator=gen, device=dev).to(dt)
            s["v"] = torch.randn((n, hkv, hd), generator=gen, device=dev).to(dt)
            s["cos"], s["sin"] = _table(s["max_len"], case["rot"], dev)
            s["q_norm"] = s["k_norm"] = None
            if case["norm"]:
                s["q_norm"] = 1 + 0.1 * torch.randn(hd, generator=gen, device=dev)
                s["k_norm"] = 1 + 0.1 * torch.randn(hd, generator=gen, device=dev)
            s["q_out"] = torch.empty((n, hq, hd), dtype=DTYPES[case["cache"]], device=dev)
        else:
            s["q"] = torch.randn((n, hq, hd), generator=gen, device=dev).to(DTYPES[case["cache"]])
            s["out"] = torch.empty((n, hq, hd), dtype=DTYPES[case["cache"]], device=dev)
    if own:  # the handles that a program keeps: the cache over its pools, the batch of a step, a status word
        from picolm_qwen_b200 import abi, runtime
        mode = abi.ROPE_NEOX if case.get("mode", "neox") == "neox" else abi.ROPE_INTERLEAVED
        s["abi_mode"] = mode
        if case["op"] == "rope":
            s["status"] = runtime.status_workspace(dev)
        else:
            cfg = abi.Config.make(1, hq, hkv, hd, s["max_len"], BASE, mode, EPS)
            s["cache"] = runtime.PagedCache(cfg, case["page"], k_pool=s["k_pool"], v_pool=s["v_pool"])
            s["batch"] = s["cache"].batch(s["pages"], s["start"], s["kv_len"], s["tokens"], s["max_new"], s["max_len"])
    return s


# -- plain forms -------------------------------------------------------------


def _rotate(x, cos, sin, rot, mode):
    """x [n, heads, hd] in fp32; cos, sin [n, rot/2]."""
    c, s = cos[:, None], sin[:, None]
    r = x[..., :rot]
    x0, x1 = (r[..., :rot // 2], r[..., rot // 2:]) if mode == "neox" else (r[..., 0::2], r[..., 1::2])
    y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
    y = torch.cat([y0, y1], -1) if mode == "neox" else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _rope(s):
    case = s["case"]
    at = s["pos"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    if case["inverse"]:
        sin = -sin
    return {n: _rotate(s[n].float(), cos, sin, case["rot"], case["mode"]).to(s[n].dtype) for n in ("q", "k")}


def _owner(s):
    """The sequence of every token, and the token's place among its sequence's new ones."""
    t = torch.arange(s["tokens"], device=s["start"].device)
    b = torch.searchsorted(s["start"][1:].long(), t, right=True)
    return b, t - s["start"].long()[b]


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _append(s):
    case, page = s["case"], s["case"]["page"]
    b, i = _owner(s)
    n_new = s["start"].long().diff()
    pos = s["kv_len"].long()[b] - n_new[b] + i
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(_normed(s["q"], s["q_norm"]), cos, sin, case["rot"], case["mode"])
    k = _rotate(_normed(s["k"], s["k_norm"]), cos, sin, case["rot"], case["mode"])
    at = s["pages"].long()[b, pos // page]
    s["k_pool"][0].permute(0, 2, 1, 3)[at, pos % page] = k.to(s["k_pool"].dtype)
    s["v_pool"][0].permute(0, 2, 1, 3)[at, pos % page] = s["v"].float().to(s["v_pool"].dtype)
    return {"q": q.to(s["k_pool"].dtype), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _attn(s):
    case = s["case"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    g, page, most = hq // hkv, case["page"], s["max_new"]
    pages = s["pages"].long()
    batch, rows = pages.shape[0], pages.shape[1] * page
    k, v = (p[0][pages].permute(0, 2, 1, 3, 4).reshape(batch, hkv, rows, hd).float() for p in (s["k_pool"], s["v_pool"]))
    start, n_new = s["start"].long(), s["start"].long().diff()
    i = torch.arange(most, device=pages.device)
    at = (start[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][at].float().view(batch, most, hkv, g, hd).permute(0, 2, 1, 3, 4).reshape(batch, hkv, most * g, hd)
    score = (q @ k.transpose(-1, -2)).mul_(hd ** -0.5).view(batch, hkv, most, g, rows)
    pos = s["kv_len"].long()[:, None] - n_new[:, None] + i
    hidden = torch.arange(rows, device=pages.device) > pos[..., None]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = p.view(batch, hkv, most * g, rows) @ v
    o = o.view(batch, hkv, most, g, hd) / p.sum(-1, keepdim=True)
    b, i = _owner(s)
    return o.permute(0, 2, 1, 3, 4)[b, i].reshape(s["tokens"], hq, hd).to(s["q"].dtype)


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"rope": _rope, "append": _append, "attn": _attn}[case["op"]](s)
    if case["op"] == "rope":
        from picolm_qwen_b200 import runtime
        runtime.rope(s["q"], s["k"], s["pos"], s["cos"], s["sin"], s["q_out"], s["k_out"], s["status"],
                     rope_mode=s["abi_mode"], inverse=case["inverse"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if case["op"] == "append":
        s["cache"].append(0, s["batch"], s["q"], s["k"], s["v"], s["cos"], s["sin"], s["q_out"], s["q_norm"],
                          s["k_norm"])
        return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    s["cache"].attend(0, s["batch"], s["q"], s["out"])
    return s["out"]


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if case["op"] == "rope":
        n, e = case["tokens"], 4 if case["dtype"] == "f32" else 2
        moved = n * (hq + hkv) * hd * e * 2 + min(n, case["rows"]) * case["rot"] * 4 + n * 4
        return {"bytes": moved, "flops": 3 * n * (hq + hkv) * case["rot"]}
    new, past = _lengths(case)
    n = sum(new)
    ids = 4 * sum(-(-(a + b) // case["page"]) for a, b in zip(new, past))
    if case["op"] == "append":
        e = 4 if case["dtype"] == "f32" else 2
        heads = hq + 2 * hkv
        moved = n * heads * hd * (e + 2) + n * case["rot"] * 4 + 4 * n
        return {"bytes": moved, "flops": n * (hq + hkv) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))}
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, past))
    moved = sum(a + b for a, b in zip(new, past)) * hkv * hd * 2 * 2 + n * hq * hd * 2 * 2 + ids
    return {"bytes": moved, "flops": 4 * hq * hd * seen}


# -- the definitions in 64 bits -------------------------------------------------


def _turn64(x, pos, cos, sin, rot, mode, sign):
    """Each pair as a complex number times e^(i sign theta) of its position, from the table's own entries."""
    half = rot // 2
    turn = torch.complex(cos.double()[pos], sign * sin.double()[pos])[:, None, :]
    y = x.double().clone()
    first = torch.arange(half, device=x.device) * (1 if mode == "neox" else 2)
    second = first + (half if mode == "neox" else 1)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        sign = -1.0 if case["inverse"] else 1.0
        return {n: _turn64(s[n], s["pos"].long(), s["cos"], s["sin"], case["rot"], case["mode"], sign) for n in ("q", "k")}
    start, total, page = s["start"].tolist(), s["kv_len"].tolist(), case["page"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(t - (e - b), t) for b, e, t in zip(start, start[1:], total)]).to(s["q"].device)
        seq = torch.cat([torch.full((e - b,), j) for j, (b, e) in enumerate(zip(start, start[1:]))]).to(s["q"].device)
        new = {}
        for n in ("q", "k"):
            x = s[n].double()
            if case["norm"]:
                x = x / (x.pow(2).sum(-1, keepdim=True) / case["hd"] + EPS).sqrt() * s[n + "_norm"].double()
            new[n] = _turn64(x, pos, s["cos"], s["sin"], case["rot"], case["mode"], 1.0)
        k, v = s["k_pool"].double(), s["v_pool"].double()
        at, row = s["pages"].long()[seq, pos // page], pos % page
        for h in range(case["hkv"]):
            k[0, at, h, row] = new["k"][:, h]
            v[0, at, h, row] = s["v"][:, h].double()
        return {"q": new["q"], "k_pool": k, "v_pool": v}
    g = case["hq"] // case["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for j, (b, e, t) in enumerate(zip(start, start[1:], total)):
        ids = s["pages"][j, :-(-t // page)].long()
        cols = torch.arange(t, device=out.device)
        rows = torch.arange(t - (e - b), t, device=out.device)
        for h in range(case["hkv"]):
            k, v = (p[0, ids, h].reshape(-1, case["hd"])[:t].double() for p in (s["k_pool"], s["v_pool"]))
            for a in range(g):
                w = s["q"][b:e, h * g + a].double() @ k.T / math.sqrt(case["hd"])
                w = torch.where(cols[None] <= rows[:, None], w, torch.full_like(w, -math.inf))
                out[b:e, h * g + a] = torch.softmax(w, -1) @ v
    return out
