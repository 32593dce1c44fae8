"""Rotary positions, the paged cache's append and its attention against their formulas in 64 bits.

Tolerances (pagedref.py derives the fp32 parts): a result rounded to 16 bits is off by half a step more,
finfo.eps / 2 of its value, or half the smallest subnormal.
"""
import numpy as np
import pytest
import torch

import pagedref as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -130, torch.float32: 2.0 ** -130}


@pytest.fixture(scope="module")
def rt():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from picolm_qwen_b200 import abi, runtime
    assert abi.lib().picoattn_device_check() == 0
    return runtime


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def f64(t):
    return t.detach().double().cpu().numpy()


def check(got, want, err, dtype, what):
    """|got - want| <= err plus one rounding to dtype (of a value up to err off)."""
    got = f64(got)
    tol = err + HALF[dtype] * (np.abs(want) + err) + TINY[dtype]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol):.3g} of "
                           f"the tolerance at {np.unravel_index(bad.argmax(), bad.shape)}")


def table(rows, rot, seed=0):
    ang = np.arange(rows)[:, None] * 1e4 ** (-np.arange(0, rot, 2) / rot) + seed
    return (torch.from_numpy(np.cos(ang).astype(np.float32)).cuda(),
            torch.from_numpy(np.sin(ang).astype(np.float32)).cuda())


# -- rope ------------------------------------------------------------------------


@pytest.mark.parametrize("n,hq,hkv,hd,rot", [
    (1, 14, 2, 64, 64), (3, 1, 1, 2, 2), (37, 5, 1, 128, 64), (129, 32, 8, 128, 128), (20, 3, 2, 80, 80),
    (11, 4, 4, 96, 34), (9, 2, 1, 256, 16), (5, 1, 3, 1024, 1000), (300, 28, 4, 64, 16),
])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("neox", [True, False])
def test_rope(rt, n, hq, hkv, hd, rot, dtype, neox):
    g, dt = gen(n + rot), DT[dtype]
    q = torch.randn((n, hq, hd), generator=g, device="cuda").to(dt)
    k = torch.randn((n, hkv, hd), generator=g, device="cuda").to(dt)
    cos, sin = table(500, rot)
    pos = torch.randint(0, 500, (n,), generator=g, device="cuda", dtype=torch.int32)
    pos[0], pos[-1] = 499, 0
    c, s = f64(cos)[pos.cpu().numpy()], f64(sin)[pos.cpu().numpy()]
    ws = rt.status_workspace()
    for inverse in (False, True):
        qo, ko = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
        rt.rope(q, k, pos, cos, sin, qo, ko, ws, rope_mode=0 if neox else 1, inverse=inverse)
        for x, y, name in ((q, qo, "q"), (k, ko, "k")):
            want, err = ref.rotate(f64(x), c, s, rot, neox, -1.0 if inverse else 1.0)
            check(y, want, err, dt, f"{name} inverse={inverse}")
            assert torch.equal(y[..., rot:], x[..., rot:])
        a, b = q.clone(), k.clone()  # in place: the same bits
        rt.rope(a, b, pos, cos, sin, a, b, ws, rope_mode=0 if neox else 1, inverse=inverse)
        assert torch.equal(a, qo) and torch.equal(b, ko)
        o = torch.full_like(q, float("nan"))
        rt.rope(q, None, pos, cos, sin, o, None, ws, rope_mode=0 if neox else 1, inverse=inverse)
        assert torch.equal(o, qo)
    assert rt.workspace_status(ws) == 0


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("off,pad", [(0, 0), (1, 0), (0, 3), (8, 64)])
def test_rope_strides_and_alignment(rt, dtype, off, pad):
    """Heads taken out of a fused projection's rows, at any element offset, in place; the rest untouched."""
    n, hq, hkv, hd, dt = 33, 6, 2, 64, DT[dtype]
    width = (hq + 2 * hkv) * hd + pad
    buf = torch.randn(n * width + off, generator=gen(5), device="cuda").to(dt)
    before = buf.clone()
    rows = buf[off:].view(n, width)
    q, k = rows[:, :hq * hd].view(n, hq, hd), rows[:, hq * hd:(hq + hkv) * hd].view(n, hkv, hd)
    want_q, want_k = q.contiguous(), k.contiguous()
    cos, sin = table(64, hd)
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    ws = rt.status_workspace()
    rt.rope(want_q, want_k, pos, cos, sin, want_q, want_k, ws)
    rt.rope(q, k, pos, cos, sin, q, k, ws)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    rest = (hq + hkv) * hd
    assert torch.equal(rows[:, rest:], before[off:].view(n, width)[:, rest:]) and torch.equal(buf[:off], before[:off])


def test_rope_one_row_for_all_tokens(rt):
    """Stride 0: one row rotated to many positions (and, backward, gradients of each)."""
    x = torch.randn((1, 4, 64), generator=gen(2), device="cuda").expand(50, 4, 64)
    cos, sin = table(50, 64)
    pos = torch.arange(50, device="cuda", dtype=torch.int32)
    out = torch.empty((50, 4, 64), device="cuda")
    ws = rt.status_workspace()
    rt.rope(x, None, pos, cos, sin, out, None, ws)
    want, err = ref.rotate(f64(x), f64(cos), f64(sin), 64, True)
    check(out, want, err, torch.float32, "broadcast")


def test_rope_bad_positions(rt):
    from picolm_qwen_b200 import abi
    x = torch.randn((6, 2, 64), generator=gen(1), device="cuda")
    cos, sin = table(10, 32)
    pos = torch.tensor([0, 10, 9, -1, 2 ** 31 - 1, 3], device="cuda", dtype=torch.int32)
    out, ws = torch.empty_like(x), rt.status_workspace()
    rt.rope(x, None, pos, cos, sin, out, None, ws)
    assert rt.workspace_status(ws) == abi.DEV_BAD_POS and rt.workspace_status(ws) == 0
    nan = torch.isnan(out).flatten(1)
    assert nan[[1, 3, 4]].all() and not nan[[0, 2, 5]].any()


@pytest.mark.parametrize("neox", [True, False])
def test_rope_inverse_is_the_gradient(rt, neox):
    """d(w . rope(x)) / dx = inverse rope(w), against differences of the forward pass itself (it is linear in x, so
    the difference quotient of step h is off by the two calls' roundings over h alone)."""
    n, hq, hd, rot, h = 3, 2, 16, 8, 2.0 ** 6
    g = gen(7)
    x, w = (torch.randn((n, hq, hd), generator=g, device="cuda") for _ in range(2))
    cos, sin = table(9, rot)
    cos, sin = cos * 1.25, sin * 1.25  # a table scaled by mscale: the gradient carries it too
    pos = torch.tensor([8, 0, 3], device="cuda", dtype=torch.int32)
    ws, mode = rt.status_workspace(), 0 if neox else 1

    def fwd(t):
        y = torch.empty_like(t)
        rt.rope(t, None, pos, cos, sin, y, None, ws, rope_mode=mode)
        return f64(y)

    grad = torch.empty_like(w)
    rt.rope(w, None, pos, cos, sin, grad, None, ws, rope_mode=mode, inverse=True)
    grad, wd = f64(grad), f64(w)
    # each call's outputs are off by at most 2.01 2^-24 of 2 * 1.25 * (|x| + h), times |w|, two outputs an element
    tol = 2 * 2 * 2.01 * 2.0 ** -24 * 2.5 * (h + 4) * 4 / h + 2.0 ** -21
    for e in range(n * hq * hd):
        d = torch.zeros(n * hq * hd, device="cuda")
        d[e] = h
        d = d.view(n, hq, hd)
        diff = ((fwd(x + d) - fwd(x)) * wd).sum() / h
        # x + d itself is rounded: by 2^-24 (h + 4) at most, an input change of that size
        assert abs(diff - grad.reshape(-1)[e]) <= tol + 2.0 ** -24 * (h + 4) * 2.5 * 4 * 2 / h


# -- the paged cache ---------------------------------------------------------------


class Batch:
    """A ragged batch over a pool whose unused rows, and rows behind each sequence's length, are NaN."""

    def __init__(self, rt, new, past, hq, hkv, hd, page, cache, layers=2, pad=0, seed=0, neox=True, lead=0):
        from picolm_qwen_b200 import abi
        g = gen(seed)
        self.new, self.past, self.hq, self.hkv, self.hd, self.page = new, past, hq, hkv, hd, page
        self.dt = DT[cache]
        self.total = [a + b for a, b in zip(new, past)]
        need = [-(-t // page) for t in self.total]
        n_pages = sum(need) + 2
        perm = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        cols = max(need) + 1
        rows, at = [], 0
        for n in need:
            rows.append(perm[at:at + n] + [-7] * (cols - n))  # entries past a sequence's rows are not read
            at += n
        self.pages = torch.tensor(rows, dtype=torch.int32, device="cuda")
        self.start = [lead]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.n_tok = self.start[-1] + pad
        self.cfg = abi.Config.make(layers, hq, hkv, hd, cols * page, 1e4, 0 if neox else 1, 1e-6)
        self.cache = rt.PagedCache(self.cfg, page, n_pages, self.dt)
        self.cache.k_pool.fill_(float("nan"))
        self.cache.v_pool.fill_(float("nan"))
        i32 = dict(dtype=torch.int32, device="cuda")
        self.q_start, self.kv_len = torch.tensor(self.start, **i32), torch.tensor(self.total, **i32)
        self.batch = self.cache.batch(self.pages, self.q_start, self.kv_len, self.n_tok, max(new), max(self.total))
        self.rand = lambda *s: torch.randn(s, generator=g, device="cuda")

    def rows(self, pool, layer, b, n):
        """The first n rows of sequence b: [n, hkv, hd]."""
        ids = self.pages[b, :-(-n // self.page)].long()
        return pool[layer, ids].permute(0, 2, 1, 3).reshape(-1, self.hkv, self.hd)[:n]

    def fill(self, layer, k_scale=0.5, v_scale=0.5, upto=None):
        """Random rows below each length (or upto[b]), in both pools."""
        for b, t in enumerate(self.total if upto is None else upto):
            ids = self.pages[b, :-(-t // self.page)].long()
            for pool, sc in ((self.cache.k_pool, k_scale), (self.cache.v_pool, v_scale)):
                x = (sc * self.rand(len(ids) * self.page, self.hkv, self.hd)).to(self.dt)
                x[t:] = float("nan")
                pool[layer, ids] = x.view(len(ids), self.page, self.hkv, self.hd).permute(0, 2, 1, 3)


def want_attn(B, layer, q, out, what, out_dt, q_scale=None):
    """Every sequence and KV head of `out` against the 64-bit form."""
    got = f64(out).reshape(-1, B.hq, B.hd)
    qd = f64(q).reshape(-1, B.hq, B.hd)
    g = B.hq // B.hkv
    for b in range(len(B.new)):
        a, e = B.start[b], B.start[b + 1]
        if a == e:
            continue
        k, v = f64(B.rows(B.cache.k_pool, layer, b, B.total[b])), f64(B.rows(B.cache.v_pool, layer, b, B.total[b]))
        for h in range(B.hq):
            w, err = ref.attention(qd[a:e, h], k[:, h // g], v[:, h // g], B.past[b], B.hd ** -0.5, HALF[B.dt], TINY[B.dt])
            tol = err + HALF[out_dt] * (np.abs(w) + err) + TINY[out_dt]
            d = np.abs(got[a:e, h] - w)
            bad = ~(d <= tol)
            assert not bad.any(), (f"{what}: sequence {b} (new {B.new[b]}, past {B.past[b]}) head {h}: {bad.sum()} of "
                                   f"{bad.size} off, worst {np.nanmax(d / tol):.3g} of the tolerance, NaN "
                                   f"{np.isnan(d).sum()}, first at {np.unravel_index(bad.argmax(), bad.shape)}")


APPENDS = [
    # new, past, hq, hkv, hd, rot, page, input, cache, neox, norm
    ([1], [0], 14, 2, 64, 64, 16, "f32", "f16", True, False),
    ([1] * 40, list(range(40)), 28, 4, 128, 128, 16, "f32", "f16", True, True),
    ([5, 0, 1, 70], [11, 3, 127, 60], 6, 3, 128, 64, 64, "f16", "f16", False, True),
    ([33, 1, 17], [0, 255, 240], 8, 8, 64, 32, 256, "bf16", "bf16", True, False),
    ([3, 2], [1, 0], 71, 1, 64, 16, 32, "f32", "bf16", False, True),
    ([130], [7], 5, 1, 128, 16, 128, "f16", "bf16", False, False),
    ([4, 9], [2, 100], 10, 5, 64, 48, 16, "bf16", "f16", True, True),
]


@pytest.mark.parametrize("new,past,hq,hkv,hd,rot,page,inp,cache,neox,norm", APPENDS)
def test_append(rt, new, past, hq, hkv, hd, rot, page, inp, cache, neox, norm):
    B = Batch(rt, new, past, hq, hkv, hd, page, cache, pad=3, lead=2, neox=neox, seed=len(new))
    B.fill(1, upto=past)
    before = B.cache.k_pool.clone(), B.cache.v_pool.clone()
    n, dt = B.n_tok, DT[inp]
    qkv = B.rand(n, hq + 2 * hkv, hd).to(dt)  # one projection's output: strided rows
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cos, sin = table(B.cfg.max_seq_len, rot)
    qn, kn = (1 + 0.1 * B.rand(hd), 1 + 0.1 * B.rand(hd)) if norm else (None, None)
    qo = torch.full((n, hq, hd), 7.0, device="cuda").to(B.dt)
    B.cache.append(1, B.batch, q, k, v, cos, sin, qo, qn, kn)
    assert B.batch.status() == 0
    assert (qo[:2] == 7).all() and (qo[B.start[-1]:] == 7).all()  # rows of no sequence
    pos = np.concatenate([np.arange(p, p + a) for a, p in zip(new, past)])
    c, s = f64(cos)[pos], f64(sin)[pos]

    def rotated(x, w):
        x, rel = f64(x)[2:B.start[-1]], 0.0
        if w is not None:
            x, rel = ref.rmsnorm(x, f64(w), 1e-6)
        y, err = ref.rotate(x, c, s, rot, neox)
        mag = ref.rotate(np.abs(x), np.abs(c), np.abs(s), rot, neox)[1] / (2.01 * 2.0 ** -24)  # |x0 c| + |x1 s|
        mag[..., rot:] = np.abs(x[..., rot:])
        return y, err + rel * mag

    y, err = rotated(q, qn)
    check(qo[2:B.start[-1]], y, err, B.dt, "q")
    y, err = rotated(k, kn)
    vd = f64(v)[2:B.start[-1]]
    seen = [torch.zeros_like(before[0], dtype=torch.bool) for _ in range(2)]
    at = 0
    for b, (a, p) in enumerate(zip(new, past)):
        if a:
            gk, gv = (B.rows(pool, 1, b, p + a)[p:] for pool in (B.cache.k_pool, B.cache.v_pool))
            check(gk, y[at:at + a], err[at:at + a], B.dt, f"k of sequence {b}")
            check(gv, vd[at:at + a], 0.0, B.dt, f"v of sequence {b}")
        for r in range(p, p + a):
            for m in seen:
                m[1, int(B.pages[b, r // page]), :, r % page] = True
        at += a
    for m, pool, old in zip(seen, (B.cache.k_pool, B.cache.v_pool), before):
        same = (pool == old) | (pool.isnan() & old.isnan())
        assert (same | m).all()  # nothing else was written


def test_append_matches_the_contiguous_cache_bit_for_bit(rt):
    """Without norm the stored keys and values are picoattn_prefill's own."""
    from picolm_qwen_b200 import abi
    n, hq, hkv, hd, page = 83, 8, 4, 128, 16
    B = Batch(rt, [n], [0], hq, hkv, hd, page, "f16")
    q, k, v = B.rand(n, hq, hd), 3 * B.rand(n, hkv, hd), B.rand(n, hkv, hd)
    k[0, 0, :8] = torch.tensor([1e-8, 6e-8, -3e-5, 65519.0, 7e4, -1e-40, 0.0, 1 + 2.0 ** -11], device="cuda")
    cfg = abi.Config.make(2, hq, hkv, hd, B.cfg.max_seq_len, 1e4)
    st = rt.AttnState(cfg)
    out = torch.empty((n, hq * hd), device="cuda")
    assert st.prefill(1, 0, q.view(n, -1), k.view(n, -1), v.view(n, -1), out) == 0
    B.cache.append(1, B.batch, q, k, v, st.rope_cos, st.rope_sin, torch.empty((n, hq, hd), device="cuda").half())
    for pool, flat in ((B.cache.k_pool, st.k_cache), (B.cache.v_pool, st.v_cache)):
        assert torch.equal(B.rows(pool, 1, 0, n).reshape(n, -1).view(torch.int16), flat[0, 1, :n])


def test_append_bad_lengths_and_pages(rt):
    from picolm_qwen_b200 import abi
    B = Batch(rt, [2, 3, 2, 1], [20, 5, 0, 9], 4, 2, 64, 16, "f16")
    before = B.cache.k_pool.clone()
    n = B.n_tok
    q, k, v = B.rand(n, 4, 64), B.rand(n, 2, 64), B.rand(n, 2, 64)
    cos, sin = table(B.cfg.max_seq_len, 64)
    qo = torch.empty((n, 4, 64), device="cuda").half()
    B.kv_len[1] = 2                 # fewer rows than its new tokens
    B.pages[3, 0] = 10 ** 6         # no such page
    B.pages[2, 0] = -1
    B.cache.append(0, B.batch, q, k, v, cos, sin, qo)
    assert B.batch.status() == abi.DEV_BAD_POS | abi.DEV_BAD_PAGE
    nan = qo.isnan().flatten(1).all(1).cpu()
    assert nan.tolist() == [False] * 2 + [True] * 3 + [False] * 3
    changed = ~((B.cache.k_pool == before) | (B.cache.k_pool.isnan() & before.isnan()))
    assert changed.sum() == 2 * 2 * 64  # sequence 0's two rows alone
    B.kv_len[:] = torch.tensor([22, 8, 2, 10 ** 6], dtype=torch.int32)  # longer than the step's bound
    B.pages[2, 0], B.pages[3, 0] = 0, 1
    B.cache.append(0, B.batch, q, k, v, cos, sin, qo)
    assert B.batch.status() == abi.DEV_BAD_POS
    assert qo.isnan().flatten(1).all(1).tolist() == [False] * 7 + [True]


ATTNS = [
    # new, past, hq, hkv, hd, page
    ([1], [0], 14, 2, 64, 16),                                   # one row
    ([1], [511], 32, 4, 64, 16),
    ([1] * 9, [0, 1, 15, 16, 17, 63, 64, 127, 128], 28, 4, 128, 16),
    ([1, 1, 1], [700, 3, 1999], 5, 1, 128, 64),
    ([1] * 70, [(37 * i) % 300 for i in range(70)], 6, 3, 128, 32),
    ([1, 0, 1], [4000, 77, 100], 16, 1, 64, 256),
    ([1], [3000], 71, 1, 64, 16),                                # more q heads per KV head than a tile of single tokens
    ([2, 1, 3], [0, 900, 260], 20, 4, 128, 16),                  # drafts
    ([4] * 3, [1000, 0, 61], 4, 4, 64, 128),
    ([16], [1000], 2, 2, 128, 16),
    ([17], [5000], 1, 1, 128, 64),
    ([1, 40, 0, 129, 2], [700, 0, 5, 300, 1], 28, 4, 128, 32),   # mixed, 7 q heads per KV head
    ([128, 64, 200], [0, 64, 1], 8, 2, 64, 16),
    ([300], [0], 8, 1, 128, 64),
    ([257, 1], [1023, 2047], 6, 2, 128, 128),
    ([90, 33], [130, 16], 9, 3, 64, 256),
    ([5], [3], 128, 1, 128, 16),                                 # 128 q heads on one KV head
    ([3, 50], [10, 0], 48, 1, 64, 32),
    ([30] * 20, [(97 * i) % 500 for i in range(20)], 4, 2, 128, 64),
]


@pytest.mark.parametrize("cache,out", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("new,past,hq,hkv,hd,page", ATTNS)
def test_attention(rt, new, past, hq, hkv, hd, page, cache, out):
    B = Batch(rt, new, past, hq, hkv, hd, page, cache, pad=5, lead=3, seed=sum(past) + hq)
    B.fill(1)
    q = B.rand(B.n_tok, hq, hd).to(B.dt)
    y = torch.full((B.n_tok, hq, hd), 7.0, device="cuda").to(DT[out])
    B.cache.attend(1, B.batch, q, y)
    assert B.batch.status() == 0
    assert (y[:3] == 7).all() and (y[B.start[-1]:] == 7).all()  # rows of no sequence
    want_attn(B, 1, q, y, "attention", DT[out])


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("new,past,hq,hkv,hd,page", [ATTNS[2], ATTNS[7], ATTNS[11], ATTNS[13], ATTNS[15]])
@pytest.mark.parametrize("kind", ["rising", "falling", "spikes", "equal", "far"])
def test_attention_of_hard_scores(rt, new, past, hq, hkv, hd, page, cache, kind):
    """Running maxima that grow at every tile, that never do, single rows that take all the weight, equal scores, and
    scores far below zero."""
    B = Batch(rt, new, past, hq, hkv, hd, page, cache, seed=11)
    B.fill(0)
    for b, t in enumerate(B.total):
        ids = B.pages[b, :-(-t // page)].long()
        r = torch.arange(len(ids) * page, device="cuda", dtype=torch.float32)
        lift = {"rising": r / 24, "falling": -r / 24, "spikes": 9.0 * (r % 97 == 96), "equal": 0 * r,
                "far": -40 + 0 * r}[kind]
        x = torch.zeros((len(ids) * page, hkv, hd), device="cuda")
        if kind not in ("equal", "far"):
            x = 0.3 * B.rand(len(ids) * page, hkv, hd)
        x[..., 0] = lift[:, None]
        x[t:] = float("nan")
        B.cache.k_pool[0, ids] = x.to(B.dt).view(len(ids), page, hkv, hd).permute(0, 2, 1, 3)
    q = B.rand(B.n_tok, hq, hd).to(B.dt)
    q[..., 0] = hd ** 0.5  # the first coordinate's score is the lift itself
    y = torch.empty((B.n_tok, hq, hd), device="cuda")
    B.cache.attend(0, B.batch, q, y)
    want_attn(B, 0, q, y, kind, torch.float32)


def test_attention_of_a_strided_q(rt):
    B = Batch(rt, [1, 30, 2], [40, 5, 100], 6, 2, 64, 16, "f16")
    B.fill(0)
    wide = B.rand(B.n_tok, 10, 64).half()
    y, z = (torch.empty((B.n_tok, 6, 64), device="cuda").half() for _ in range(2))
    B.cache.attend(0, B.batch, wide[:, 2:8], y)
    B.cache.attend(0, B.batch, wide[:, 2:8].contiguous(), z)
    assert torch.equal(y, z)
    want_attn(B, 0, wide[:, 2:8], y, "strided", torch.float16)


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [40, 1, 3, 70, 9]])
def test_attention_bad_lengths_and_pages(rt, new):
    """A bad sequence gives NaN in its own rows and its status bit; the others are as ever."""
    from picolm_qwen_b200 import abi
    B = Batch(rt, new, [300, 20, 50, 10, 400], 8, 2, 128, 16, "f16")
    B.fill(0)
    q = B.rand(B.n_tok, 8, 128).half()
    good, y = (torch.empty((B.n_tok, 8, 128), device="cuda").half() for _ in range(2))
    B.cache.attend(0, B.batch, q, good)
    assert B.batch.status() == 0

    def expect(bits, bad):
        y.fill_(7)
        B.cache.attend(0, B.batch, q, y)
        assert B.batch.status() == bits
        for b in range(5):
            rows = slice(B.start[b], B.start[b + 1])
            if b in bad:
                assert y[rows].isnan().all(), b
            else:
                assert torch.equal(y[rows], good[rows]) or \
                    (f64(y[rows]) - f64(good[rows])).max() < 0.01, b  # another split of the rows: other roundings

    pages, lens = B.pages.clone(), B.kv_len.clone()
    B.pages[0, 2] = B.cache.k_pool.shape[1]
    B.pages[3, 0] = -1
    expect(abi.DEV_BAD_PAGE, {0, 3})
    B.pages.copy_(pages)
    B.kv_len[1] = 0
    B.kv_len[4] = 1 << 30
    expect(abi.DEV_BAD_POS, {1, 4})
    B.kv_len.copy_(lens)
    expect(0, set())
    B.kv_len.fill_(0)
    expect(abi.DEV_BAD_POS, {0, 1, 2, 3, 4})


def test_attention_of_no_new_tokens(rt):
    """A step whose sequences all have nothing new writes nothing."""
    B = Batch(rt, [1, 1], [30, 40], 4, 2, 64, 16, "f16")
    B.fill(0)
    B.q_start.fill_(0)
    y = torch.full((2, 4, 64), 7.0, device="cuda").half()
    B.cache.attend(0, B.batch, B.rand(2, 4, 64).half(), y)
    assert (y == 7).all() and B.batch.status() == 0


def gpu_attn(B, layer, q):
    """The 64-bit form on the GPU, for batches too large for want_attn, with its error bound's main terms: the weights'
    rounding (u |v| weighted), and a score error of hd 2^-23 sum|q k|; 2^-16 for the fp32 sums of up to 16,384 rows
    (n / 8 additions of 2^-23, twice) and the exponential."""
    out = torch.zeros((B.n_tok, B.hq, B.hd), dtype=torch.float64, device="cuda")
    err = torch.zeros_like(out)
    g = B.hq // B.hkv
    for b, (n, t) in enumerate(zip(B.new, B.total)):
        if n == 0:
            continue
        k, v = (B.rows(p, layer, b, t).double() for p in (B.cache.k_pool, B.cache.v_pool))
        x = q[B.start[b]:B.start[b] + n].double()
        hidden = torch.arange(t, device="cuda") > (t - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(B.hq):
            s = (x[:, h] @ k[:, h // g].T) * B.hd ** -0.5
            mag = (x[:, h].abs() @ k[:, h // g].abs().T).amax(-1, keepdim=True) * B.hd ** -0.5
            p = s.masked_fill(hidden, -np.inf).softmax(-1)
            out[B.start[b]:B.start[b] + n, h] = p @ v[:, h // g]
            w, most = p @ v[:, h // g].abs(), v[:, h // g].abs().max()
            # weights below the type's normal range are off by TINY each, of a sum of at least 1
            err[B.start[b]:B.start[b] + n, h] = (HALF[B.dt] + 2 * B.hd * 2.0 ** -23 * mag + 2.0 ** -16) * w + \
                t * TINY[B.dt] * most
    return out, err


@pytest.mark.parametrize("seed", range(10))
def test_random_batches_one_after_the_other(rt, seed):
    """Two ragged batches of other shapes, run in turn without waiting: every call's outputs against the 64-bit form."""
    import random
    rng = random.Random(seed)
    two = []
    for i in range(2):
        hq, hkv, hd = rng.choice([(32, 4, 64), (14, 2, 64), (28, 4, 128), (32, 8, 128), (40, 8, 128), (6, 3, 64)])
        ones, chunks = (rng.randrange(0, 30), rng.randrange(1, 4)) if (seed + i) % 4 else (rng.randrange(1, 40), 0)
        new = [1] * ones + [rng.randrange(2, 400) for _ in range(chunks)]
        rng.shuffle(new)
        past = [rng.randrange(0, 2000) for _ in new]
        B = Batch(rt, new, past, hq, hkv, hd, rng.choice([16, 32, 64, 128, 256]), rng.choice(["f16", "bf16"]), layers=1,
                  pad=rng.randrange(3), seed=seed)
        B.fill(0)
        B.q = B.rand(B.n_tok, hq, hd).to(B.dt)
        B.outs = [torch.full((B.n_tok, hq, hd), float("nan"), device="cuda", dtype=B.dt) for _ in range(6)]
        two.append(B)
    torch.cuda.synchronize()
    for r in range(6):
        for B in two:
            B.cache.attend(0, B.batch, B.q, B.outs[r])
    for B in two:
        assert B.batch.status() == 0
        want, err = gpu_attn(B, 0, B.q)
        tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]
        for r, y in enumerate(B.outs):
            d = (y.double() - want).abs()[:B.start[-1]]
            bad = ~(d <= tol[:B.start[-1]])
            assert not bad.any(), (f"run {r}: {int(bad.sum())} off, worst {float((d / tol[:B.start[-1]]).max()):.3g} of the "
                                   f"tolerance, first at {bad.nonzero()[0].tolist()}")


@pytest.mark.parametrize("seed", range(24))
def test_random_batches_of_few_rows(rt, seed):
    """Tokens and short drafts, one sequence to hundreds, short and long: streams inside a CTA, cut over several, cut near
    their ends, more streams than CTAs; twice in turn with a batch of one sequence."""
    import random
    rng = random.Random(100 + seed)
    two = []
    for one in (False, True):
        hq, hkv, hd = rng.choice([(32, 4, 64), (14, 2, 64), (28, 4, 128), (32, 8, 128), (40, 8, 128), (6, 3, 64), (16, 1, 128)])
        most = rng.choice([1, 16 // (hq // hkv), 32 // (hq // hkv)])
        n = 1 if one else rng.choice([2, 5, 17, 33, 60, 150])
        longest = rng.choice([20, 300, 700, 1500] + ([6000, 16000] if one else [3000] if n < 40 else []))
        new = [rng.randrange(0 if n > 4 else 1, most + 1) for _ in range(n)]
        new[0] = most
        past = [rng.choice([longest, rng.randrange(longest), rng.randrange(16)]) for _ in new]
        B = Batch(rt, new, past, hq, hkv, hd, rng.choice([16, 32, 64, 128, 256]), rng.choice(["f16", "bf16"]), layers=1,
                  pad=rng.randrange(3), seed=seed)
        B.fill(0)
        B.q = B.rand(B.n_tok, hq, hd).to(B.dt)
        B.outs = [torch.full((B.n_tok, hq, hd), float("nan"), device="cuda", dtype=B.dt) for _ in range(2)]
        two.append(B)
    torch.cuda.synchronize()
    for r in range(2):
        for B in two:
            B.cache.attend(0, B.batch, B.q, B.outs[r])
    for B in two:
        assert B.batch.status() == 0
        want, err = gpu_attn(B, 0, B.q)
        tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]
        for r, y in enumerate(B.outs):
            d = (y.double() - want).abs()[:B.start[-1]]
            bad = ~(d <= tol[:B.start[-1]])
            assert not bad.any(), (f"run {r}: {int(bad.sum())} off, worst {float((d / tol[:B.start[-1]]).max()):.3g} of the "
                                   f"tolerance, first at {bad.nonzero()[0].tolist()}")


@pytest.mark.parametrize("n,past", [(3, 5000), (200, 900), (200, 100)])
def test_bad_lengths_among_few_rows(rt, n, past):
    """Sequences outside the host's bounds beside good ones: NaN in their rows, the others' rows as ever, in each way that a
    batch of single tokens is split."""
    from picolm_qwen_b200 import abi
    B = Batch(rt, [1] * n, [past] * n, 4, 2, 128, 64, "f16")
    B.fill(0)
    q = B.rand(B.n_tok, 4, 128).half()
    want, err = gpu_attn(B, 0, q)
    off = [1, n - 1]
    B.kv_len[off[0]] = 0
    B.kv_len[off[1]] = past + 1000000
    y = torch.zeros((B.n_tok, 4, 128), device="cuda").half()
    B.cache.attend(0, B.batch, q, y)
    assert B.batch.status() == abi.DEV_BAD_POS
    keep = [i for i in range(n) if i not in off]
    assert y[off].isnan().all()
    tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]
    assert ((y.double() - want).abs() <= tol)[keep].all()


def test_many_sequences(rt):
    """More sequences than a block has threads, some of them empty."""
    n = 1500
    new = [(i % 3 != 1) * 1 for i in range(n)]
    B = Batch(rt, new, [(i * 7) % 41 for i in range(n)], 4, 2, 64, 16, "f16")
    B.fill(0)
    q = B.rand(B.n_tok, 4, 64).half()
    y = torch.empty((B.n_tok, 4, 64), device="cuda").half()
    B.cache.attend(0, B.batch, q, y)
    want_attn(B, 0, q, y, "many", torch.float16)
    new = [(i % 3) * 5 for i in range(n)]  # chunks of up to 10 tokens
    B = Batch(rt, new, [(i * 7) % 41 for i in range(n)], 8, 2, 64, 16, "f16")
    B.fill(0)
    q = B.rand(B.n_tok, 8, 64).half()
    y = torch.empty((B.n_tok, 8, 64), device="cuda").half()
    B.cache.attend(0, B.batch, q, y)
    want_attn(B, 0, q, y, "many chunks", torch.float16)


def test_long_cache_past_32_bit_offsets(rt):
    """A layer whose pools pass 2^32 bytes, its sequence's pages at the far end."""
    hkv, hd, page = 8, 128, 256
    n_pages = 9000  # 9000 * 8 * 256 * 128 * 2 = 4.7 GB a pool
    from picolm_qwen_b200 import abi
    cfg = abi.Config.make(1, 16, hkv, hd, 4096, 1e4)
    cache = rt.PagedCache(cfg, page, n_pages)
    g = gen(3)
    for new, past in ((1, 600), (70, 600)):
        pages = torch.tensor([[8999, 3, 8998]], dtype=torch.int32, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        batch = cache.batch(pages, torch.tensor([0, new], **i32), torch.tensor([past + new], **i32), new, new, 700)
        for pool in (cache.k_pool, cache.v_pool):
            pool[0, [8999, 3, 8998]] = (0.5 * torch.randn((3, hkv, page, hd), generator=g, device="cuda")).half()
        cos, sin = table(4096, hd)
        q, k, v = (torch.randn((new, h, hd), generator=g, device="cuda") for h in (16, hkv, hkv))
        qo, y = (torch.empty((new, 16, hd), device="cuda").half() for _ in range(2))
        cache.append(0, batch, q, k, v, cos, sin, qo)
        cache.attend(0, batch, qo, y)
        assert batch.status() == 0
        kk, vv = (f64(p[0, pages[0].long()].permute(0, 2, 1, 3).reshape(-1, hkv, hd)[:past + new])
                  for p in (cache.k_pool, cache.v_pool))
        assert np.abs(vv[past:] - f64(v)).max() < 0.01
        for h in (0, 15):
            w, err = ref.attention(f64(qo)[:, h], kk[:, h // 2], vv[:, h // 2], past, hd ** -0.5, 2.0 ** -11, 2.0 ** -25)
            check(y[:, h], w, err, torch.float16, f"head {h}")




def test_steps_together_match_one_prefill(rt):
    """append -> attend in chunks of every size, then single tokens, two layers: the last step's outputs and the cache
    rows are those of one call over everything."""
    from picolm_qwen_b200 import abi
    hq, hkv, hd, page = 8, 2, 64, 16
    lens, g = [60, 33, 90], gen(4)
    cols = 6
    perm = torch.randperm(18, generator=g, device="cuda").to(torch.int32).view(3, cols)
    cfg = abi.Config.make(2, hq, hkv, hd, 96, 1e4)
    full = [torch.randn((sum(lens), h, hd), generator=g, device="cuda") for h in (hq, hkv, hkv)]
    off = np.cumsum([0] + lens)
    cos, sin = table(96, 32)
    i32 = dict(dtype=torch.int32, device="cuda")

    def step(cache, layer, spans):
        """spans[b] = (first, last) positions of sequence b in this step."""
        idx = torch.cat([torch.arange(off[b] + a, off[b] + e) for b, (a, e) in enumerate(spans)]).cuda()
        n = [e - a for a, e in spans]
        batch = cache.batch(perm, torch.tensor(np.cumsum([0] + n), **i32), torch.tensor([e for _, e in spans], **i32),
                            len(idx), max(n), 96)
        q, k, v = (t[idx].contiguous() for t in full)
        qo, y = torch.empty_like(q).half(), torch.empty_like(q)
        cache.append(layer, batch, q, k, v, cos, sin, qo)
        cache.attend(layer, batch, qo, y)
        assert batch.status() == 0
        return dict(zip(idx.tolist(), y))

    one, many = (rt.PagedCache(cfg, page, 18) for _ in range(2))
    for layer in range(2):
        want = step(one, layer, [(0, n) for n in lens])
        got, at = {}, [0, 0, 0]
        for sizes in ([20, 1, 64], [1, 3, 1], [2, 0, 5], [16, 9, 1], [1, 1, 1], [1, 0, 1], [19, 19, 17]):
            spans = [(a, min(n, a + s)) for a, n, s in zip(at, lens, sizes)]
            at = [e for _, e in spans]
            got.update(step(many, layer, spans))
        assert at == lens and sorted(got) == sorted(want)
        for b in range(3):  # every allocated row that was appended
            for pa, pb in ((one.k_pool, many.k_pool), (one.v_pool, many.v_pool)):
                ra, rb = (p[layer, perm[b].long()].permute(0, 2, 1, 3).reshape(-1, hkv, hd)[:lens[b]] for p in (pa, pb))
                assert torch.equal(ra, rb)
        a, w = torch.stack([got[i] for i in sorted(got)]), torch.stack([want[i] for i in sorted(want)])
        # both within the weights' rounding of the formula: |v| < 5, 2 * 2^-11 * mean |v| and the fp32 sums
        assert (a - w).abs().max() <= 2 * 2.0 ** -11 * 5


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 7]])
def test_captured_step_replayed_with_other_lengths(rt, new):
    """A step captured once, replayed after the page table and lengths changed, next to another captured step with its
    own workspace on another stream."""
    past = [200, 31, 500]
    two = []
    for seed in (1, 2):
        B = Batch(rt, new, past, 8, 2, 128, 16, "f16", seed=seed)
        B.batch = B.cache.batch(B.pages, B.q_start, B.kv_len, B.n_tok, max(new), B.cfg.max_seq_len)
        B.fill(0)
        B.q = [B.rand(B.n_tok, h, 128) for h in (8, 2, 2)]
        B.tab = table(B.cfg.max_seq_len, 128)
        B.qo, B.y = (torch.empty((B.n_tok, 8, 128), device="cuda").half() for _ in range(2))
        B.stream, B.graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        B.stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(B.stream):
            B.cache.append(0, B.batch, *B.q, *B.tab, B.qo)  # first use outside the capture
            B.cache.attend(0, B.batch, B.qo, B.y)
            B.stream.synchronize()
            with torch.cuda.graph(B.graph, stream=B.stream):
                B.cache.append(0, B.batch, *B.q, *B.tab, B.qo)
                B.cache.attend(0, B.batch, B.qo, B.y)
        two.append(B)
    torch.cuda.synchronize()
    for past2 in ([200, 31, 500], [100, 8, 77], [0, 0, 0]):
        for B in two:
            B.past, B.total = past2, [a + b for a, b in zip(new, past2)]
            B.kv_len.copy_(torch.tensor(B.total, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for B in two:
                with torch.cuda.stream(B.stream):
                    B.graph.replay()
        torch.cuda.synchronize()
        for B in two:
            assert B.batch.status() == 0
            want_attn(B, 0, B.qo, B.y, f"replayed with {past2}", torch.float16)


def test_repeated_calls_give_the_same_bits(rt):
    B = Batch(rt, [1, 200, 3, 1], [3000, 100, 900, 64], 8, 2, 128, 16, "bf16")
    B.fill(0)
    q = B.rand(B.n_tok, 8, 128).bfloat16()
    first = torch.empty((B.n_tok, 8, 128), device="cuda")
    B.cache.attend(0, B.batch, q, first)
    for _ in range(20):
        y = torch.empty_like(first)
        B.cache.attend(0, B.batch, q, y)
        assert torch.equal(y, first)


def test_refusals_of_the_python_entries(rt):
    from picolm_qwen_b200 import abi
    B = Batch(rt, [1, 2], [3, 4], 4, 2, 64, 16, "f16")
    q = B.rand(3, 4, 64).half()
    out = torch.empty_like(q)
    with pytest.raises(ValueError):
        B.cache.attend(0, B.batch, q.float(), out)
    with pytest.raises(ValueError):
        B.cache.attend(0, B.batch, q[:2], out)
    with pytest.raises(ValueError):
        B.cache.attend(0, B.batch, q.cpu(), out)
    with pytest.raises(ValueError):
        B.cache.attend(0, B.batch, q.transpose(0, 1).contiguous().transpose(0, 1), out)
    with pytest.raises(abi.PicoAttnError):
        B.cache.attend(2, B.batch, q, out)
    with pytest.raises(abi.PicoAttnError):
        B.cache.batch(B.pages, B.q_start, B.kv_len, 3, 2, 10 ** 6)
        B.cache.attend(0, B.cache.batch(B.pages, B.q_start, B.kv_len, 3, 2, 10 ** 6), q, out)
    cos, sin = table(8, 64)  # fewer rows than positions
    with pytest.raises(ValueError):
        B.cache.append(0, B.batch, q, q[:, :2].contiguous(), q[:, :2].contiguous(), cos, sin, out)
    with pytest.raises(ValueError):
        rt.rope(q, None, torch.zeros(3, device="cuda"), cos, sin, out, None, rt.status_workspace())
