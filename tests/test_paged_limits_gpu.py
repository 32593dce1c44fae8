"""The paged operators where a step is at the edge of what its description allows, against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

import pagedref as ref
from test_paged_gpu import HALF, TINY, Batch, f64, gpu_attn, rt, table  # noqa: F401

pytestmark = pytest.mark.gpu

U_P = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}     # a weight's rounding
TINY_P = {"f16": 2.0 ** -32, "bf16": 2.0 ** -130}  # the largest weight that may vanish, of a largest of 1


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("new,past", [([1], [300]), ([1, 3], [3000, 700]), ([40], [300]), ([70, 9], [200, 3000])])
@pytest.mark.parametrize("strong_last", [False, True])
def test_weights_far_below_the_largest(rt, new, past, cache, strong_last):  # noqa: F811
    """One key takes nearly all of the weight and its V is 0, so that the output is what the others add up to: 2^-26 to
    2^-28 each.  Tolerance: ref.attention's, with weights off by half a step or by 2^-32 of the largest."""
    hq, hkv, hd, page = 4, 2, 64, 16
    B = Batch(rt, new, past, hq, hkv, hd, page, cache, layers=1)
    for b, t in enumerate(B.total):
        ids = B.pages[b, :-(-t // page)].long()
        r = torch.arange(len(ids) * page, device="cuda")
        strong = past[b] - 1 if strong_last else 0
        far = -18.5 + 0.5 * (r % 3 - 1)  # natural units: 2^-26 to 2^-27.4
        k = torch.zeros((len(ids) * page, hkv, hd), device="cuda")
        k[..., 0] = torch.where(r == strong, 0.0, far)[:, None]
        v = torch.where(r == strong, 0.0, 1.0)[:, None, None].expand_as(k).clone()
        k[t:], v[t:] = float("nan"), float("nan")
        for pool, x in ((B.cache.k_pool, k), (B.cache.v_pool, v)):
            pool[0, ids] = x.to(B.dt).view(len(ids), page, hkv, hd).permute(0, 2, 1, 3)
    q = torch.zeros((B.n_tok, hq, hd), device="cuda")
    q[..., 0] = hd ** 0.5
    q = q.to(B.dt)
    y = torch.full((B.n_tok, hq, hd), float("nan"), device="cuda")
    B.cache.attend(0, B.batch, q, y)
    assert B.batch.status() == 0
    got, qd = f64(y), f64(q)
    for b in range(len(new)):
        a, e = B.start[b], B.start[b + 1]
        k, v = (f64(B.rows(p, 0, b, B.total[b])) for p in (B.cache.k_pool, B.cache.v_pool))
        for h in range(hq):
            w, err = ref.attention(qd[a:e, h], k[:, h // 2], v[:, h // 2], past[b], hd ** -0.5, U_P[cache], TINY_P[cache])
            d = np.abs(got[a:e, h] - w)
            tol = err + 2.0 ** -24 * w
            assert (w > 0).all() and (d <= tol).all(), f"sequence {b} head {h}: {(d / tol).max():.3g} of the tolerance"


@pytest.mark.parametrize("new,past", [([2000], [40]), ([1, 1], [600, 40])])
def test_a_workspace_that_a_prefill_used(rt, new, past):  # noqa: F811
    """Calls one after the other may share a workspace, those of the contiguous entries too."""
    from picolm_qwen_b200 import abi
    hq, hkv, hd, n = 32, 8, 64, 700
    B = Batch(rt, new, past, hq, hkv, hd, 16, "f16")
    B.fill(0)
    q = B.rand(B.n_tok, hq, hd).half()
    want, got = (torch.full((B.n_tok, hq, hd), float("nan"), device="cuda").half() for _ in range(2))
    B.cache.attend(0, B.batch, q, want)
    cfg = abi.Config.make(1, hq, hkv, hd, n, 1e4)
    st = rt.AttnState(cfg)
    out = torch.empty((n, hq * hd), device="cuda")
    assert st.prefill(0, 0, B.rand(n, hq * hd), B.rand(n, hkv * hd), B.rand(n, hkv * hd), out,
                      workspace=B.batch.workspace) == 0
    B.cache.attend(0, B.batch, q, got)
    assert B.batch.status() == 0 and torch.equal(got, want)


I32 = 2 ** 31 - 1
SPANS = [  # q_start of three sequences whose own rows would be 0-1, 2-4, 5
    [6, 2, -1, 6],                # ends before their beginnings, then a beginning below 0
    [0, 2, 2 * 10 ** 9, 6],       # past n_tok, then before it
    [I32, -I32 - 1, 0, 6],        # whose difference passes 32 bits
    [-5, 2, I32, -2],
    [-I32 - 1, I32, 6, 6],
    [0, 2, 5, I32],
]


@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("form", ["streams", "slices", "blocks", "cut blocks"])
def test_attention_of_spans_outside_the_batch(rt, spans, form):  # noqa: F811
    """In each way that a batch is split.  Any values in q_start: a sequence with rows outside [0, n_tok), or an end before its beginning, is flagged; the
    rows of the step that it covers are NaN, those of no sequence are not written, a good sequence's are the formula's."""
    from picolm_qwen_b200 import abi
    past = 3000 if form in ("slices", "cut blocks") else 40
    B = Batch(rt, [2, 3, 1], [past] * 3, 8, 2, 64, 16, "f16", layers=1)
    B.batch = B.cache.batch(B.pages, B.q_start, B.kv_len, 6, 6 if form in ("streams", "slices") else 30,
                            B.cfg.max_seq_len)
    B.fill(0)
    q = B.rand(8, 8, 64).half()[1:7]  # a row more on both sides of q and out
    area = torch.full((8, 8, 64), 7.0, device="cuda").half()
    want, err = gpu_attn(B, 0, q)
    tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]
    B.q_start.copy_(torch.tensor(spans, dtype=torch.int64).to(torch.int32))
    B.cache.attend(0, B.batch, q, area[1:7])
    assert B.batch.status() == abi.DEV_BAD_POS
    assert (area[[0, 7]] == 7).all()
    for t in range(6):
        covers = [b for b in range(3) if max(spans[b], 0) <= t < min(spans[b + 1], 6)]
        bad = [b for b in covers if not 0 <= spans[b] <= spans[b + 1] <= 6]
        y = area[1 + t]
        if not covers:
            assert (y == 7).all(), t
        elif bad:
            assert y.isnan().all(), t
        elif spans[covers[0]:covers[0] + 2] == B.start[covers[0]:covers[0] + 2]:
            assert ((y.double() - want[t]).abs() <= tol[t]).all(), t
        else:
            assert y.isfinite().all(), t


def test_append_of_a_decreasing_q_start(rt):  # noqa: F811
    """Tokens that are not their sequence's own by its span: flagged, NaN, and no row of the cache is written for them."""
    from picolm_qwen_b200 import abi
    hq, hkv, hd, page, n = 4, 2, 64, 16, 100
    B = Batch(rt, [n, 0, 3], [7, 40, 21], hq, hkv, hd, page, "f16", layers=2)
    B.fill(1, upto=B.past)
    pools = B.cache.k_pool, B.cache.v_pool
    before = [p.clone() for p in pools]
    B.batch = B.cache.batch(B.pages, B.q_start, B.kv_len, n, n, max(B.total))
    B.q_start.copy_(torch.tensor([0, n, 2, 5], dtype=torch.int32))
    q, k, v = B.rand(n, hq, hd), B.rand(n, hkv, hd), B.rand(n, hkv, hd)
    qo = torch.full((n, hq, hd), 7.0, device="cuda").half()
    B.cache.append(1, B.batch, q, k, v, *table(B.cfg.max_seq_len, hd), qo)
    assert B.batch.status() == abi.DEV_BAD_POS
    nan = qo.isnan().flatten(1)
    assert not nan[:2].any() and nan[2:].all()  # 2 to 4 go to the second sequence by number, the others to the third
    written = {(0, 7): 0, (0, 8): 1}  # positions of the first sequence
    for pool, old in zip(pools, before):
        same = ((pool == old) | (pool.isnan() & old.isnan())).all(-1)  # [layer, page, head, row]
        changed = {(i, p, r) for i, p, h, r in (~same).nonzero().tolist()}
        assert changed == {(1, int(B.pages[b, r // page]), r % page) for b, r in written}
    for (b, r), t in written.items():
        assert (B.rows(pools[1], 1, b, r + 1)[r].float() - v[t]).abs().max() <= 2.0 ** -11 * 8  # |v| < 8


@pytest.mark.parametrize("new,past", [([1, 2, 1], [40, 300, 9]), ([1, 2, 1], [9000, 3000, 40]), ([5, 7], [9000, 40])])
def test_waits_that_give_up(rt, new, past):  # noqa: F811
    """With the sticky timeout bit set, every wait of the call gives up unless its phase is there already: rows are the
    formula's, NaN or as they were, the bit stays until it is read, the next call is as ever; so is a call on another
    workspace beside it."""
    from picolm_qwen_b200 import abi
    B = Batch(rt, new, past, 8, 2, 64, 16, "f16", layers=1)
    B.fill(0)
    other = B.cache.batch(B.pages, B.q_start, B.kv_len, B.n_tok, max(new), max(B.total))
    q = B.rand(B.n_tok, 8, 64).half()
    want, err = gpu_attn(B, 0, q)
    tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]
    good = lambda y: ((y.double() - want).abs() <= tol).all(-1)  # noqa: E731
    side, rest = torch.cuda.Stream(), torch.empty_like(q)
    y = torch.full_like(q, 7.0)
    B.batch.workspace[0] = abi.DEV_TIMEOUT
    torch.cuda.synchronize()
    for _ in range(20):
        B.cache.attend(0, B.batch, q, y)
        B.cache.attend(0, other, q, rest, stream=side)
    side.synchronize()
    assert B.batch.status() == abi.DEV_TIMEOUT and other.status() == 0
    assert good(rest).all()
    assert (good(y) | (y == 7).all(-1) | y.isnan().all(-1)).all()
    y.fill_(7.0)
    B.cache.attend(0, B.batch, q, y)
    assert B.batch.status() == 0 and good(y).all()


@pytest.mark.parametrize("new,past", [([40, 1], [30, 9]), ([400, 1, 33], [900, 3000, 40]), ([2000], [40])])
def test_waits_of_chunks_that_give_up(rt, new, past):  # noqa: F811
    """The same for the chunk kernel, whose outputs are not defined then: nothing but them is written, a call on another
    workspace beside it and the next one are as ever."""
    from picolm_qwen_b200 import abi
    B = Batch(rt, new, past, 8, 2, 64, 16, "f16", layers=1)
    B.fill(0)
    other = B.cache.batch(B.pages, B.q_start, B.kv_len, B.n_tok, max(new), max(B.total))
    q = B.rand(B.n_tok, 8, 64).half()
    want, err = gpu_attn(B, 0, q)
    tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]
    good = lambda y: ((y.double() - want).abs() <= tol).all()  # noqa: E731
    side, rest = torch.cuda.Stream(), torch.empty_like(q)
    area = torch.full((B.n_tok + 2, 8, 64), 7.0, device="cuda").half()
    B.batch.workspace[0] = abi.DEV_TIMEOUT
    torch.cuda.synchronize()
    for _ in range(20):
        B.cache.attend(0, B.batch, q, area[1:-1])
        B.cache.attend(0, other, q, rest, stream=side)
    side.synchronize()
    assert B.batch.status() == abi.DEV_TIMEOUT and other.status() == 0
    assert good(rest) and (area[[0, -1]] == 7).all()
    B.cache.attend(0, B.batch, q, area[1:-1])
    assert B.batch.status() == 0 and good(area[1:-1])


@pytest.mark.parametrize("bad", ["kv_len", "rows"])
def test_append_flags_sequences_without_a_row(rt, bad):  # noqa: F811
    """A sequence outside the bounds is flagged whether or not one of the call's rows is its own, as by the attention."""
    from picolm_qwen_b200 import abi
    B = Batch(rt, [3, 0, 0], [20, 9, 4], 4, 2, 64, 16, "f16", layers=1)
    B.fill(0)
    q, k, v = B.rand(3, 4, 64), B.rand(3, 2, 64), B.rand(3, 2, 64)
    tab = table(B.cfg.max_seq_len, 64)
    want, got = (torch.full((3, 4, 64), float("nan"), device="cuda").half() for _ in range(2))
    B.cache.append(0, B.batch, q, k, v, *tab, want)
    assert B.batch.status() == 0
    if bad == "kv_len":
        B.kv_len[1] = -1
    else:
        B.q_start[3] = 5  # the last sequence's rows lie behind n_tok
    for name in ("append", "attend"):
        if name == "append":
            B.cache.append(0, B.batch, q, k, v, *tab, got)
        else:
            B.cache.attend(0, B.batch, got, torch.empty_like(got))
        assert B.batch.status() == abi.DEV_BAD_POS, name
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [40, 1, 3, 70, 9]])
def test_good_sequences_beside_bad_ones(rt, new):  # noqa: F811
    """Bad pages and lengths beside good sequences, whose rows are the formula's."""
    from picolm_qwen_b200 import abi
    B = Batch(rt, new, [300, 20, 50, 10, 400], 8, 2, 128, 16, "f16", layers=1)
    B.fill(0)
    q = B.rand(B.n_tok, 8, 128).half()
    want, err = gpu_attn(B, 0, q)
    tol = err + HALF[B.dt] * (want.abs() + err) + TINY[B.dt]

    def expect(bits, bad):
        y = torch.full((B.n_tok, 8, 128), 7.0, device="cuda").half()
        B.cache.attend(0, B.batch, q, y)
        assert B.batch.status() == bits
        for b in range(5):
            rows = slice(B.start[b], B.start[b + 1])
            if b in bad:
                assert y[rows].isnan().all(), b
            else:
                d = (y[rows].double() - want[rows]).abs()
                assert (d <= tol[rows]).all(), f"sequence {b}: {float((d / tol[rows]).max()):.3g} of the tolerance"

    pages = B.pages.clone()
    B.pages[0, 2] = B.cache.k_pool.shape[1]
    B.pages[3, 0] = -1
    expect(abi.DEV_BAD_PAGE, {0, 3})
    B.pages.copy_(pages)
    B.kv_len[1] = 0
    B.kv_len[4] = 1 << 30
    expect(abi.DEV_BAD_POS, {1, 4})


def test_one_token_tensors_of_any_stride(rt):  # noqa: F811
    """A dimension of size 1 may have any stride, such as one token's heads turned to the front."""
    hq, hkv, hd = 4, 2, 64
    B = Batch(rt, [1], [35], hq, hkv, hd, 16, "f16", layers=1)
    B.fill(0, upto=[35])
    cos, sin = table(B.cfg.max_seq_len, hd)
    pos, ws = torch.tensor([35], device="cuda", dtype=torch.int32), rt.status_workspace()
    plain = [B.rand(1, h, hd).half() for h in (hq, hkv, hkv)]
    turned = [torch.empty_strided(t.shape, (hd, hd, 1), device="cuda", dtype=t.dtype).copy_(t) for t in plain]
    got = []
    for q, k, v in (plain, turned):
        assert q.is_contiguous()
        r, o, qo = (torch.empty_strided(q.shape, q.stride(), device="cuda", dtype=q.dtype) for _ in range(3))
        rk = torch.empty_strided(k.shape, k.stride(), device="cuda", dtype=k.dtype)
        rt.rope(q, k, pos, cos, sin, r, rk, ws)
        B.cache.append(0, B.batch, q, k, v, cos, sin, qo)
        B.cache.attend(0, B.batch, qo, o)
        got.append([t.clone() for t in (r, rk, qo, o, B.rows(B.cache.k_pool, 0, 0, 36), B.rows(B.cache.v_pool, 0, 0, 36))])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_refuses_what_lies_on_another_device(rt):  # noqa: F811
    """A batch of another device's cache, a stream of another device (made up: one GPU is enough)."""
    B = Batch(rt, [1], [3], 4, 2, 64, 16, "f16", layers=1)
    B.fill(0)
    q = B.rand(1, 4, 64).half()
    y = torch.empty_like(q)
    k, tab = B.rand(1, 2, 64).half(), table(B.cfg.max_seq_len, 64)

    class Stream:
        device_index, cuda_stream = B.cache.index + 1, torch.cuda.current_stream().cuda_stream

    with pytest.raises(ValueError):
        B.cache.attend(0, B.batch, q, y, stream=Stream())
    with pytest.raises(ValueError):
        rt.rope(q, None, B.kv_len, *tab, y, None, rt.status_workspace(), stream=Stream())
    B.batch.index = B.cache.index + 1
    with pytest.raises(ValueError):
        B.cache.attend(0, B.batch, q, y)
    with pytest.raises(ValueError):
        B.cache.append(0, B.batch, q, k, k, *tab, y)


def test_status_of_a_step_on_another_stream(rt):  # noqa: F811
    from picolm_qwen_b200 import abi
    B = Batch(rt, [1, 1], [30, 40], 4, 2, 64, 16, "f16", layers=1)
    B.fill(0)
    B.pages[1, 0] = -1
    q = B.rand(2, 4, 64).half()
    y = torch.empty_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # some 25 ms
    B.cache.attend(0, B.batch, q, y, stream=side)
    assert B.batch.status(side) == abi.DEV_BAD_PAGE
    assert B.batch.status() == 0


def test_a_batch_dropped_while_another_stream_uses_it(rt):  # noqa: F811
    """The memory of a batch is not handed out again before its calls on other streams are through."""
    B = Batch(rt, [1, 1], [30, 4000], 4, 2, 64, 16, "f16", layers=1)
    B.fill(0)
    q = B.rand(2, 4, 64).half()
    want, y = torch.empty_like(q), torch.empty_like(q)
    B.cache.attend(0, B.batch, q, want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for explicit in (True, False):
        batch = B.cache.batch(B.pages, B.q_start, B.kv_len, 2, 1, max(B.total))
        n, at = batch.workspace.numel(), batch.workspace.data_ptr()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)  # some 50 ms
            if not explicit:
                B.cache.attend(0, batch, q, y)
        if explicit:
            B.cache.attend(0, batch, q, y, stream=side)
        del batch
        other = torch.empty(n, dtype=torch.uint8, device="cuda")
        assert not side.query() and other.data_ptr() != at
        side.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("spans", SPANS + [[0, 2, 5, 6]])
@pytest.mark.parametrize("norm", [False, True])
def test_append_of_spans_outside_the_batch(rt, spans, norm):  # noqa: F811
    """Any values in q_start: only rows of good sequences' own positions are stored, and they hold what the good step
    stores; q_out rows are the good step's or NaN, and none outside the step is written."""
    from picolm_qwen_b200 import abi
    hq, hkv, hd, page = 4, 2, 64, 16
    B = Batch(rt, [2, 3, 1], [7, 40, 21], hq, hkv, hd, page, "f16", layers=2)
    B.batch = B.cache.batch(B.pages, B.q_start, B.kv_len, 6, 6, B.cfg.max_seq_len)
    B.fill(0, upto=B.past)
    pools = B.cache.k_pool, B.cache.v_pool
    before = [p.clone() for p in pools]
    q, k, v = B.rand(6, hq, hd), B.rand(6, hkv, hd), B.rand(6, hkv, hd)
    w = (1 + 0.1 * B.rand(hd), 1 + 0.1 * B.rand(hd)) if norm else (None, None)
    tab = table(B.cfg.max_seq_len, hd)
    good = torch.empty((6, hq, hd), device="cuda").half()
    B.cache.append(0, B.batch, q, k, v, *tab, good, *w)
    assert B.batch.status() == 0
    full = [p.clone() for p in pools]
    for p, old in zip(pools, before):
        p.copy_(old)
    B.q_start.copy_(torch.tensor(spans, dtype=torch.int64).to(torch.int32))
    area = torch.full((8, hq, hd), 7.0, device="cuda").half()
    B.cache.append(0, B.batch, q, k, v, *tab, area[1:7], *w)
    ok = [0 <= a <= e <= 6 and e - a <= t for a, e, t in zip(spans, spans[1:], B.total)]
    assert B.batch.status() == (0 if all(ok) else abi.DEV_BAD_POS)
    assert (area[[0, 7]] == 7).all()
    same_as_good = spans[:2] == [0, 2], spans[1:3] == [2, 5], spans[2:4] == [5, 6]
    for t in range(6):
        b = 0 if t < 2 else (1 if t < 5 else 2)
        y = area[1 + t]
        if all(ok) or (same_as_good[b] and spans == sorted(spans)):
            assert torch.equal(y, good[t])
        else:  # of another span, of a bad one, of none
            assert y.isfinite().all() if not y.isnan().any() else y.isnan().all()
    for p, old, new in zip(pools, before, full):
        same = ((p == old) | (p.isnan() & old.isnan())).all(-1)
        changed = {(i, g, r) for i, g, h, r in (~same).nonzero().tolist()}
        mine = {(0, int(B.pages[b, r // page]), r % page) for b in range(3) if ok[b]
                for r in range(B.total[b] - (spans[b + 1] - spans[b]), B.total[b])}
        assert changed <= mine
        if all(ok):
            assert changed == mine and torch.equal(p.view(torch.int16), new.view(torch.int16))


@pytest.mark.parametrize("wtype", ["F16", "Q8_0", "Q4_K"])
def test_a_layer_of_the_librarys_own_projections(rt, wtype):  # noqa: F811
    """matvec -> append -> attend -> matvec, as a host with a paged cache runs a layer, beside decode_layer on the same rows in
    slabs.  Both are within 2e-3 + 1e-2 |x| of the reference's chain by the tests of decode_layer (rows and outputs to
    fp32 rounding of the projections, one step of fp16 in the new cache rows)."""
    from picolm_qwen_b200 import abi
    from tests import weightgen as wg
    hq, hkv, hd, dim, page = 16, 4, 64, 1024, 16
    past = [0, 76, 599]
    t = {v: k for k, v in wg.NAMES.items()}[wtype]
    rng = np.random.default_rng(8)
    B = Batch(rt, [1, 1, 1], past, hq, hkv, hd, page, "f16", layers=2)
    B.fill(1, upto=past)
    st = rt.AttnState(B.cfg, n_seqs=3, max_ctx=B.cfg.max_seq_len)
    for b, n in enumerate(past):
        for pool, slab in ((B.cache.k_pool, st.k_cache), (B.cache.v_pool, st.v_cache)):
            slab[b, 1, :n] = B.rows(pool, 1, b, n).reshape(n, hkv * hd).view(torch.int16)
    shapes = ((dim, hq * hd), (dim, hkv * hd), (dim, hkv * hd), (hq * hd, dim))
    w = [torch.from_numpy(wg.make(t, n_in, n_out, rng)).cuda() for n_in, n_out in shapes]
    bias = [0.1 * B.rand(n_out) for _, n_out in shapes]
    proj = rt.LayerProj(*w, (t,) * 4, *bias)
    xb, x = B.rand(3, dim), B.rand(3, dim)
    slab_x = x.clone()
    st.decode_layer(1, dim, xb, proj, torch.tensor(past, dtype=torch.int32, device="cuda"), slab_x)
    q, k, v = (torch.empty((3, n_out), device="cuda") for _, n_out in shapes[:3])
    for y, wy, by, (n_in, n_out) in zip((q, k, v), w, bias, shapes):
        rt.matvec(wy, t, n_in, n_out, xb, y, by)
    qo, out = torch.empty((3, hq * hd), device="cuda").half(), torch.empty((3, hq * hd), device="cuda")
    B.cache.append(1, B.batch, q, k, v, st.rope_cos, st.rope_sin, qo)
    B.cache.attend(1, B.batch, qo, out)
    rt.matvec(w[3], t, hq * hd, dim, out, x, bias[3], accumulate=True)
    assert B.batch.status() == 0 and st.status() == 0
    assert ((x - slab_x).abs() <= 2 * (2e-3 + 1e-2 * slab_x.abs())).all()
    for b, n in enumerate(past):
        for pool, slab in ((B.cache.k_pool, st.k_cache), (B.cache.v_pool, st.v_cache)):
            a, e = B.rows(pool, 1, b, n + 1)[n].reshape(-1).view(torch.int16).int(), slab[b, 1, n].int()
            assert (a - e).abs().max() <= 1
