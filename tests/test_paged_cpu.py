"""Argument checks of the rotary and paged-cache entries, and the scaled RoPE tables, on the host: no GPU is used.

A call that passes every check goes on to the device check, so on a host without a GPU an accepted call returns
PICOATTN_EDEVICE or PICOATTN_ECUDA and a refused one its own status.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from picolm_qwen_b200 import abi

if torch.cuda.is_available():  # accepted calls would launch on the made-up addresses below
    pytest.skip("host-only checks", allow_module_level=True)

L = abi.lib()
ACCEPTED = (abi.PICOATTN_EDEVICE, abi.PICOATTN_ECUDA)
A = 0x100000  # made-up addresses, far apart, never dereferenced
ADDR = {n: A + (i << 32) for i, n in enumerate(
    ["q", "k", "v", "q_out", "k_out", "out", "kp", "vp", "table", "start", "len", "cos", "sin", "ws", "pos", "qn", "kn"])}


def cfg(**kw):
    base = dict(n_layers=2, n_heads=28, n_kv_heads=4, head_dim=128, max_seq_len=1024, rope_freq_base=1e6,
                rope_mode=abi.ROPE_NEOX, qk_norm_eps=1e-6)
    base.update(kw)
    return abi.Config(**base)


def cache(**kw):
    d = dict(n_pages=100, page_size=16, dtype=abi.DTYPE_F16, k=ADDR["kp"], v=ADDR["vp"])
    d.update(kw)
    return abi.PagedCacheDesc(*[d[n] for n, _ in abi.PagedCacheDesc._fields_])


def batch(**kw):
    d = dict(n_seqs=3, n_tok=10, max_new=4, max_len=1024, page_cols=64, page_table=ADDR["table"], q_start=ADDR["start"],
             kv_len=ADDR["len"])
    d.update(kw)
    return abi.PagedBatchDesc(*[d[n] for n, _ in abi.PagedBatchDesc._fields_])


def rope(dtype=abi.DTYPE_F16, mode=0, hd=64, rot=64, n=5, rows=100, q=None, k=None, ws_bytes=256, **over):
    p = dict(pos=ADDR["pos"], cos=ADDR["cos"], sin=ADDR["sin"], ws=ADDR["ws"])
    p.update(over)
    q = q or abi.RopeRows(ADDR["q"], 8 * 64, ADDR["q_out"], 8 * 64, 8)
    args = abi.RopeArgs(dtype, mode, hd, rot, 0, n, rows, over.get("tensors", 2 if k else 1), p["pos"], p["cos"],
                        p["sin"], q, k or abi.RopeRows())
    return L.picoattn_rope(C.byref(args), p["ws"], ws_bytes, None)


def append(c=None, ca=None, b=None, layer=0, dtype=abi.DTYPE_F16, rot=128, ws_bytes=1 << 30, **over):
    p = dict(q=ADDR["q"], qs=28 * 128, k=ADDR["k"], ks=512, v=ADDR["v"], vs=512, qn=None, kn=None, cos=ADDR["cos"],
             sin=ADDR["sin"], q_out=ADDR["q_out"], ws=ADDR["ws"])
    p.update(over)
    args = abi.PagedAppendArgs(dtype, rot, p["q"], p["qs"], p["k"], p["ks"], p["v"], p["vs"], p["qn"], p["kn"],
                               p["cos"], p["sin"], p["q_out"])
    return L.picoattn_paged_append(C.byref(c or cfg()), C.byref(ca or cache()), layer, C.byref(b or batch()),
                                   C.byref(args), p["ws"], ws_bytes, None)


def attn(c=None, ca=None, b=None, layer=0, out_dtype=abi.DTYPE_F16, ws_bytes=1 << 30, **over):
    p = dict(q=ADDR["q"], qs=28 * 128, out=ADDR["out"], ws=ADDR["ws"])
    p.update(over)
    return L.picoattn_paged_attn(C.byref(c or cfg()), C.byref(ca or cache()), layer, C.byref(b or batch()), p["q"],
                                 p["qs"], out_dtype, p["out"], p["ws"], ws_bytes, None)


def test_accepted_calls_reach_the_device_check():
    assert rope() in ACCEPTED
    assert append() in ACCEPTED
    assert append(q=None, q_out=None) in ACCEPTED
    assert append(qn=ADDR["qn"], kn=ADDR["kn"], rot=16) in ACCEPTED
    assert attn() in ACCEPTED
    assert attn(out_dtype=abi.DTYPE_F32) in ACCEPTED
    # shapes the contiguous entries do not take
    assert attn(c=cfg(n_heads=9, n_kv_heads=3, head_dim=64), qs=9 * 64) in ACCEPTED
    assert attn(c=cfg(n_heads=71, n_kv_heads=1, head_dim=64), qs=71 * 64) in ACCEPTED


INV, UNS, RNG, SPACE = abi.PICOATTN_EINVAL, abi.PICOATTN_EUNSUPPORTED, abi.PICOATTN_ERANGE, abi.PICOATTN_ENOSPACE


@pytest.mark.parametrize("kw,want", [
    (dict(dtype=7), INV), (dict(mode=2), INV), (dict(hd=63), INV), (dict(rot=0), INV), (dict(rot=66), INV),
    (dict(rot=31), INV), (dict(hd=2048, rot=2048), UNS), (dict(n=0), INV), (dict(rows=0), INV), (dict(pos=None), INV),
    (dict(pos=ADDR["pos"] + 2), INV), (dict(cos=None), INV), (dict(sin=ADDR["sin"] + 1), INV),
    (dict(ws=None), SPACE), (dict(ws_bytes=255), SPACE), (dict(ws=ADDR["ws"] + 4), SPACE),
    (dict(q=abi.RopeRows(None, 512, ADDR["q_out"], 512, 8)), INV),
    (dict(q=abi.RopeRows(ADDR["q"], 512, ADDR["q_out"], 511, 8)), INV),          # output rows overlap
    (dict(q=abi.RopeRows(ADDR["q"], -1, ADDR["q_out"], 512, 8)), INV),
    (dict(q=abi.RopeRows(ADDR["q"] + 1, 512, ADDR["q_out"], 512, 8)), INV),      # not element aligned
    (dict(q=abi.RopeRows(ADDR["q"], 512, ADDR["q"] + 64, 512, 8)), INV),         # overlaps, not in place
    (dict(q=abi.RopeRows(ADDR["q"], 512, ADDR["q"], 1024, 8)), INV),             # same start, other stride
    (dict(q=abi.RopeRows(ADDR["q"], 512, ADDR["q_out"], 512, 0)), INV),
    (dict(tensors=3), INV), (dict(tensors=2), INV),
    (dict(k=abi.RopeRows(ADDR["k"], 512, ADDR["q_out"], 512, 8)), INV),          # both outputs at one place
    (dict(k=abi.RopeRows(ADDR["q_out"], 512, ADDR["k_out"], 512, 8)), INV),      # q's output over k
])
def test_rope_refuses(kw, want):
    assert rope(**kw) == want


def test_rope_takes_interleaved_rows_of_one_projection_in_place():
    e = 2
    q = abi.RopeRows(ADDR["q"], 768, ADDR["q"], 768, 8)
    k = abi.RopeRows(ADDR["q"] + 512 * e, 768, ADDR["q"] + 512 * e, 768, 2)
    assert rope(q=q, k=k) in ACCEPTED
    k = abi.RopeRows(ADDR["q"] + 480 * e, 768, ADDR["q"] + 480 * e, 768, 2)  # k's heads begin inside q's
    assert rope(q=q, k=k) == INV


@pytest.mark.parametrize("kw,want", [
    (dict(c=cfg(n_heads=30)), INV), (dict(c=cfg(head_dim=96)), UNS), (dict(c=cfg(n_heads=129, n_kv_heads=1)), UNS),
    (dict(c=cfg(rope_mode=3)), INV), (dict(c=cfg(max_seq_len=0)), INV),
    (dict(ca=cache(page_size=24)), UNS), (dict(ca=cache(page_size=8)), UNS), (dict(ca=cache(page_size=512)), UNS),
    (dict(ca=cache(page_size=0)), INV), (dict(ca=cache(dtype=abi.DTYPE_F32)), UNS), (dict(ca=cache(dtype=9)), INV),
    (dict(ca=cache(n_pages=0)), INV), (dict(ca=cache(k=None)), INV), (dict(ca=cache(v=ADDR["vp"] + 8)), INV),
    (dict(ca=cache(n_pages=1 << 26)), UNS),
    (dict(b=batch(n_seqs=0)), INV), (dict(b=batch(n_tok=0)), INV), (dict(b=batch(max_new=0)), INV),
    (dict(b=batch(page_cols=0)), INV), (dict(b=batch(n_tok=1 << 27)), UNS), (dict(b=batch(page_table=None)), INV), (dict(b=batch(q_start=None)), INV),
    (dict(b=batch(kv_len=ADDR["len"] + 2)), INV),
    (dict(b=batch(max_len=1025)), RNG), (dict(b=batch(max_len=0)), RNG), (dict(b=batch(max_new=2000)), RNG),
    (dict(b=batch(page_cols=63)), RNG),
    (dict(layer=2), INV), (dict(layer=-1), INV), (dict(ws=None), SPACE), (dict(ws=ADDR["ws"] + 8), SPACE),
    (dict(ws_bytes=255), SPACE),
])
def test_paged_entries_refuse(kw, want):
    assert append(**kw) == want
    assert attn(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(dtype=5), INV), (dict(k=None), INV), (dict(v=None), INV), (dict(q=None), INV), (dict(q_out=None), INV),
    (dict(cos=None), INV), (dict(qn=ADDR["qn"]), INV), (dict(rot=0), INV), (dict(rot=130), INV), (dict(rot=24), UNS),
    (dict(q=ADDR["q"] + 8), INV), (dict(ks=516), INV), (dict(vs=-512), INV), (dict(q_out=ADDR["q_out"] + 2), INV),
    (dict(q_out=ADDR["q"] + 256), INV), (dict(q_out=ADDR["k"]), INV),
])
def test_append_refuses(kw, want):
    assert append(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), INV), (dict(out=None), INV), (dict(q=ADDR["q"] + 8), INV), (dict(out=ADDR["out"] + 4), INV),
    (dict(qs=28 * 128 - 8), INV), (dict(qs=28 * 128 + 4), INV), (dict(out_dtype=8), INV),
    (dict(out_dtype=abi.DTYPE_BF16), UNS), (dict(out=ADDR["q"]), INV),
])
def test_attn_refuses(kw, want):
    assert attn(**kw) == want


@pytest.mark.parametrize("kw,want", [
    # a head's blocks x key tiles past 32 bits: 2 tokens a block at 128 q heads per KV head, 36 at 7
    (dict(c=cfg(n_heads=128, n_kv_heads=1, max_seq_len=1 << 20), b=batch(n_tok=1 << 20, max_new=1 << 20, max_len=1 << 20,
                                                                        page_cols=1 << 16), qs=128 * 128), UNS),
    (dict(c=cfg(n_heads=128, n_kv_heads=1, max_seq_len=1 << 20), b=batch(n_tok=1 << 20, max_new=1 << 16, max_len=1 << 20,
                                                                        page_cols=1 << 16), qs=128 * 128,
          out=ADDR["q"] + (1 << 40)), None),
    (dict(b=batch(n_seqs=(1 << 29) + 1)), UNS),  # sequences x KV heads past 32 bits
])
def test_attn_refuses_what_its_work_list_cannot_count(kw, want):
    st = attn(**kw)
    assert st in ACCEPTED if want is None else st == want


def test_packed_arguments_have_the_structs_layout():
    """abi.ROPE_ARGS / PAGED_APPEND_ARGS pack what the C structs (and their ctypes forms) hold."""
    r = abi.RopeArgs(1, 0, 64, 32, 1, 7, 99, 2, 11, 12, 13, abi.RopeRows(21, 22, 23, 24, 25),
                     abi.RopeRows(31, 32, 33, 34, 35))
    assert bytes(r) == abi.ROPE_ARGS.pack(1, 0, 64, 32, 1, 7, 99, 2, 11, 12, 13, 21, 22, 23, 24, 25, 31, 32, 33, 34, 35)
    a = abi.PagedAppendArgs(2, 48, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11)
    assert bytes(a) == abi.PAGED_APPEND_ARGS.pack(2, 48, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11)


def test_workspace_size():
    assert L.picoattn_paged_workspace_size(C.byref(cfg()), 1) >= 256
    assert L.picoattn_paged_workspace_size(C.byref(cfg()), 0) == 0
    assert L.picoattn_paged_workspace_size(C.byref(cfg(head_dim=96)), 4) == 0


def scaled(c, **kw):
    d = dict(rot_dim=0, kind=abi.ROPE_SCALE_NONE, factor=1.0, orig_ctx=0, low=1.0, high=32.0, mscale=1.0)
    d.update(kw)
    sc = abi.RopeScaling(*[d[n] for n, _ in abi.RopeScaling._fields_])
    half = (d["rot_dim"] or c.head_dim) // 2
    cos, sin = np.full((c.max_seq_len, half), np.nan, np.float32), np.full((c.max_seq_len, half), np.nan, np.float32)
    return L.picoattn_rope_scaled_table(C.byref(c), C.byref(sc), cos.ctypes.data, sin.ctypes.data), cos, sin


@pytest.mark.parametrize("kw,freq", [
    (dict(), lambda f, i, r: f),
    (dict(rot_dim=32), lambda f, i, r: f),
    (dict(kind=1, factor=4.0), lambda f, i, r: f / 4),
    (dict(kind=2, factor=8.0, rot_dim=64), lambda f, i, r: (1e4 * 8 ** (r / (r - 2))) ** (-2 * i / r)),
    (dict(kind=3, factor=4.0, orig_ctx=2048, low=1.0, high=32.0, mscale=0.1 * math.log(4) + 1), None),
])
def test_scaled_table(kw, freq):
    c = cfg(max_seq_len=9000, rope_freq_base=1e4)
    st, cos, sin = scaled(c, **kw)
    assert st == abi.PICOATTN_OK
    rot = kw.get("rot_dim") or 128
    i = np.arange(rot // 2)
    f = 1e4 ** (-2 * i / rot)
    if freq is None:
        turns = 2048 * f / (2 * np.pi)
        w = np.clip((turns - 1) / 31, 0, 1)
        f = (1 - w) * f / 4 + w * f
        assert w[0] == 1 and w[-1] == 0  # fast pairs as they were, slow ones interpolated
    else:
        f = freq(f, i, rot)
    ms = np.float64(np.float32(kw.get("mscale", 1.0)))
    ang = np.arange(9000)[:, None] * f
    # angles below 9000 in 64 bits are off by 1e-12 at most; one rounding to fp32
    assert np.abs(cos - ms * np.cos(ang)).max() <= 2.0 ** -24 * ms + 1e-9
    assert np.abs(sin - ms * np.sin(ang)).max() <= 2.0 ** -24 * ms + 1e-9


@pytest.mark.parametrize("kw", [
    dict(rot_dim=3), dict(rot_dim=130), dict(kind=9), dict(kind=1, factor=0.5), dict(kind=1, factor=math.inf),
    dict(kind=2, factor=2.0, rot_dim=2), dict(kind=3, factor=2.0), dict(kind=3, factor=2.0, orig_ctx=10, low=3, high=3),
    dict(mscale=0.0), dict(mscale=math.nan),
])
def test_scaled_table_refuses(kw):
    assert scaled(cfg(max_seq_len=4), **kw)[0] == abi.PICOATTN_EINVAL
