"""Device-side attention state: the B200 counterpart of the reference's RunState
attention buffers (key_cache/val_cache, rope_cos/rope_sin, cpp/model.hpp:158-174,
allocated in cpp/model.hpp:1003-1017), plus the call that replaces the inline
attention block of Model::forward (cpp/model.hpp:326-418).

PyTorch is used only to own device memory and streams; every computation is a
call into libpicoattn.so through the C ABI.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import abi


def rope_table(cfg: abi.Config) -> tuple[np.ndarray, np.ndarray]:
    """Host RoPE table built by the library exactly as the reference builds it."""
    half = cfg.head_dim // 2
    cos = np.empty((cfg.max_seq_len, half), np.float32)
    sin = np.empty((cfg.max_seq_len, half), np.float32)
    abi.check(abi.lib().picoattn_rope_table(C.byref(cfg), cos.ctypes.data, sin.ctypes.data), "rope_table")
    return cos, sin


def stream_handle(stream: torch.cuda.Stream | None = None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def matvec(w: torch.Tensor, w_type: int, n_in: int, n_out: int, x: torch.Tensor, out: torch.Tensor,
           bias: torch.Tensor | None = None, accumulate: bool = False,
           stream: torch.cuda.Stream | None = None) -> None:
    """out[v] (=|+=) W . x[v] (+ bias) on the device (TensorOps::matmul_bias,
    cpp/tensor.hpp:110-143); w holds the GGUF blocks as uint8."""
    n_vec = x.numel() // n_in
    st = abi.lib().picoattn_matvec(w.data_ptr(), w_type, abi.ptr(bias), n_in, n_out, n_vec, x.data_ptr(),
                                   out.data_ptr(), 1 if accumulate else 0, stream_handle(stream))
    abi.check(st, "picoattn_matvec")


class LayerProj:
    """One layer's q/k/v/o weights on the device (uint8 GGUF blocks) and fp32 biases."""

    def __init__(self, wq, wk, wv, wo, types, bq=None, bk=None, bv=None, bo=None):
        self.tensors = (wq, wk, wv, wo, bq, bk, bv, bo)  # kept alive with the struct
        self.struct = abi.LayerWeights(
            wq.data_ptr(), wk.data_ptr(), wv.data_ptr(), wo.data_ptr(), *types,
            abi.ptr(bq), abi.ptr(bk), abi.ptr(bv), abi.ptr(bo))


class FfnProj:
    """One layer's FFN weights on the device (uint8 GGUF blocks) and fp32 biases."""

    def __init__(self, w_gate, w_up, w_down, types, b_gate=None, b_down=None):
        self.tensors = (w_gate, w_up, w_down, b_gate, b_down)  # kept alive with the struct
        self.struct = abi.FfnWeights(w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), *types,
                                     abi.ptr(b_gate), abi.ptr(b_down))


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, stream: torch.cuda.Stream | None = None):
    """out = rmsnorm(x) * weight per row of x [n_vec, dim] (TensorOps::rmsnorm, cpp/tensor.hpp:146-176)."""
    dim = weight.numel()
    abi.check(abi.lib().picoattn_rmsnorm(x.data_ptr(), weight.data_ptr(), out.data_ptr(), dim, x.numel() // dim,
                                         stream_handle(stream)), "picoattn_rmsnorm")


class Scratch:
    """A grow-only device byte buffer for the calls that take a workspace."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.buf = None

    def get(self, n: int) -> torch.Tensor:
        if self.buf is None or self.buf.numel() < n:
            self.buf = torch.zeros(max(n, 256), dtype=torch.uint8, device=self.device)
        return self.buf


def ffn(proj: "FfnProj", ffn_norm_w: torch.Tensor, n_ffn: int, x: torch.Tensor, scratch: "Scratch",
        stream: torch.cuda.Stream | None = None) -> None:
    """The FFN block and its residual in place on x [n_vec, dim] (cpp/model.hpp:429-452)."""
    dim = ffn_norm_w.numel()
    n_vec = x.numel() // dim
    n = abi.lib().picoattn_ffn_workspace_size(dim, n_ffn, n_vec)
    ws = scratch.get(n)
    abi.check(abi.lib().picoattn_ffn(C.byref(proj.struct), ffn_norm_w.data_ptr(), dim, n_ffn, n_vec, x.data_ptr(),
                                     ws.data_ptr(), ws.numel(), stream_handle(stream)), "picoattn_ffn")


def logits(x: torch.Tensor, output_norm_w: torch.Tensor, w_out: torch.Tensor, w_type: int, vocab: int,
           out: torch.Tensor, scratch: "Scratch", stream: torch.cuda.Stream | None = None) -> None:
    """out [n_vec, vocab] = W_out . rmsnorm(x) (cpp/model.hpp:454-457)."""
    dim = output_norm_w.numel()
    n_vec = x.numel() // dim
    ws = scratch.get(abi.lib().picoattn_logits_workspace_size(dim, n_vec))
    abi.check(abi.lib().picoattn_logits(x.data_ptr(), output_norm_w.data_ptr(), w_out.data_ptr(), w_type, dim, vocab,
                                        n_vec, out.data_ptr(), ws.data_ptr(), ws.numel(), stream_handle(stream)),
              "picoattn_logits")


_DTYPES = {torch.float32: abi.DTYPE_F32, torch.float16: abi.DTYPE_F16, torch.bfloat16: abi.DTYPE_BF16}

# the current stream's handle without building a Stream object, where this torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _dtype(t: torch.Tensor) -> int:
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise TypeError(f"dtype {t.dtype}: float32, float16 or bfloat16")
    return d


def _heads(t: torch.Tensor, n: int, heads: int, hd: int, what: str) -> int:
    """The row stride of t, [n, heads, hd] or [n, heads*hd], each row's heads contiguous (one row's may be any number)."""
    shape, st = t.shape, t.stride()
    if len(shape) == 3:
        if shape == (n, heads, hd) and st[2] == 1 and (st[1] == hd or heads == 1):
            return st[0] if n != 1 else heads * hd
    elif shape == (n, heads * hd) and st[1] == 1:
        return st[0] if n != 1 else heads * hd
    raise ValueError(f"{what}: [{n}, {heads}, {hd}] or [{n}, {heads * hd}] with contiguous rows, got {tuple(shape)} "
                     f"strides {st}")


def _check_table(cos: torch.Tensor, sin: torch.Tensor, rows: int) -> int:
    """rot_dim of a pair of tables."""
    shape = cos.shape
    if not (cos.dtype is torch.float32 and sin.dtype is torch.float32 and len(shape) == 2 and sin.shape == shape and
            shape[0] >= rows and cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"rope tables: contiguous fp32 [>= {rows}, rot_dim/2], got {tuple(shape)} {cos.dtype}, "
                         f"{tuple(sin.shape)} {sin.dtype}")
    return 2 * shape[1]


def _same_device(index: int, what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: a tensor on {t.device}, the others on device {index}")


def _stream(index: int, stream, what: str) -> int:
    """The handle of `stream` (None: the current one) of device `index`."""
    if index < 0:
        raise ValueError(f"{what}: tensors on the CPU")
    if stream is None:
        return _raw_stream(index)
    if stream.device_index != index:
        raise ValueError(f"{what}: a stream of device {stream.device_index}, tensors on device {index}")
    return stream.cuda_stream


def _launch(index: int, handle: int, what: str, call, *args) -> None:
    """call(*args, handle) with device `index` current (whichever the caller has), its error raised."""
    if torch.cuda.current_device() == index:
        st = call(*args, handle)
    else:
        with torch.cuda.device(index):
            st = call(*args, handle)
    if st:
        abi.check(st, what)


def status_workspace(device: str | torch.device = "cuda") -> torch.Tensor:
    """A workspace for calls that need only the status word (`rope`)."""
    return torch.zeros(256, dtype=torch.uint8, device=device)


def workspace_status(ws: torch.Tensor, stream: torch.cuda.Stream | None = None) -> int:
    """The sticky device status bits (abi.DEV_*) of a workspace, after the calls on `stream` (default: the current
    one); waits for that stream and clears them."""
    v = C.c_uint32(0)
    index = ws.get_device()
    _launch(index, _stream(index, stream, "workspace_status"), "workspace_status",
            lambda handle: abi.lib().picoattn_workspace_status(ws.data_ptr(), handle, C.byref(v)))
    return v.value


def rope_scaled_table(cfg: abi.Config, rot_dim: int = 0, kind: int = abi.ROPE_SCALE_NONE, factor: float = 1.0,
                      orig_ctx: int = 0, low: float = 1.0, high: float = 32.0,
                      mscale: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """Host RoPE tables [max_seq_len, rot_dim/2] for scaled contexts and partial heads."""
    half = (rot_dim or cfg.head_dim) // 2
    cos = np.empty((cfg.max_seq_len, half), np.float32)
    sin = np.empty((cfg.max_seq_len, half), np.float32)
    sc = abi.RopeScaling(rot_dim, kind, factor, orig_ctx, low, high, mscale)
    abi.check(abi.lib().picoattn_rope_scaled_table(C.byref(cfg), C.byref(sc), cos.ctypes.data, sin.ctypes.data),
              "picoattn_rope_scaled_table")
    return cos, sin


def rope(q: torch.Tensor, k: torch.Tensor | None, pos: torch.Tensor, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
         q_out: torch.Tensor, k_out: torch.Tensor | None, workspace: torch.Tensor,
         rope_mode: int = abi.ROPE_NEOX, inverse: bool = False, stream: torch.cuda.Stream | None = None) -> None:
    """q_out, k_out = q, k [n_tok, heads, head_dim] rotated by pos [n_tok] int32
    (the first 2 * rope_cos.shape[1] elements of each head); the outputs may be
    the inputs.  inverse: the opposite rotation, which is the backward pass."""
    n, heads, hd = q.shape
    dt, index = q.dtype, q.get_device()
    rot = _check_table(rope_cos, rope_sin, 1)
    if pos.dtype is not torch.int32 or pos.shape != (n,) or not pos.is_contiguous():
        raise ValueError(f"pos: contiguous int32 [{n}], got {tuple(pos.shape)} {pos.dtype}")
    if q_out.dtype is not dt or (k is None) != (k_out is None):
        raise ValueError("q_out: of q's type; k and k_out both or neither")
    _same_device(index, "rope", pos, rope_cos, rope_sin, q_out, k, k_out, workspace)
    rows = (q.data_ptr(), _heads(q, n, heads, hd, "q"), q_out.data_ptr(), _heads(q_out, n, heads, hd, "q_out"), heads)
    if k is None:
        krows = (0, 0, 0, 0, 0)
    else:
        kh = k.shape[1]
        if k.dtype is not dt or k_out.dtype is not dt:
            raise ValueError("k, k_out: of q's type")
        krows = (k.data_ptr(), _heads(k, n, kh, hd, "k"), k_out.data_ptr(), _heads(k_out, n, kh, hd, "k_out"), kh)
    _launch(index, _stream(index, stream, "rope"), "picoattn_rope", abi.lib().picoattn_rope,
            abi.ROPE_ARGS.pack(_dtype(q), rope_mode, hd, rot, 1 if inverse else 0, n, rope_cos.shape[0],
                               1 if k is None else 2, pos.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(),
                               *rows, *krows),
            workspace.data_ptr(), workspace.numel())


class PagedBatch:
    """The sequences of one step (picoattn_paged_batch_t) with the workspace its calls use.

    page_table [n_seqs, page_cols], q_start [n_seqs+1], kv_len [n_seqs]: int32 on the
    cache's device; their values may change between calls (a captured step reads
    them when it is replayed).  n_tok: rows of q, k, v and out; max_new, max_len:
    bounds on a sequence's new tokens and rows.  Steps that may run at the same
    time need batches of their own.  The workspace's header is cleared on the
    current stream; a step on another one waits for that first."""

    def __init__(self, cache: "PagedCache", page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                 n_tok: int, max_new: int, max_len: int):
        n = kv_len.numel()
        for name, t, shape in (("page_table", page_table, (n, page_table.shape[-1])), ("q_start", q_start, (n + 1,)),
                               ("kv_len", kv_len, (n,))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name}: contiguous int32 {shape}, got {tuple(t.shape)} {t.dtype}")
        _same_device(cache.index, "batch", page_table, q_start, kv_len)
        self.index = cache.index
        self.tensors = (page_table, q_start, kv_len)  # kept alive with the struct
        self.n_tok = n_tok
        self.desc = abi.PagedBatchDesc(n, n_tok, max_new, max_len, page_table.shape[1], page_table.data_ptr(),
                                       q_start.data_ptr(), kv_len.data_ptr())
        ws = abi.lib().picoattn_paged_workspace_size(C.byref(cache.cfg), n)
        if ws == 0:
            raise abi.PicoAttnError(abi.PICOATTN_EUNSUPPORTED, "paged_workspace_size")
        self.workspace = torch.empty(ws, dtype=torch.uint8, device=cache.device)
        self.workspace[:256].zero_()  # its header
        self.ref, self.ws_ptr, self.ws_bytes = C.addressof(self.desc), self.workspace.data_ptr(), ws
        # streams that the allocator knows the workspace to be used on
        self.streams = {_raw_stream(self.index)} if self.index >= 0 else set()

    def stream(self, stream: torch.cuda.Stream | None, what: str) -> int:
        """The handle of a call's stream.  Where it is not the batch's own, the batch's memory is not handed out again
        before the call is through, even if the batch is dropped."""
        handle = _stream(self.index, stream, what)
        if handle not in self.streams:
            s = torch.cuda.current_stream(self.index) if stream is None else stream
            for t in (self.workspace, *self.tensors):
                t.record_stream(s)
            self.streams.add(handle)
        return handle

    def status(self, stream: torch.cuda.Stream | None = None) -> int:
        """workspace_status of the batch: `stream` is the one that its calls ran on."""
        return workspace_status(self.workspace, stream)


class PagedCache:
    """Keys and values of many sequences in pages [n_layers, n_pages, n_kv_heads,
    page_size, head_dim] (fp16 or bf16): append a ragged batch's new tokens and
    attend over them.  The caller deals the pages out (PagedBatch.page_table)."""

    def __init__(self, cfg: abi.Config, page_size: int, n_pages: int | None = None,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda",
                 k_pool: torch.Tensor | None = None, v_pool: torch.Tensor | None = None):
        if k_pool is None:
            shape = (cfg.n_layers, n_pages, cfg.n_kv_heads, page_size, cfg.head_dim)
            k_pool = torch.zeros(shape, dtype=dtype, device=device)
            v_pool = torch.zeros(shape, dtype=dtype, device=device)
        want = (cfg.n_layers, k_pool.shape[1], cfg.n_kv_heads, page_size, cfg.head_dim)
        for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
            if tuple(t.shape) != want or t.dtype != k_pool.dtype or not t.is_contiguous():
                raise ValueError(f"{name}: contiguous {want}, got {tuple(t.shape)} {t.dtype}")
        self.cfg, self.k_pool, self.v_pool, self.device = cfg, k_pool, v_pool, k_pool.device
        self.index = k_pool.get_device()
        _same_device(self.index, "PagedCache", v_pool)
        self.dtype = k_pool.dtype
        self.desc = abi.PagedCacheDesc(k_pool.shape[1], page_size, _dtype(k_pool), k_pool.data_ptr(),
                                       v_pool.data_ptr())
        self.cfg_ref, self.ref = C.addressof(cfg), C.addressof(self.desc)
        self.shape = (cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, cfg.max_seq_len)
        abi.check(abi.lib().picoattn_paged_check(C.byref(cfg), C.byref(self.desc)), "picoattn_paged_check")

    def batch(self, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, n_tok: int, max_new: int,
              max_len: int) -> PagedBatch:
        return PagedBatch(self, page_table, q_start, kv_len, n_tok, max_new, max_len)

    def append(self, layer: int, batch: PagedBatch, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
               rope_cos: torch.Tensor, rope_sin: torch.Tensor, q_out: torch.Tensor | None,
               q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> None:
        """k, v [n_tok, n_kv_heads, head_dim] into their pages, q [n_tok, n_heads,
        head_dim] rotated into q_out (of the cache's type); the first
        2 * rope_cos.shape[1] elements of each head rotate."""
        n, dt = batch.n_tok, k.dtype
        hq, hkv, hd, max_rows = self.shape
        rot = _check_table(rope_cos, rope_sin, max_rows)
        if v.dtype is not dt or (q is None) != (q_out is None):
            raise ValueError("q, k, v of one type; q and q_out both or neither")
        q_ptr = q_stride = out_ptr = 0
        if q is not None:
            if q.dtype is not dt or q_out.dtype is not self.dtype or not q_out.is_contiguous():
                raise ValueError(f"q of k's type, q_out contiguous {self.dtype}, got {q.dtype}, {q_out.dtype}")
            q_ptr, q_stride, out_ptr = q.data_ptr(), _heads(q, n, hq, hd, "q"), q_out.data_ptr()
            _heads(q_out, n, hq, hd, "q_out")
        qn = kn = 0
        if q_norm_w is not None or k_norm_w is not None:
            for w in (q_norm_w, k_norm_w):
                if w is None or w.dtype is not torch.float32 or w.numel() != hd or not w.is_contiguous():
                    raise ValueError(f"norm weights: both, contiguous fp32 [{hd}]")
            qn, kn = q_norm_w.data_ptr(), k_norm_w.data_ptr()
        _same_device(self.index, "append", q, k, v, rope_cos, rope_sin, q_out, q_norm_w, k_norm_w)
        if batch.index != self.index:
            raise ValueError(f"append: a batch on device {batch.index}, the cache on device {self.index}")
        _launch(self.index, batch.stream(stream, "append"), "picoattn_paged_append", abi.lib().picoattn_paged_append, self.cfg_ref, self.ref,
                layer, batch.ref,
                abi.PAGED_APPEND_ARGS.pack(_dtype(k), rot, q_ptr, q_stride, k.data_ptr(), _heads(k, n, hkv, hd, "k"),
                                           v.data_ptr(), _heads(v, n, hkv, hd, "v"), qn, kn, rope_cos.data_ptr(),
                                           rope_sin.data_ptr(), out_ptr),
                batch.ws_ptr, batch.ws_bytes)

    def attend(self, layer: int, batch: PagedBatch, q: torch.Tensor, out: torch.Tensor,
               stream: torch.cuda.Stream | None = None) -> None:
        """out [n_tok, n_heads, head_dim] (the cache's type or fp32) = causal attention
        of the rotated queries q (the cache's type) over their sequences' rows."""
        n = batch.n_tok
        hq, _, hd, _ = self.shape
        if q.dtype is not self.dtype or not out.is_contiguous():
            raise ValueError(f"q: {self.dtype}, out: contiguous; got {q.dtype}, strides {out.stride()}")
        _heads(out, n, hq, hd, "out")
        _same_device(self.index, "attend", q, out)
        if batch.index != self.index:
            raise ValueError(f"attend: a batch on device {batch.index}, the cache on device {self.index}")
        _launch(self.index, batch.stream(stream, "attend"), "picoattn_paged_attn", abi.lib().picoattn_paged_attn, self.cfg_ref, self.ref,
                layer, batch.ref, q.data_ptr(), _heads(q, n, hq, hd, "q"), _dtype(out), out.data_ptr(), batch.ws_ptr,
                batch.ws_bytes)


class AttnState:
    """KV caches of n_seqs sequences in the reference layout plus RoPE tables.

    k_cache/v_cache: int16 tensors [n_seqs, n_layers, max_seq_len, kv_dim]
    (fp16 bit patterns; int16 is only the container type).
    """

    def __init__(self, cfg: abi.Config, n_seqs: int = 1, device: str | torch.device = "cuda",
                 max_ctx: int | None = None, rope: tuple[np.ndarray, np.ndarray] | None = None):
        self.cfg = cfg
        self.n_seqs = n_seqs
        self.device = torch.device(device)
        shape = (n_seqs, cfg.n_layers, cfg.max_seq_len, cfg.kv_dim)
        self.k_cache = torch.zeros(shape, dtype=torch.int16, device=self.device)
        self.v_cache = torch.zeros(shape, dtype=torch.int16, device=self.device)
        cos, sin = rope if rope is not None else rope_table(cfg)
        self.rope_cos = torch.from_numpy(cos).to(self.device)
        self.rope_sin = torch.from_numpy(sin).to(self.device)
        per = cfg.n_layers * cfg.max_seq_len * cfg.kv_dim * 2
        kb, vb = self.k_cache.data_ptr(), self.v_cache.data_ptr()
        self.k_ptrs = torch.tensor([kb + i * per for i in range(n_seqs)], dtype=torch.int64, device=self.device)
        self.v_ptrs = torch.tensor([vb + i * per for i in range(n_seqs)], dtype=torch.int64, device=self.device)
        self.max_ctx = max_ctx if max_ctx is not None else cfg.max_seq_len
        ws = abi.lib().picoattn_decode_workspace_size(C.byref(cfg), n_seqs, self.max_ctx)
        if ws == 0:
            raise abi.PicoAttnError(abi.PICOATTN_EUNSUPPORTED, "decode_workspace_size")
        self.workspace = torch.zeros(ws, dtype=torch.uint8, device=self.device)
        abi.check(abi.lib().picoattn_workspace_init(self.workspace.data_ptr(), ws, stream_handle()), "ws init")

    # -- the call that replaces cpp/model.hpp:326-418 ---------------------------
    def decode(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor,
               out: torch.Tensor, q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
               max_ctx: int | None = None, stream: torch.cuda.Stream | None = None) -> None:
        """q [B, Hq*hd], k/v [B, kvd] fp32, pos [B] int32 (device), out [B, Hq*hd] fp32."""
        B = q.shape[0]
        st = abi.lib().picoattn_decode(
            C.byref(self.cfg), layer, B, max_ctx if max_ctx is not None else self.max_ctx,
            q.data_ptr(), k.data_ptr(), v.data_ptr(), abi.ptr(q_norm_w), abi.ptr(k_norm_w),
            self.rope_cos.data_ptr(), self.rope_sin.data_ptr(), self.k_ptrs.data_ptr(), self.v_ptrs.data_ptr(),
            pos.data_ptr(), out.data_ptr(), self.workspace.data_ptr(), self.workspace.numel(),
            stream_handle(stream))
        abi.check(st, "picoattn_decode")

    def decode_layer(self, layer: int, dim: int, xb: torch.Tensor, proj: LayerProj, pos: torch.Tensor,
                     x: torch.Tensor, q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                     stream: torch.cuda.Stream | None = None) -> None:
        """The attention block from the normalised hidden state xb [B, dim] into
        the residual x [B, dim] (cpp/model.hpp:318-427): projections, decode step,
        output projection added to x."""
        B = xb.shape[0]
        if getattr(self, "layer_ws", None) is None or self.layer_ws_key != (dim, B):
            n = abi.lib().picoattn_decode_layer_workspace_size(C.byref(self.cfg), dim, B, self.max_ctx)
            if n == 0:
                raise abi.PicoAttnError(abi.PICOATTN_EUNSUPPORTED, "decode_layer_workspace_size")
            self.layer_ws = torch.zeros(n, dtype=torch.uint8, device=self.device)
            self.layer_ws_key = (dim, B)
            abi.check(abi.lib().picoattn_workspace_init(self.layer_ws.data_ptr(), n, stream_handle(stream)),
                      "ws init")
        st = abi.lib().picoattn_decode_layer(
            C.byref(self.cfg), layer, dim, B, self.max_ctx, xb.data_ptr(), C.byref(proj.struct),
            abi.ptr(q_norm_w), abi.ptr(k_norm_w), self.rope_cos.data_ptr(), self.rope_sin.data_ptr(),
            self.k_ptrs.data_ptr(), self.v_ptrs.data_ptr(), pos.data_ptr(), x.data_ptr(),
            self.layer_ws.data_ptr(), self.layer_ws.numel(), stream_handle(stream))
        abi.check(st, "picoattn_decode_layer")

    def decode_block(self, layer: int, dim: int, n_ffn: int, x: torch.Tensor, attn_norm_w: torch.Tensor,
                     proj: LayerProj, ffn_norm_w: torch.Tensor, ffn_proj: FfnProj, pos: torch.Tensor,
                     q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                     stream: torch.cuda.Stream | None = None) -> None:
        """One whole layer of the decode step on the residual x [B, dim] in place
        (cpp/model.hpp:315-452): attention norm, the attention block, the FFN block."""
        B = x.shape[0]
        key = (dim, n_ffn, B)
        if getattr(self, "block_ws", None) is None or self.block_ws_key != key:
            n = abi.lib().picoattn_decode_block_workspace_size(C.byref(self.cfg), dim, n_ffn, B, self.max_ctx)
            if n == 0:
                raise abi.PicoAttnError(abi.PICOATTN_EUNSUPPORTED, "decode_block_workspace_size")
            self.block_ws = torch.zeros(n, dtype=torch.uint8, device=self.device)
            self.block_ws_key = key
            abi.check(abi.lib().picoattn_workspace_init(self.block_ws.data_ptr(), n, stream_handle(stream)),
                      "ws init")
        st = abi.lib().picoattn_decode_block(
            C.byref(self.cfg), layer, dim, n_ffn, B, self.max_ctx, attn_norm_w.data_ptr(), C.byref(proj.struct),
            ffn_norm_w.data_ptr(), C.byref(ffn_proj.struct), abi.ptr(q_norm_w), abi.ptr(k_norm_w),
            self.rope_cos.data_ptr(), self.rope_sin.data_ptr(), self.k_ptrs.data_ptr(), self.v_ptrs.data_ptr(),
            pos.data_ptr(), x.data_ptr(), self.block_ws.data_ptr(), self.block_ws.numel(), stream_handle(stream))
        abi.check(st, "picoattn_decode_block")

    def block_status(self) -> int:
        v = C.c_uint32(0)
        abi.check(abi.lib().picoattn_workspace_status(self.block_ws.data_ptr(), stream_handle(), C.byref(v)))
        return v.value

    def decode_one(self, layer: int, pos: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   out: torch.Tensor, q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                   seq: int = 0, stream: torch.cuda.Stream | None = None) -> int:
        """Model::forward-shaped call: one sequence, host position.  Returns the status."""
        return abi.lib().picoattn_decode_one(
            C.byref(self.cfg), layer, pos, q.data_ptr(), k.data_ptr(), v.data_ptr(),
            abi.ptr(q_norm_w), abi.ptr(k_norm_w), self.rope_cos.data_ptr(), self.rope_sin.data_ptr(),
            self.k_cache[seq].data_ptr(), self.v_cache[seq].data_ptr(), out.data_ptr(),
            self.workspace.data_ptr(), self.workspace.numel(), stream_handle(stream))

    # -- KV-cache persistence in the C engine's KVCP format (picolm/model.c:870-983)
    def kvcp_save(self, path: str, n_pos: int, seq: int = 0, stream: torch.cuda.Stream | None = None) -> None:
        """Rows 0..n_pos-1 of every layer of sequence `seq` -> a KVCP file (kvcache_save)."""
        abi.check(abi.lib().picoattn_kvcp_save(C.byref(self.cfg), n_pos, self.k_cache[seq].data_ptr(),
                                               self.v_cache[seq].data_ptr(), path.encode(), stream_handle(stream)),
                  "picoattn_kvcp_save")

    def kvcp_load(self, path: str, seq: int = 0, stream: torch.cuda.Stream | None = None) -> int:
        """A KVCP file -> rows 0..n_pos-1 of sequence `seq`; returns n_pos, or 0 when
        the file is missing or does not fit this model (kvcache_load's contract)."""
        n = C.c_int32(0)
        st = abi.lib().picoattn_kvcp_load(C.byref(self.cfg), path.encode(), self.k_cache[seq].data_ptr(),
                                          self.v_cache[seq].data_ptr(), C.byref(n), stream_handle(stream))
        if st in (abi.PICOATTN_EIO, abi.PICOATTN_EFORMAT):
            return 0
        abi.check(st, "picoattn_kvcp_load")
        return n.value

    # -- the call that replaces cpp/model.hpp:493-593 (forward_batch) ------------
    def prefill(self, layer: int, start_pos: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                out: torch.Tensor, q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                seq: int = 0, workspace: torch.Tensor | None = None, stages: int = 0x3,
                stream: torch.cuda.Stream | None = None) -> int:
        """q [n, Hq*hd], k/v [n, kvd] fp32 or fp16 (device); out [n, Hq*hd] fp32.  Returns the status."""
        n = q.shape[0]
        dtype = abi.DTYPE_F16 if q.dtype == torch.float16 else abi.DTYPE_F32
        if workspace is None:
            workspace = self.prefill_workspace(n)
        return abi.lib().picoattn_prefill_staged(
            C.byref(self.cfg), layer, n, start_pos, dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(),
            abi.ptr(q_norm_w), abi.ptr(k_norm_w), self.rope_cos.data_ptr(), self.rope_sin.data_ptr(),
            self.k_cache[seq].data_ptr(), self.v_cache[seq].data_ptr(), out.data_ptr(),
            workspace.data_ptr(), workspace.numel(), stream_handle(stream), stages)

    def prefill_workspace(self, n_tok: int) -> torch.Tensor:
        n = abi.lib().picoattn_prefill_workspace_size(C.byref(self.cfg), n_tok)
        if n == 0:
            raise abi.PicoAttnError(abi.PICOATTN_EUNSUPPORTED, "prefill_workspace_size")
        ws = getattr(self, "_pf_ws", None)
        if ws is None or ws.numel() < n:
            ws = torch.zeros(n, dtype=torch.uint8, device=self.device)
            self._pf_ws = ws
        return ws

    def status(self) -> int:
        v = C.c_uint32(0)
        abi.check(abi.lib().picoattn_workspace_status(self.workspace.data_ptr(), stream_handle(), C.byref(v)))
        return v.value
