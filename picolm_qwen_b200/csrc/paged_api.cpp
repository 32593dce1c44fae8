// paged_api.cpp -- the extern "C" boundary of the rotary and paged-cache entries
// declared in include/picoattn.h: argument checks and dispatch.
#include <cmath>
#include <cstdint>

#include <cuda_runtime.h>

#include "paged_internal.h"
#include "picoattn.h"

using namespace picoattn;

namespace {

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

size_t elem_size(int32_t dtype) { return dtype == PICOATTN_DTYPE_F32 ? 4 : 2; }

bool dtype_ok(int32_t d) {
    return d == PICOATTN_DTYPE_F32 || d == PICOATTN_DTYPE_F16 || d == PICOATTN_DTYPE_BF16;
}

bool mode_ok(int32_t m) { return m == PICOATTN_ROPE_NEOX || m == PICOATTN_ROPE_INTERLEAVED; }

// The bytes from the first to past the last element of n rows.
struct Extent {
    uintptr_t lo, hi;
};
Extent extent(const void* p, int64_t rows, int64_t stride, int64_t row_elems, size_t es) {
    return {(uintptr_t)p, (uintptr_t)p + (uintptr_t)((rows - 1) * stride + row_elems) * es};
}
bool overlap(const Extent& a, const Extent& b) { return a.lo < b.hi && b.lo < a.hi; }

// Whether two sets of rows share an element: apart, or rows of one common
// stride that interleave (heads of one projection's output), where their
// columns modulo the stride tell.
bool rows_overlap(const void* p, int64_t ps, int64_t pw, const void* q, int64_t qs, int64_t qw, int64_t n, size_t es) {
    if (!overlap(extent(p, n, ps, pw, es), extent(q, n, qs, qw, es))) return false;
    if (ps != qs || ps < pw || ps < qw) return true;
    const int64_t bytes = ps * (int64_t)es, pb = pw * (int64_t)es, qb = qw * (int64_t)es;
    int64_t d = ((intptr_t)q - (intptr_t)p) % bytes;
    if (d < 0) d += bytes;  // q's rows start d bytes into p's
    return d < pb || d + qb > bytes;
}

constexpr int64_t kMaxStride = int64_t(1) << 28;   // keeps n_tok * stride in bytes inside 64 bits

int32_t rope_rows(const picoattn_rope_rows_t* r, int32_t hd, int32_t n_tok, size_t es, RopeRows* out) {
    if (!r->x || !r->out || r->n_heads <= 0 || r->n_heads > (1 << 20)) return PICOATTN_EINVAL;
    const int64_t w = r->n_heads * hd;
    if (r->x_stride < 0 || r->x_stride > kMaxStride || r->out_stride < w || r->out_stride > kMaxStride)
        return PICOATTN_EINVAL;
    if (!aligned(r->x, es) || !aligned(r->out, es)) return PICOATTN_EINVAL;
    const bool in_place = r->x == r->out && (r->x_stride == r->out_stride || n_tok == 1);
    if (!in_place && rows_overlap(r->x, r->x_stride, w, r->out, r->out_stride, w, n_tok, es)) return PICOATTN_EINVAL;
    *out = {r->x, r->out, r->x_stride, r->out_stride, (int)r->n_heads};
    return PICOATTN_OK;
}

int32_t batch_check(const picoattn_config_t* cfg, const picoattn_paged_cache_t* c, const picoattn_paged_batch_t* b,
                    int32_t layer, const void* ws, size_t ws_bytes, PagedBatch* out) {
    const int32_t st = picoattn_paged_check(cfg, c);
    if (st != PICOATTN_OK) return st;
    if (!b || !b->page_table || !b->q_start || !b->kv_len) return PICOATTN_EINVAL;
    if (!aligned(b->page_table, 4) || !aligned(b->q_start, 4) || !aligned(b->kv_len, 4)) return PICOATTN_EINVAL;
    if (layer < 0 || layer >= cfg->n_layers) return PICOATTN_EINVAL;
    if (b->n_seqs <= 0 || b->n_tok <= 0 || b->max_new <= 0 || b->page_cols <= 0) return PICOATTN_EINVAL;
    // the kernels count heads of tokens in 32 bits
    if ((int64_t)b->n_tok * (cfg->n_heads + 2 * (int64_t)cfg->n_kv_heads) > INT32_MAX) return PICOATTN_EUNSUPPORTED;
    if (b->max_len <= 0 || b->max_len > cfg->max_seq_len || b->max_new > b->max_len ||
        b->max_len > (int64_t)b->page_cols * c->page_size)
        return PICOATTN_ERANGE;
    if (!ws || !aligned(ws, 16) || ws_bytes < picoattn_paged_workspace_size(cfg, b->n_seqs)) return PICOATTN_ENOSPACE;
    int shift = 4;
    while ((1 << shift) < c->page_size) shift++;
    *out = {b->n_seqs,    b->n_tok,     b->max_new, b->max_len, b->page_cols,
            c->n_pages,   c->page_size, shift,      b->page_table, b->q_start,
            b->kv_len,    reinterpret_cast<unsigned int*>(const_cast<void*>(ws))};
    return PICOATTN_OK;
}

size_t layer_elems(const picoattn_config_t* cfg, const picoattn_paged_cache_t* c) {
    return (size_t)c->n_pages * cfg->n_kv_heads * c->page_size * cfg->head_dim;
}

}  // namespace

extern "C" {

int32_t picoattn_rope_scaled_table(const picoattn_config_t* c, const picoattn_rope_scaling_t* sc, float* cos_out,
                                   float* sin_out) {
    if (!c || !sc || !cos_out || !sin_out || c->max_seq_len <= 0 || c->head_dim <= 0 || c->head_dim % 2)
        return PICOATTN_EINVAL;
    const int rot = sc->rot_dim ? sc->rot_dim : c->head_dim;
    if (rot < 2 || rot % 2 || rot > c->head_dim || !(c->rope_freq_base > 0.f) || !std::isfinite(c->rope_freq_base))
        return PICOATTN_EINVAL;
    if (sc->kind < PICOATTN_ROPE_SCALE_NONE || sc->kind > PICOATTN_ROPE_SCALE_BY_PARTS) return PICOATTN_EINVAL;
    if (!(sc->mscale > 0.f) || !std::isfinite(sc->mscale)) return PICOATTN_EINVAL;
    if (sc->kind != PICOATTN_ROPE_SCALE_NONE && !(sc->factor >= 1.f && std::isfinite(sc->factor))) return PICOATTN_EINVAL;
    if (sc->kind == PICOATTN_ROPE_SCALE_NTK && rot == 2) return PICOATTN_EINVAL;
    if (sc->kind == PICOATTN_ROPE_SCALE_BY_PARTS &&
        (sc->orig_ctx <= 0 || !(sc->low < sc->high) || !std::isfinite(sc->low) || !std::isfinite(sc->high)))
        return PICOATTN_EINVAL;
    const double factor = sc->factor;
    double base = c->rope_freq_base;
    if (sc->kind == PICOATTN_ROPE_SCALE_NTK) base *= std::pow(factor, (double)rot / (rot - 2));
    const int half = rot / 2;
    for (int i = 0; i < half; i++) {
        double f = std::pow(base, -2.0 * i / rot);
        if (sc->kind == PICOATTN_ROPE_SCALE_LINEAR) f /= factor;
        if (sc->kind == PICOATTN_ROPE_SCALE_BY_PARTS) {
            const double turns = sc->orig_ctx * f / 6.283185307179586476925;
            double w = (turns - sc->low) / ((double)sc->high - sc->low);
            w = w < 0 ? 0 : (w > 1 ? 1 : w);
            f = (1 - w) * f / factor + w * f;
        }
        for (int p = 0; p < c->max_seq_len; p++) {
            cos_out[(size_t)p * half + i] = (float)(sc->mscale * std::cos(p * f));
            sin_out[(size_t)p * half + i] = (float)(sc->mscale * std::sin(p * f));
        }
    }
    return PICOATTN_OK;
}

int32_t picoattn_rope(const picoattn_rope_args_t* r, void* workspace, size_t workspace_bytes,
                      picoattn_stream_t stream) {
    if (!r || !dtype_ok(r->dtype) || !mode_ok(r->rope_mode)) return PICOATTN_EINVAL;
    const int32_t hd = r->head_dim, n = r->n_tok;
    if (hd < 2 || hd % 2 || r->rot_dim < 2 || r->rot_dim % 2 || r->rot_dim > hd) return PICOATTN_EINVAL;
    if (hd > 1024) return PICOATTN_EUNSUPPORTED;
    if (n <= 0 || r->table_rows <= 0 || !r->pos || !r->rope_cos || !r->rope_sin) return PICOATTN_EINVAL;
    if (r->n_tensors != 1 && r->n_tensors != 2) return PICOATTN_EINVAL;
    if (!aligned(r->pos, 4) || !aligned(r->rope_cos, 4) || !aligned(r->rope_sin, 4)) return PICOATTN_EINVAL;
    const size_t es = elem_size(r->dtype);
    const picoattn_rope_rows_t &q = r->q, &k = r->k;
    RopeArgs a{};
    int32_t st = rope_rows(&q, hd, n, es, &a.t[0]);
    if (st == PICOATTN_OK && r->n_tensors == 2) st = rope_rows(&k, hd, n, es, &a.t[1]);
    if (st != PICOATTN_OK) return st;
    if (r->n_tensors == 2) {  // neither output may touch the other tensor
        const int64_t qw = q.n_heads * hd, kw = k.n_heads * hd;
        if (rows_overlap(q.out, q.out_stride, qw, k.out, k.out_stride, kw, n, es) ||
            rows_overlap(q.out, q.out_stride, qw, k.x, k.x_stride, kw, n, es) ||
            rows_overlap(k.out, k.out_stride, kw, q.x, q.x_stride, qw, n, es))
            return PICOATTN_EINVAL;
    }
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < kWsHeaderBytes) return PICOATTN_ENOSPACE;
    st = picoattn_device_check();
    if (st != PICOATTN_OK) return st;
    a.dtype = r->dtype, a.mode = r->rope_mode, a.hd = hd, a.rot = r->rot_dim, a.inverse = r->inverse ? 1 : 0;
    a.n_tok = n, a.table_rows = r->table_rows;
    a.pos = r->pos, a.cos_t = r->rope_cos, a.sin_t = r->rope_sin;
    a.status = static_cast<unsigned int*>(workspace);
    return cuda_status(launch_rope(a, (cudaStream_t)stream));
}

int32_t picoattn_paged_check(const picoattn_config_t* c, const picoattn_paged_cache_t* p) {
    if (!c || !p) return PICOATTN_EINVAL;
    if (c->n_layers <= 0 || c->n_heads <= 0 || c->n_kv_heads <= 0 || c->max_seq_len <= 0) return PICOATTN_EINVAL;
    if (c->n_heads % c->n_kv_heads != 0 || c->head_dim <= 0 || !mode_ok(c->rope_mode)) return PICOATTN_EINVAL;
    if (!(c->qk_norm_eps >= 0.f)) return PICOATTN_EINVAL;
    if (c->head_dim != 64 && c->head_dim != 128) return PICOATTN_EUNSUPPORTED;
    if (c->n_heads / c->n_kv_heads > 128 || c->n_heads > 4096) return PICOATTN_EUNSUPPORTED;
    if (p->n_pages <= 0 || !p->k || !p->v || !aligned(p->k, 16) || !aligned(p->v, 16)) return PICOATTN_EINVAL;
    if (p->dtype != PICOATTN_DTYPE_F16 && p->dtype != PICOATTN_DTYPE_BF16)
        return dtype_ok(p->dtype) ? PICOATTN_EUNSUPPORTED : PICOATTN_EINVAL;
    const int s = p->page_size;
    if (s <= 0) return PICOATTN_EINVAL;
    if (s != 16 && s != 32 && s != 64 && s != 128 && s != 256) return PICOATTN_EUNSUPPORTED;
    // rows of a layer's pool are addressed by 32-bit tensor coordinates
    if ((int64_t)p->n_pages * c->n_kv_heads * s > INT32_MAX) return PICOATTN_EUNSUPPORTED;
    return PICOATTN_OK;
}

size_t picoattn_paged_workspace_size(const picoattn_config_t* c, int32_t n_seqs) {
    if (!c || n_seqs <= 0 || c->n_heads <= 0 || c->n_kv_heads <= 0 || c->n_heads % c->n_kv_heads) return 0;
    if ((c->head_dim != 64 && c->head_dim != 128) || c->n_heads / c->n_kv_heads > 128) return 0;
    return paged_workspace_bytes(*c, n_seqs);
}

int32_t picoattn_paged_append(const picoattn_config_t* cfg, const picoattn_paged_cache_t* cache, int32_t layer,
                              const picoattn_paged_batch_t* batch, const picoattn_paged_append_args_t* r,
                              void* workspace, size_t workspace_bytes, picoattn_stream_t stream) {
    PagedAppendArgs a{};
    int32_t st = batch_check(cfg, cache, batch, layer, workspace, workspace_bytes, &a.b);
    if (st != PICOATTN_OK) return st;
    if (!r || !dtype_ok(r->in_dtype) || !r->k || !r->v || !r->rope_cos || !r->rope_sin ||
        (r->q == nullptr) != (r->q_out == nullptr) || (r->q_norm_w == nullptr) != (r->k_norm_w == nullptr))
        return PICOATTN_EINVAL;
    if (!aligned(r->rope_cos, 4) || !aligned(r->rope_sin, 4) || !aligned(r->q_norm_w, 4) || !aligned(r->k_norm_w, 4))
        return PICOATTN_EINVAL;
    if (r->rot_dim <= 0 || r->rot_dim % 2 || r->rot_dim > cfg->head_dim) return PICOATTN_EINVAL;
    if (r->rot_dim % 16) return PICOATTN_EUNSUPPORTED;
    const size_t es = elem_size(r->in_dtype);
    const int64_t qw = (int64_t)cfg->n_heads * cfg->head_dim, kw = (int64_t)cfg->n_kv_heads * cfg->head_dim;
    const int64_t n = batch->n_tok, per16 = 16 / (int64_t)es;
    auto rows_ok = [&](const void* p, int64_t stride) {
        return aligned(p, 16) && stride >= 0 && stride <= kMaxStride && stride % per16 == 0;
    };
    if ((r->q && !rows_ok(r->q, r->q_stride)) || !rows_ok(r->k, r->k_stride) || !rows_ok(r->v, r->v_stride))
        return PICOATTN_EINVAL;
    if (r->q_out) {
        if (!aligned(r->q_out, 16)) return PICOATTN_EINVAL;
        const Extent o = extent(r->q_out, n, qw, qw, 2);
        if (overlap(o, extent(r->q, n, r->q_stride, qw, es)) || overlap(o, extent(r->k, n, r->k_stride, kw, es)) ||
            overlap(o, extent(r->v, n, r->v_stride, kw, es)))
            return PICOATTN_EINVAL;
    }
    st = picoattn_device_check();
    if (st != PICOATTN_OK) return st;
    const size_t slab = layer * layer_elems(cfg, cache);
    a.hq = cfg->n_heads, a.hkv = cfg->n_kv_heads, a.hd = cfg->head_dim, a.rot = r->rot_dim, a.mode = cfg->rope_mode;
    a.in_dtype = r->in_dtype, a.cache_dtype = cache->dtype, a.eps = cfg->qk_norm_eps;
    a.q = r->q, a.k = r->k, a.v = r->v, a.qs = r->q_stride, a.ks = r->k_stride, a.vs = r->v_stride;
    a.qn_w = r->q_norm_w, a.kn_w = r->k_norm_w, a.cos_t = r->rope_cos, a.sin_t = r->rope_sin, a.q_out = r->q_out;
    a.k_pool = static_cast<uint16_t*>(cache->k) + slab, a.v_pool = static_cast<uint16_t*>(cache->v) + slab;
    return cuda_status(launch_paged_append(a, (cudaStream_t)stream));
}

int32_t picoattn_paged_attn(const picoattn_config_t* cfg, const picoattn_paged_cache_t* cache, int32_t layer,
                            const picoattn_paged_batch_t* batch, const void* q, int64_t q_stride, int32_t out_dtype,
                            void* out, void* workspace, size_t workspace_bytes, picoattn_stream_t stream) {
    PagedAttnArgs a{};
    int32_t st = batch_check(cfg, cache, batch, layer, workspace, workspace_bytes, &a.b);
    if (st != PICOATTN_OK) return st;
    if (!q || !out || !aligned(q, 16) || !aligned(out, 16)) return PICOATTN_EINVAL;
    if (!dtype_ok(out_dtype)) return PICOATTN_EINVAL;
    if (out_dtype != PICOATTN_DTYPE_F32 && out_dtype != cache->dtype) return PICOATTN_EUNSUPPORTED;
    const int64_t qw = (int64_t)cfg->n_heads * cfg->head_dim;
    if (q_stride < qw || q_stride > kMaxStride || q_stride % 8) return PICOATTN_EINVAL;
    // the chunk kernel's work list counts a head's blocks, their costs and the batch's blocks in 32 bits
    const int64_t per = 2 * (128 / (cfg->n_heads / cfg->n_kv_heads));
    const int64_t blocks = (batch->max_new + per - 1) / per, tiles = (batch->max_len + 127) / 128;
    if (blocks * (4 * tiles + 4) > INT32_MAX ||
        (batch->n_tok / per + (int64_t)batch->n_seqs) * cfg->n_kv_heads > INT32_MAX)
        return PICOATTN_EUNSUPPORTED;
    if (overlap(extent(out, batch->n_tok, qw, qw, elem_size(out_dtype)), extent(q, batch->n_tok, q_stride, qw, 2)))
        return PICOATTN_EINVAL;
    st = picoattn_device_check();
    if (st != PICOATTN_OK) return st;
    const size_t slab = layer * layer_elems(cfg, cache);
    a.hq = cfg->n_heads, a.hkv = cfg->n_kv_heads, a.g = a.hq / a.hkv, a.hd = cfg->head_dim;
    a.dtype = cache->dtype, a.out_dtype = out_dtype, a.qs = q_stride, a.q = q, a.out = out;
    a.k_pool = static_cast<const uint16_t*>(cache->k) + slab, a.v_pool = static_cast<const uint16_t*>(cache->v) + slab;
    a.ws = static_cast<uint8_t*>(workspace) + kWsHeaderBytes;
    return cuda_status(launch_paged_attn(a, (cudaStream_t)stream));
}

}  // extern "C"
