// paged_attn.cu -- causal attention of a ragged batch's new tokens over a paged
// cache (picoattn_paged_attn): out = softmax(q K^T / sqrt(hd)) V over rows 0..pos.
#include <algorithm>
#include <cmath>

#include "paged_common.cuh"

namespace picoattn {

namespace {

// One warp per (token, q head), one cache row at a time, online softmax in the
// log2 domain: running maximum m, sum l and output o, rescaled when m grows.
template <class T, int HD>
__global__ void __launch_bounds__(128) paged_attn_rows_kernel(PagedAttnArgs a) {
    constexpr int E = HD / 32;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); u < (long long)a.b.n_tok * a.hq;
         u += (long long)gridDim.x * 4) {
        const int tok = (int)(u / a.hq), h = (int)(u % a.hq), kvh = h / a.g;
        int b = 0;
        while (b < a.b.n_seqs && a.b.q_start[b + 1] <= tok) b++;
        if (b >= a.b.n_seqs || tok < a.b.q_start[b]) continue;
        const SeqSpan sp = seq_span(a.b, b);
        float o[E], q[E], m = -INFINITY, l = 0.f;
        bool bad = !sp.ok;
        if (bad && lane == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_POS);
        for (int e = 0; e < E; e++) {
            o[e] = 0.f;
            q[e] = bad ? 0.f : Elem<T>::load(static_cast<const T*>(a.q) + tok * a.qs + h * HD + lane * E + e) * scale;
        }
        const int rows = bad ? 0 : sp.len - sp.n + (tok - sp.t0) + 1;
        for (int r = 0; r < rows; r++) {
            const int page = a.b.page_table[(size_t)b * a.b.page_cols + (r >> a.b.page_shift)];
            if (page < 0 || page >= a.b.n_pages) {
                if (lane == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_PAGE);
                bad = true;
                break;
            }
            const size_t at = (((size_t)page * a.hkv + kvh) * a.b.page_size + (r & (a.b.page_size - 1))) * HD + lane * E;
            float s = 0.f;
            for (int e = 0; e < E; e++) s += q[e] * Elem<T>::load(static_cast<const T*>(a.k_pool) + at + e);
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            const float mn = fmaxf(m, s), keep = ex2(m - mn), p = ex2(s - mn);
            m = mn;
            l = l * keep + p;
            for (int e = 0; e < E; e++) o[e] = o[e] * keep + p * Elem<T>::load(static_cast<const T*>(a.v_pool) + at + e);
        }
        for (int e = 0; e < E; e++) {
            const float y = bad ? __int_as_float(0x7fc00000) : o[e] / l;
            const size_t at = ((size_t)tok * a.hq + h) * HD + lane * E + e;
            if (a.out_dtype == PICOATTN_DTYPE_F32) static_cast<float*>(a.out)[at] = y;
            else static_cast<T*>(a.out)[at] = Elem<T>::round(y);
        }
    }
}

}  // namespace

size_t paged_workspace_bytes(const picoattn_config_t& cfg, int n_seqs) {
    return kWsHeaderBytes + paged_few_bytes(cfg.head_dim, n_seqs);
}

cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t stream) {
    if (paged_few_fits(a)) return launch_paged_few(a, stream);
    const unsigned grid = (unsigned)std::min<long long>(((long long)a.b.n_tok * a.hq + 3) / 4, 1 << 20);
    auto go = [&](auto kernel) { return launch_pdl(kernel, dim3(grid), dim3(128), 0, stream, a); };
    if (a.dtype == PICOATTN_DTYPE_F16)
        return a.hd == 64 ? go(paged_attn_rows_kernel<__half, 64>) : go(paged_attn_rows_kernel<__half, 128>);
    return a.hd == 64 ? go(paged_attn_rows_kernel<__nv_bfloat16, 64>) : go(paged_attn_rows_kernel<__nv_bfloat16, 128>);
}

}  // namespace picoattn
