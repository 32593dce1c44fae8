// paged_append.cu -- a ragged batch's new keys and values into their pages, and
// its queries rotated for the attention (picoattn_paged_append).
//
// Per new token: QK-RMSNorm x / sqrt(mean(x^2) + eps) * w of every q and k head
// (fp32, when the weights are given), rotation of the first rot_dim elements at
// the token's position kv_len - n_new + i, rounding to the cache's type.
#include <algorithm>

#include "paged_common.cuh"

namespace picoattn {

namespace {

constexpr int kAppendWarps = 8;

// The sequence of token row t: the number of q_start[1..] entries <= t, 32 at a
// time (q_start does not decrease).  n_seqs: none.
__device__ __forceinline__ int seq_of(const PagedBatch& a, int t, int lane) {
    int b = 0;
    for (int i = 0; i < a.n_seqs; i += 32) {
        const bool le = i + lane < a.n_seqs && a.q_start[i + lane + 1] <= t;
        b += __popc(__ballot_sync(0xffffffffu, le));
    }
    return b;
}

// The lane's two pieces of one head, widened to fp32.
template <class TI>
__device__ __forceinline__ void load_pieces(float (&x)[16], const TI* head, const PieceAt& at) {
    if constexpr (sizeof(TI) == 4) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            Elem<float>::unpack(*reinterpret_cast<const uint4*>(head + at.a + 4 * i), x + 4 * i);
            Elem<float>::unpack(*reinterpret_cast<const uint4*>(head + at.b + 4 * i), x + 8 + 4 * i);
        }
    } else {
        Elem<TI>::unpack(*reinterpret_cast<const uint4*>(head + at.a), x);
        Elem<TI>::unpack(*reinterpret_cast<const uint4*>(head + at.b), x + 8);
    }
}

template <class TC, bool CACHE>
__device__ __forceinline__ void store_pieces(const float (&x)[16], TC* head, const PieceAt& at) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        w[i] = CACHE ? Elem<TC>::cache2(x[2 * i], x[2 * i + 1]) : Elem<TC>::pack2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(head + at.a) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(head + at.b) = make_uint4(w[4], w[5], w[6], w[7]);
}

// A warp step = up to HPS heads of one kind (q, k or v) of one token, hd/16
// lanes a head.
template <class TI, class TC, int HD>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_append_kernel(PagedAppendArgs a) {
    constexpr int LPH = HD / 16, HPS = 32 / LPH;
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int p = lane % LPH;
    const bool neox = a.mode == PICOATTN_ROPE_NEOX;
    const int qsteps = a.q ? (a.hq + HPS - 1) / HPS : 0, ksteps = (a.hkv + HPS - 1) / HPS;
    const int per_tok = qsteps + 2 * ksteps;
    const long long steps = (long long)a.b.n_tok * per_tok;
    for (long long u = (long long)blockIdx.x * kAppendWarps + warp; u < steps; u += (long long)gridDim.x * kAppendWarps) {
        const int tok = (int)(u / per_tok);
        int st = (int)(u - (long long)tok * per_tok);
        const int kind = st < qsteps ? 0 : (st < qsteps + ksteps ? 1 : 2);
        st -= kind == 0 ? 0 : (kind == 1 ? qsteps : qsteps + ksteps);
        const int heads = kind == 0 ? a.hq : a.hkv;
        const int h = st * HPS + lane / LPH;
        const bool live = h < heads;
        const int b = seq_of(a.b, tok, lane);
        if (b >= a.b.n_seqs) continue;            // a row behind the last sequence
        const SeqSpan sp = seq_span(a.b, b);
        if (tok < sp.t0) continue;                // a row before the first sequence
        const PieceAt at = piece_at<8>(p, a.rot, neox);
        TC* q_out = static_cast<TC*>(a.q_out) + ((long long)tok * a.hq + h) * HD;
        if (!sp.ok) {
            if (lane == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_POS);
            float nan[16];
#pragma unroll
            for (int j = 0; j < 16; j++) nan[j] = __int_as_float(0x7fc00000);
            if (kind == 0 && live) store_pieces<TC, false>(nan, q_out, at);
            continue;
        }
        const int pos = sp.len - sp.n + (tok - sp.t0);
        const TI* src = static_cast<const TI*>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v)) +
                        tok * (kind == 0 ? a.qs : (kind == 1 ? a.ks : a.vs)) + (long long)(live ? h : 0) * HD;
        float x[16];
        load_pieces(x, src, at);
        if (kind != 2) {
            if (a.qn_w) {
                const float* w = kind == 0 ? a.qn_w : a.kn_w;
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 16; j++) ss += x[j] * x[j];
#pragma unroll
                for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float scale = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(ss / (float)HD, a.eps)));
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[j] = __fmul_rn(__fmul_rn(x[j], scale), w[at.a + j]);
                    x[8 + j] = __fmul_rn(__fmul_rn(x[8 + j], scale), w[at.b + j]);
                }
            }
            if (at.rotated) {
                const float* cr = a.cos_t + (size_t)pos * (a.rot / 2) + at.pair;
                const float* sr = a.sin_t + (size_t)pos * (a.rot / 2) + at.pair;
                float c[8], s[8];
#pragma unroll
                for (int j = 0; j < 8; j++) c[j] = cr[j], s[j] = sr[j];
                rotate_pieces<8>(x, c, s, neox);
            }
        }
        if (kind == 0) {
            if (live) store_pieces<TC, false>(x, q_out, at);
            continue;
        }
        const int page = a.b.page_table[(size_t)b * a.b.page_cols + (pos >> a.b.page_shift)];
        if (page < 0 || page >= a.b.n_pages) {
            if (lane == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_PAGE);
            continue;
        }
        TC* pool = static_cast<TC*>(kind == 1 ? a.k_pool : a.v_pool);
        const size_t row = ((size_t)page * a.hkv + h) * a.b.page_size + (pos & (a.b.page_size - 1));
        if (live) store_pieces<TC, true>(x, pool + row * HD, at);
    }
}

template <class TI, class TC>
cudaError_t launch_types(const PagedAppendArgs& a, cudaStream_t stream) {
    const int hps = 32 / (a.hd / 16);
    const long long steps =
        (long long)a.b.n_tok * ((a.q ? (a.hq + hps - 1) / hps : 0) + 2 * ((a.hkv + hps - 1) / hps));
    const unsigned grid =
        (unsigned)std::min<long long>((steps + kAppendWarps - 1) / kAppendWarps, 8LL * device_sm_count());
    return launch_pdl(a.hd == 64 ? paged_append_kernel<TI, TC, 64> : paged_append_kernel<TI, TC, 128>, dim3(grid),
                      dim3(kAppendWarps * 32), 0, stream, a);
}

template <class TC>
cudaError_t launch_cache(const PagedAppendArgs& a, cudaStream_t stream) {
    switch (a.in_dtype) {
        case PICOATTN_DTYPE_F32: return launch_types<float, TC>(a, stream);
        case PICOATTN_DTYPE_F16: return launch_types<__half, TC>(a, stream);
        default: return launch_types<__nv_bfloat16, TC>(a, stream);
    }
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t stream) {
    return a.cache_dtype == PICOATTN_DTYPE_F16 ? launch_cache<__half>(a, stream) : launch_cache<__nv_bfloat16>(a, stream);
}

}  // namespace picoattn
