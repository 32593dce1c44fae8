// paged_append.cu -- a ragged batch's new keys and values into their pages, and
// its queries rotated for the attention (picoattn_paged_append).
//
// Per new token: QK-RMSNorm x / sqrt(mean(x^2) + eps) * w of every q and k head
// (fp32, when the weights are given), rotation of the first rot_dim elements at
// the token's position kv_len - n_new + i, rounding to the cache's type.
#include <algorithm>
#include <type_traits>

#include "paged_common.cuh"

namespace picoattn {

namespace {

constexpr int kAppendWarps = 4;  // 8 (and half the blocks): 3% slower

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
// lanes a head; a unit = up to kSteps steps of one kind of one token.  Bound by
// latency and instruction issue (some 250 instructions per step of 512 elements with
// QK-norm and its share of the lookups; 80 registers, so 24 warps an SM): the loads
// of a unit are issued first, its token's sequence, position, page and table entries
// are found while they travel, and units are numbered kind by kind, so that the
// warps of an SM run the same code.  Measured: 2,048 tokens of 32/8 heads of 128 with QK-norm in fp16 13.5 us
// (51 MB: 3.8 TB/s, 0.58 of the copy rate, as the contiguous prefill's prep kernel
// takes); 64 tokens 3.0 us.  Slower: a ring of cp.async copies of the next units
// 20.5 us (its shared memory comes out of the cache that the lookups live in), the
// next unit's loads issued before this one's work 16 (100 registers), 64 registers
// 17, a step a unit 18.
constexpr int kSteps = 2;

struct AppendSplit {
    int q_per, kv_per;            // units per token: q; k (and as many v)
    unsigned q_units, kv_units;   // all q units, all k (or v) units
};

template <class TI, class TC, int HD>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_append_kernel(PagedAppendArgs a, AppendSplit sp) {
    constexpr int LPH = HD / 16, HPS = 32 / LPH, W = sizeof(TI) == 4 ? 4 : 2, E = 16 / sizeof(TI);
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x == 0) {  // the bounds of all sequences, those without a row in this call too
        bool bad = false;
        for (int b = threadIdx.x; b < a.b.n_seqs; b += kAppendWarps * 32) bad |= !seq_span(a.b, b).ok;
        if (bad) atomicOr(a.b.status, PICOATTN_DEV_BAD_POS);
        return;
    }
    const bool neox = a.mode == PICOATTN_ROPE_NEOX;
    const PieceAt at = piece_at<8>(lane % LPH, a.rot, neox);
    const bool vec = (((uintptr_t)a.cos_t | (uintptr_t)a.sin_t | (uintptr_t)a.qn_w | (uintptr_t)a.kn_w) & 15) == 0;
    const unsigned units = sp.q_units + 2 * sp.kv_units;
    for (unsigned u = (blockIdx.x - 1) * kAppendWarps + warp; u < units; u += (gridDim.x - 1) * kAppendWarps) {
        const int kind = u < sp.q_units ? 0 : (u < sp.q_units + sp.kv_units ? 1 : 2);
        const unsigned i0 = u - (kind == 0 ? 0 : (kind == 1 ? sp.q_units : sp.q_units + sp.kv_units));
        const unsigned per = kind == 0 ? sp.q_per : sp.kv_per, tok = i0 / per;
        const int h0 = (int)(i0 - tok * per) * (kSteps * HPS) + lane / LPH, heads = kind == 0 ? a.hq : a.hkv;
        const TI* src = static_cast<const TI*>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v)) +
                        tok * (kind == 0 ? a.qs : (kind == 1 ? a.ks : a.vs)) + h0 * HD;
        uint4 w[kSteps][W];
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
            for (int j = 0; j < W; j++)
                w[i][j] = h0 + i * HPS < heads
                              ? *reinterpret_cast<const uint4*>(src + i * HPS * HD + (j < W / 2 ? at.a + E * j
                                                                                               : at.b + E * (j - W / 2)))
                              : make_uint4(0, 0, 0, 0);
        const int b = seq_of(a.b, (int)tok, lane);
        if (b >= a.b.n_seqs) continue;       // a row behind the last sequence
        const SeqSpan span = seq_span(a.b, b);
        if (b == 0 && (int)tok < span.t0) continue;  // a row before the first sequence
        // seq_of takes q_start as not decreasing: one that decreases (and is flagged) may give a sequence without this
        // token
        const bool ok = span.ok && (int)tok >= span.t0 && (int)tok - span.t0 < span.n;
        const int pos = ok ? span.len - span.n + ((int)tok - span.t0) : 0;
        TC* dst = static_cast<TC*>(a.q_out) + ((long long)tok * a.hq + h0) * HD;
        int hop = HPS * HD;
        if (kind != 0) {
            if (!ok) continue;
            const int page = a.b.page_table[(size_t)b * a.b.page_cols + (pos >> a.b.page_shift)];
            if (page < 0 || page >= a.b.n_pages) {
                if (lane == 0) atomicOr(a.b.status, PICOATTN_DEV_BAD_PAGE);
                continue;
            }
            dst = static_cast<TC*>(kind == 1 ? a.k_pool : a.v_pool) +
                  (((size_t)page * a.hkv + h0) * a.b.page_size + (pos & (a.b.page_size - 1))) * HD;
            hop *= a.b.page_size;
        }
        if (kind == 2) {  // v: the cache's rounding alone
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                if (h0 + i * HPS >= heads) break;
                if constexpr (std::is_same<TI, TC>::value) {  // the bits themselves
                    *reinterpret_cast<uint4*>(dst + (size_t)i * hop + at.a) = w[i][0];
                    *reinterpret_cast<uint4*>(dst + (size_t)i * hop + at.b) = w[i][1];
                } else {
                    float x[16];
#pragma unroll
                    for (int j = 0; j < W; j++) Elem<TI>::unpack(w[i][j], x + E * j);
                    store_pieces<TC, true>(x, dst + (size_t)i * hop, at);
                }
            }
            continue;
        }
        float c[8], s[8], g[16];
        if (at.rotated) {
            load_f32<8>(c, a.cos_t + (size_t)pos * (a.rot / 2) + at.pair, vec);
            load_f32<8>(s, a.sin_t + (size_t)pos * (a.rot / 2) + at.pair, vec);
        }
        if (a.qn_w) {
            const float* nw = kind == 0 ? a.qn_w : a.kn_w;
            load_f32<8>(g, nw + at.a, vec);
            load_f32<8>(g + 8, nw + at.b, vec);
        }
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
            float x[16];
#pragma unroll
            for (int j = 0; j < W; j++) Elem<TI>::unpack(w[i][j], x + E * j);
            if (a.qn_w) {
                uint64_t s2 = 0;
#pragma unroll
                for (int j = 0; j < 16; j += 2) s2 = f2_fma(f2_pack(x[j], x[j + 1]), f2_pack(x[j], x[j + 1]), s2);
                float lo, hi;
                f2_unpack(s2, lo, hi);
                float ss = lo + hi;
#pragma unroll
                for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float r = rsqrtf(ss * (1.0f / HD) + a.eps);
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    f2_unpack(f2_mul(f2_mul(f2_pack(x[j], x[j + 1]), f2_pack(r, r)), f2_pack(g[j], g[j + 1])), x[j],
                              x[j + 1]);
                // the sums above follow another order than the reference's, so the
                // rotation need not round as it does either
                if (at.rotated) rotate_pieces_fused<8>(x, c, s, neox);
            } else if (at.rotated) {
                rotate_pieces<8>(x, c, s, neox);
            }
            if (h0 + i * HPS >= heads) continue;
            if (kind == 1) {
                store_pieces<TC, true>(x, dst + (size_t)i * hop, at);
            } else {
                if (!ok) {
#pragma unroll
                    for (int j = 0; j < 16; j++) x[j] = __int_as_float(0x7fc00000);
                }
                store_pieces<TC, false>(x, dst + (size_t)i * hop, at);
            }
        }
    }
}

template <class TI, class TC, int HD>
cudaError_t launch_hd(const PagedAppendArgs& a, cudaStream_t stream) {
    constexpr int HPU = kSteps * 32 / (HD / 16);  // heads per unit
    AppendSplit sp{};
    sp.q_per = a.q ? (a.hq + HPU - 1) / HPU : 0;
    sp.kv_per = (a.hkv + HPU - 1) / HPU;
    const long long units = (long long)a.b.n_tok * (sp.q_per + 2 * sp.kv_per);
    sp.q_units = (unsigned)a.b.n_tok * sp.q_per;
    sp.kv_units = (unsigned)a.b.n_tok * sp.kv_per;
    const unsigned grid = (unsigned)std::min<long long>((units + kAppendWarps - 1) / kAppendWarps, 12LL * device_sm_count());
    return launch_pdl(paged_append_kernel<TI, TC, HD>, dim3(1 + grid), dim3(kAppendWarps * 32), 0, stream, a, sp);
}

template <class TI, class TC>
cudaError_t launch_types(const PagedAppendArgs& a, cudaStream_t stream) {
    return a.hd == 64 ? launch_hd<TI, TC, 64>(a, stream) : launch_hd<TI, TC, 128>(a, stream);
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
