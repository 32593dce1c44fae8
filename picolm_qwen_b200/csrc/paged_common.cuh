// paged_common.cuh -- element types, rotations and the ragged batch of the
// rotary and paged-cache kernels.
#pragma once

#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_common.cuh"
#include "paged_internal.h"

namespace picoattn {

// Sixteen-byte pieces of each element type as fp32 values and back.  pack()
// rounds to nearest even; store_cache() is the rounding of a cache row, which
// for fp16 is the reference's half-up rule (f32_to_f16_ref).
template <class T>
struct Elem;

template <>
struct Elem<float> {
    static constexpr int V = 4;  // elements per 16 bytes
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y);
        x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ float round(float x) { return x; }
};

template <>
struct Elem<__half> {
    static constexpr int V = 8;
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_half2(lo, hi); }
    static __device__ __forceinline__ uint32_t cache2(float lo, float hi) { return f32x2_to_f16_ref(lo, hi); }
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
    }
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};

template <>
struct Elem<__nv_bfloat16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint32_t cache2(float lo, float hi) { return pack2(lo, hi); }
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {  // a bf16 is the upper half of the fp32 of its value
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
    }
    static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
};

// (x0, x1) -> (x0 c - x1 s, x0 s + x1 c), products and sums rounded one by one
// as in the attention step's prep kernels, so a rotated key rounds to the same
// cache bits there and here.
__device__ __forceinline__ void rotate_pair(float& x0, float& x1, float c, float s) {
    const float a = x0, b = x1;
    x0 = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    x1 = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
}

// N consecutive fp32 of a table or weight row, which need only 4-byte alignment:
// in 16-byte loads where `vec` says that its rows start on 16 bytes.
template <int N>
__device__ __forceinline__ void load_f32(float* x, const float* p, bool vec) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(p + j);
            x[j] = f.x, x[j + 1] = f.y, x[j + 2] = f.z, x[j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = p[j];
    }
}

// Where a lane's two 16-byte pieces (V elements each) of a head lie, so that
// both members of every pair it rotates are its own.  Lane p of the hd/(2V) a
// head takes: rotated part first (NeoX: pieces p of both halves; interleaved:
// two adjacent pieces), then the part that stays, two adjacent pieces a lane.
// rot_dim is a multiple of 2V.
struct PieceAt {
    int a, b;      // first elements of the two pieces
    int pair;      // first table column (rotated lanes)
    bool rotated;
};
template <int V>
__device__ __forceinline__ PieceAt piece_at(int p, int rot, bool neox) {
    PieceAt r;
    r.rotated = 2 * V * p < rot;
    if (r.rotated && neox) r.a = V * p, r.b = rot / 2 + V * p, r.pair = V * p;
    else r.a = 2 * V * p, r.b = 2 * V * p + V, r.pair = V * p;
    return r;
}

// Rotates the lane's 2V elements x with its V table entries, each product and
// sum rounded (rotate_pair).
template <int V>
__device__ __forceinline__ void rotate_pieces(float* x, const float* c, const float* s, bool neox) {
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (neox) rotate_pair(x[j], x[V + j], c[j], s[j]);
        else rotate_pair(x[2 * j], x[2 * j + 1], c[j], s[j]);
    }
}

// The same with one product of each output fused into the sum (one rounding
// less), in packed pairs of fp32 where the layout gives them (the same bits): a
// third of the instructions.
__device__ __forceinline__ void rotate_pair_fused(float& x0, float& x1, float c, float s) {
    const float a = x0, b = x1;
    x0 = __fmaf_rn(a, c, -__fmul_rn(b, s));
    x1 = __fmaf_rn(a, s, __fmul_rn(b, c));
}
template <int V>
__device__ __forceinline__ void rotate_pieces_fused(float* x, const float* c, const float* s, bool neox) {
    if (neox) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const uint64_t c2 = f2_pack(c[j], c[j + 1]), s2 = f2_pack(s[j], s[j + 1]), n2 = f2_pack(-s[j], -s[j + 1]);
            const uint64_t x0 = f2_pack(x[j], x[j + 1]), x1 = f2_pack(x[V + j], x[V + j + 1]);
            f2_unpack(f2_fma(x0, c2, f2_mul(x1, n2)), x[j], x[j + 1]);
            f2_unpack(f2_fma(x0, s2, f2_mul(x1, c2)), x[V + j], x[V + j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) rotate_pair_fused(x[2 * j], x[2 * j + 1], c[j], s[j]);
    }
}

// The softmax weights go into the product with V in the cache's 16 bits: that is
// what its tensor instructions take, and it moves an output by at most half a step
// of the type times the weighted mean of |v|.  An fp16 weight is subnormal below
// 2^-14 and nothing below 2^-25, which over a long context is more than that: all
// of 131,072 keys at 2^-26 of a strong one make up 0.2% of the output.  So the
// running maximum is held `lift` (log2) too low and every weight is 2^lift times as
// large; sums and outputs carry the factor and it cancels at the end.  bf16 has
// fp32's range.
template <class T>
__host__ __device__ constexpr float weight_lift(int lift) {
    return std::is_same<T, __half>::value ? (float)lift : 0.f;
}

// Orders this thread's shared-memory writes before later async-proxy (TMA) accesses of them.
__device__ __forceinline__ void fence_proxy_async_shared() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// a / b for non-negative a and positive b, in 32 bits where they fit (a tenth of the instructions).
__device__ __forceinline__ long long quotient(long long a, long long b) {
    if (((unsigned long long)(a | b) >> 32) == 0) return (unsigned)a / (unsigned)b;
    return a / b;
}

// ---- the ragged batch ---------------------------------------------------------

struct SeqSpan {
    int t0, n, len;  // first row, new tokens, cache rows with the new tokens
    bool ok;         // within the host's bounds (n == 0: nothing to do)
};

__device__ __forceinline__ SeqSpan seq_span(const PagedBatch& a, int b) {
    SeqSpan s;
    s.t0 = a.q_start[b];
    const int t1 = a.q_start[b + 1];
    s.len = a.kv_len[b];
    s.n = (int)((unsigned)t1 - (unsigned)s.t0);  // wraps only for spans that fail the range test
    s.ok = s.t0 >= 0 && t1 >= s.t0 && t1 <= a.n_tok && s.n <= a.max_new && s.len >= s.n && s.len <= a.max_len;
    return s;
}

// The rows of a sequence outside the bounds that lie inside [0, n_tok).
struct RowRange {
    int first, end;  // end - first does not wrap, whatever 32-bit values the span has
};
__device__ __forceinline__ RowRange rows_inside(const PagedBatch& a, int b) {
    const int t0 = max(a.q_start[b], 0);
    return {t0, max(t0, min(a.q_start[b + 1], a.n_tok))};
}

}  // namespace picoattn
