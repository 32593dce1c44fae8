// rope.cu -- rotary positions of q and k on their own (picoattn_rope).
//
// y0 = x0 c - x1 s, y1 = x0 s + x1 c for the pairs of the first rot_dim elements
// of every head, c and s from the table row of the token's position; the other
// elements are copied.  The inverse (s negated) is the transpose and so the
// backward pass.
#include <algorithm>

#include "paged_common.cuh"

namespace picoattn {

namespace {

// Any head_dim, rot_dim and alignment: one warp rotates the pairs (and copies
// the rest) of one head of one token, an element pair per lane.  An element an
// access: 2,048 tokens of 32 + 8 heads of 96 in fp16 18.7 us (31 MB,
// 1.7 TB/s); of 128, which the kernel below takes, 6.3 us.
template <class T>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int heads = a.t[0].heads + a.t[1].heads;
    const long long warps = (long long)gridDim.x * (blockDim.x / 32);
    for (long long u = (long long)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); u < (long long)a.n_tok * heads;
         u += warps) {
        const int tok = (int)(u / heads);
        int h = (int)(u - (long long)tok * heads);
        const RopeRows& r = h < a.t[0].heads ? a.t[0] : a.t[1];
        if (h >= a.t[0].heads) h -= a.t[0].heads;
        const T* x = static_cast<const T*>(r.x) + tok * r.x_stride + (long long)h * a.hd;
        T* y = static_cast<T*>(r.out) + tok * r.out_stride + (long long)h * a.hd;
        const int p = a.pos[tok];
        if (p < 0 || p >= a.table_rows) {
            if (lane == 0) atomicOr(a.status, PICOATTN_DEV_BAD_POS);
            for (int e = lane; e < a.hd; e += 32) y[e] = Elem<T>::round(__int_as_float(0x7fc00000));
            continue;
        }
        const int half = a.rot / 2;
        const float* cr = a.cos_t + (size_t)p * half;
        const float* sr = a.sin_t + (size_t)p * half;
        for (int i = lane; i < half; i += 32) {
            const int e0 = a.mode == PICOATTN_ROPE_NEOX ? i : 2 * i, e1 = a.mode == PICOATTN_ROPE_NEOX ? i + half : 2 * i + 1;
            float x0 = Elem<T>::load(x + e0), x1 = Elem<T>::load(x + e1);
            rotate_pair_fused(x0, x1, cr[i], a.inverse ? -sr[i] : sr[i]);
            y[e0] = Elem<T>::round(x0);
            y[e1] = Elem<T>::round(x1);
        }
        if (x != y)
            for (int e = a.rot + lane; e < a.hd; e += 32) y[e] = x[e];
    }
}

// The same with 16-byte accesses: a lane holds two pieces of V elements of a
// head (both members of its pairs, piece_at), LPH = hd / 2V lanes a head, so a
// warp step takes 32 / LPH heads of one token.  Memory-bound (one read and one
// write of every element): a unit is up to kSteps steps of one tensor of one
// token, whose loads are all issued before the first rotation and which share
// the lane's table entries.  Measured at 8,192 tokens of 32 + 8 heads of 128 in
// bf16, far positions: 28.5 us = 6.0 TB/s, 0.93 of the copy rate (4 steps: 31 us,
// more registers and so fewer warps); 2,047 tokens of 28 + 4 heads in fp32, half
// of each rotated, backward: 13.6 us = 5.0 TB/s (2 steps: 13.8).
template <class T>
constexpr int kSteps = sizeof(T) == 4 ? 4 : 2;
constexpr int kBlocksPerSm = 12;  // in the grid: warps take several units in turn

struct RopeSplit {
    int lph_shift, per_unit, q_units, units_per_tok;  // per_unit: steps of a unit
    unsigned units;
};

template <class T>
__global__ void __launch_bounds__(256) rope_vec_kernel(RopeArgs a, RopeSplit sp) {
    constexpr int V = Elem<T>::V;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int hps = 32 >> sp.lph_shift;
    const bool neox = a.mode == PICOATTN_ROPE_NEOX;
    const PieceAt at = piece_at<V>(lane & ((1 << sp.lph_shift) - 1), a.rot, neox);
    const bool vec = (((uintptr_t)a.cos_t | (uintptr_t)a.sin_t) & 15) == 0 && a.rot % 8 == 0;  // whole rows
    for (unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5); u < sp.units; u += gridDim.x * 8) {
        const unsigned tok = u / (unsigned)sp.units_per_tok;
        int part = (int)(u - tok * (unsigned)sp.units_per_tok);
        const bool second = part >= sp.q_units;
        if (second) part -= sp.q_units;
        const RopeRows& r = a.t[second ? 1 : 0];
        const int pos = a.pos[tok];
        const int h0 = part * sp.per_unit * hps + (lane >> sp.lph_shift);
        const T* src = static_cast<const T*>(r.x) + tok * r.x_stride + (long long)h0 * a.hd;
        T* dst = static_cast<T*>(r.out) + tok * r.out_stride + (long long)h0 * a.hd;
        const bool ok = pos >= 0 && pos < a.table_rows;
        if (!ok && lane == 0) atomicOr(a.status, PICOATTN_DEV_BAD_POS);
        // an element that stays need not move when the rotation is in place
        const bool still = ok && !at.rotated && src == dst;
        const int n = still ? 0 : min(sp.per_unit, (r.heads - h0 + hps - 1) / hps);
        const int hop = hps * a.hd;
        uint4 w[kSteps<T>][2];
#pragma unroll
        for (int i = 0; i < kSteps<T>; i++)
            if (i < n) {
                w[i][0] = *reinterpret_cast<const uint4*>(src + i * hop + at.a);
                w[i][1] = *reinterpret_cast<const uint4*>(src + i * hop + at.b);
            }
        float c[V], s[V];
        if (ok && at.rotated) {
            load_f32<V>(c, a.cos_t + (size_t)pos * (a.rot / 2) + at.pair, vec);
            load_f32<V>(s, a.sin_t + (size_t)pos * (a.rot / 2) + at.pair, vec);
            if (a.inverse) {
#pragma unroll
                for (int j = 0; j < V; j++) s[j] = -s[j];
            }
        }
#pragma unroll
        for (int i = 0; i < kSteps<T>; i++) {
            if (i >= n) break;
            if (at.rotated || !ok) {
                float x[2 * V];
                Elem<T>::unpack(w[i][0], x);
                Elem<T>::unpack(w[i][1], x + V);
                if (ok) {
                    rotate_pieces_fused<V>(x, c, s, neox);
                } else {
#pragma unroll
                    for (int j = 0; j < 2 * V; j++) x[j] = __int_as_float(0x7fc00000);
                }
                w[i][0] = Elem<T>::pack(x);
                w[i][1] = Elem<T>::pack(x + V);
            }
            *reinterpret_cast<uint4*>(dst + i * hop + at.a) = w[i][0];
            *reinterpret_cast<uint4*>(dst + i * hop + at.b) = w[i][1];
        }
    }
}

template <class T>
cudaError_t launch_type(const RopeArgs& a, cudaStream_t stream) {
    constexpr int V = Elem<T>::V;
    const int sms = device_sm_count();
    const int lph = a.hd / (2 * V);
    bool vec = a.hd % (2 * V) == 0 && lph <= 32 && (lph & (lph - 1)) == 0 && a.rot % (2 * V) == 0;
    for (const RopeRows& r : a.t)
        if (r.heads && ((((uintptr_t)r.x | (uintptr_t)r.out) & 15) || r.x_stride % V || r.out_stride % V)) vec = false;
    RopeSplit sp{};
    if (vec) {
        while ((1 << sp.lph_shift) < lph) sp.lph_shift++;
        const int hps = 32 / lph, qs = (a.t[0].heads + hps - 1) / hps, ks = (a.t[1].heads + hps - 1) / hps;
        // Several steps a unit once that still gives every SM its warps; below, a
        // step a unit: the call is as short as one round of loads
        for (sp.per_unit = kSteps<T>; sp.per_unit > 1; sp.per_unit /= 2)
            if ((long long)a.n_tok * ((qs + ks) / sp.per_unit) >= 32LL * sms) break;
        sp.q_units = (qs + sp.per_unit - 1) / sp.per_unit;
        sp.units_per_tok = sp.q_units + (ks + sp.per_unit - 1) / sp.per_unit;
        const long long units = (long long)a.n_tok * sp.units_per_tok;
        if (units < (1LL << 31)) {  // the kernel counts in 32 bits
            sp.units = (unsigned)units;
            const unsigned grid = (unsigned)std::min<long long>((units + 7) / 8, (long long)kBlocksPerSm * sms);
            return launch_pdl(rope_vec_kernel<T>, dim3(grid), dim3(256), 0, stream, a, sp);
        }
    }
    const long long units = (long long)a.n_tok * (a.t[0].heads + a.t[1].heads);
    const unsigned grid = (unsigned)std::min<long long>((units + 7) / 8, 8LL * sms);
    return launch_pdl(rope_kernel<T>, dim3(grid), dim3(256), 0, stream, a);
}

}  // namespace

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t stream) {
    switch (a.dtype) {
        case PICOATTN_DTYPE_F32: return launch_type<float>(a, stream);
        case PICOATTN_DTYPE_F16: return launch_type<__half>(a, stream);
        default: return launch_type<__nv_bfloat16>(a, stream);
    }
}

}  // namespace picoattn
