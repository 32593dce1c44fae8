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

// One warp rotates the pairs (and copies the rest) of one head of one token,
// an element pair per lane: any head_dim, rot_dim and alignment.
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
            rotate_pair(x0, x1, cr[i], a.inverse ? -sr[i] : sr[i]);
            y[e0] = Elem<T>::round(x0);
            y[e1] = Elem<T>::round(x1);
        }
        if (x != y)
            for (int e = a.rot + lane; e < a.hd; e += 32) y[e] = x[e];
    }
}

}  // namespace

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t stream) {
    const long long units = (long long)a.n_tok * (a.t[0].heads + a.t[1].heads);
    const unsigned grid = (unsigned)std::min<long long>((units + 7) / 8, 8LL * device_sm_count());
    auto go = [&](auto kernel) { return launch_pdl(kernel, dim3(grid), dim3(256), 0, stream, a); };
    switch (a.dtype) {
        case PICOATTN_DTYPE_F32: return go(rope_kernel<float>);
        case PICOATTN_DTYPE_F16: return go(rope_kernel<__half>);
        default: return go(rope_kernel<__nv_bfloat16>);
    }
}

}  // namespace picoattn
