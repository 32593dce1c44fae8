// paged_internal.h -- launch descriptors of the rotary and paged-cache kernels.
#pragma once

#include <cstddef>
#include <cstdint>
#include <utility>

#include <cuda_runtime.h>

#include "picoattn_internal.h"

namespace picoattn {

// Launch with programmatic stream serialisation (see pdl_wait in device_common.cuh).
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
    return e != cudaSuccess ? e : cudaGetLastError();
}

struct RopeRows {
    const void* x;
    void* out;
    long long x_stride, out_stride;
    int heads;
};

struct RopeArgs {
    RopeRows t[2];  // q, k (heads 0: none)
    int dtype, mode, hd, rot, inverse, n_tok, table_rows;
    const int* pos;
    const float* cos_t;
    const float* sin_t;
    unsigned int* status;
};
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t stream);

// picoattn_paged_batch_t, with the cache's shape
struct PagedBatch {
    int n_seqs, n_tok, max_new, max_len, page_cols, n_pages, page_size, page_shift;
    const int* page_table;
    const int* q_start;
    const int* kv_len;
    unsigned int* status;
};

struct PagedAppendArgs {
    PagedBatch b;
    int hq, hkv, hd, rot, mode, in_dtype, cache_dtype;
    float eps;
    const void* q;
    const void* k;
    const void* v;
    long long qs, ks, vs;  // row strides in elements
    const float* qn_w;
    const float* kn_w;
    const float* cos_t;
    const float* sin_t;
    void* q_out;
    void* k_pool;  // this layer's pages [n_pages][hkv][page_size][hd]
    void* v_pool;
};
cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t stream);

struct PagedAttnArgs {
    PagedBatch b;
    int hq, hkv, g, hd, dtype, out_dtype;
    long long qs;
    const void* q;
    const void* k_pool;
    const void* v_pool;
    void* out;
    uint8_t* ws;  // workspace past the header
};
cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t stream);
// Few query rows per KV head and sequence (paged_few.cu)
bool paged_few_fits(const PagedAttnArgs& a);
size_t paged_few_bytes(int hd);
cudaError_t launch_paged_few(const PagedAttnArgs& a, cudaStream_t stream);
// Any batch (paged_chunk.cu)
size_t paged_chunk_bytes(int hd);
cudaError_t launch_paged_chunk(const PagedAttnArgs& a, cudaStream_t stream);
size_t paged_workspace_bytes(const picoattn_config_t& cfg, int n_seqs);

}  // namespace picoattn
