// paged_attn.cu -- which kernels a paged attention call takes (picoattn_paged_attn).
#include <algorithm>

#include "paged_internal.h"

namespace picoattn {

// Both paths keep their partial results in the same place: a call runs one of them.
size_t paged_workspace_bytes(const picoattn_config_t& cfg, int n_seqs) {
    return kWsHeaderBytes + align_up(std::max(paged_few_bytes(cfg.head_dim), paged_chunk_bytes(cfg.head_dim)), 256);
}

cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t stream) {
    return paged_few_fits(a) ? launch_paged_few(a, stream) : launch_paged_chunk(a, stream);
}

}  // namespace picoattn
