// Attention over a paged cache: bfloat16.

#include "paged_mma.cuh"

namespace da {

cudaError_t paged_attention_bf16(const PagedParams &p, int head_dim, cudaStream_t stream) {
    return paged_mma<__nv_bfloat16>(p, head_dim, stream);
}

}  // namespace da
