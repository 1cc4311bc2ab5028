// Attention over a paged cache: float16.

#include "paged_mma.cuh"

namespace da {

cudaError_t paged_attention_f16(const PagedParams &p, int head_dim, cudaStream_t stream) {
    return paged_mma<__half>(p, head_dim, stream);
}

}  // namespace da
