// Rotary positions and the append to a paged cache: bfloat16.

#include "rotate.cuh"

namespace da {

int rotate_bf16(const RotateParams &p, bool paged, int n_batch, bool half, int v, cudaStream_t stream) {
    return rotate_any<__nv_bfloat16>(p, paged, n_batch, half, v, stream);
}

}  // namespace da
