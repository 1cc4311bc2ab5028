// Rotary positions and the append to a paged cache: float32.

#include "rotate.cuh"

namespace da {

int rotate_f32(const RotateParams &p, bool paged, int n_batch, bool half, int v, cudaStream_t stream) {
    return rotate_any<float>(p, paged, n_batch, half, v, stream);
}

}  // namespace da
