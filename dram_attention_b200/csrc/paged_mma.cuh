// Attention over a paged cache, 16-bit element types: the two products of a 16-token unit on tensor cores.
//
// A KV head has a handful of query rows, far below the 64 rows of the smallest tcgen05.mma tile, and memory is what bounds
// the kernel; warp-level mma.sync m16n8k16 needs an eighth of the instructions of CUDA-core arithmetic and no more.
//   S = Q K^T   A = query rows in registers, B = key rows by ldmatrix
//   O += P V    A = the weights, straight from S's accumulators, B = value rows by ldmatrix.trans
// A token's rows lie 16 bytes apart from a multiple of 128 bytes in shared memory, so that the eight row addresses of an
// ldmatrix tile fall into distinct banks for every head size that is a multiple of 16.  Two tokens to a gap halve the number of
// copies and have two rows in the same banks: faster for 64 channels (64 sequences of 16 000 tokens, 2 heads: 88 us, so 84) and 256
// (64 of 5000: 123, so 116), slower between them (60 of 3000, 8 heads of 80 and 96: 74 and 86 us, 79 and 93; 128 channels equal).
#pragma once

#include <type_traits>

#include "mma_sync.cuh"
#include "paged_attn.cuh"

namespace da {

constexpr int paged_mma_together(int head_dim) { return head_dim == 64 || head_dim == 256 ? 2 : 1; }
constexpr int paged_mma_stage(int head_dim) { return kPagedUnit * 4 * head_dim + kPagedUnit / paged_mma_together(head_dim) * 16; }

// FULL: up to 16 query rows; otherwise up to 8 (rows 8..15 of the tile are zero and nothing is kept of them).
// LONG: a warp may have more than kPagedRun units of one item.  The tensor cores cut off the low bits of the sums that they add to,
// always towards zero, so an accumulator that they keep loses up to 2^-23 of itself with every product: float16 outputs of equal
// weights and values near 1 are 1e-4 too small on average for 131 072 tokens in one warp and 4e-3 for a million, against half a step
// of 5e-4.  A LONG unit's product is made alone and added in float32, rounded to nearest (1e-6).  Batches that need none of it would
// take 3 % longer by it with 64 channels, 8 % with 256 (registers spill: 64 x 2000 tokens 53.3 us, 58.1), the same with 96 and 128.
template <typename T, int D_, bool FULL, bool LONG>
struct PagedMma {
    using Elem = T;
    static constexpr int kD = D_, kRows = FULL ? 16 : 8;
    static constexpr int ROWB = kD * 2, kTogether = paged_mma_together(kD), kStageBytes = paged_mma_stage(kD);
    static constexpr int KSTEPS = kD / 16, NT = kD / 8, NR = FULL ? 2 : 1;
    static constexpr int kScratch = 0;
    // Weights, in (0, 1], and all that is summed with them are kept kWeight times as large: float16 has nothing between 0 and 2^-24, and
    // many weights down there are a share of the sum (32 000 of 2.8e-8 beside one of 1: 0.0009, half a step is 0.0005).  So they are
    // lost below 2^-40 of the largest; bfloat16 has the range of float32.  Scaling them takes 2 % of 256 channels and twelve rows (64 x
    // 2000 tokens, 2 heads: 55.8 us, so 57.0), elsewhere less than the clock varies.
    static constexpr float kWeight = std::is_same<T, __half>::value ? 32768.f : 1.f;
    __device__ __forceinline__ static constexpr int offset(int t) { return t * 2 * ROWB + t / kTogether * 16; }
    static_assert(kD % 16 == 0, "whole k-steps");

    struct State {
        uint32_t q[NR][2][KSTEPS];    // A fragments: [row half][k half][k-step]
        float m[NR], l[NR];           // row maximum (the same in the four lanes of a row), this lane's share of the weight sum
        float o[NT][4];               // (rows 8..15: of no meaning unless FULL)
    };

    __device__ __forceinline__ static void begin(State &st, const PagedParams &p, int b, int head, int group, int rows, int lane, unsigned char *) {
        const int head0 = head * p.rep + group * p.group_rows;
#pragma unroll
        for (int half = 0; half < NR; ++half) {
            const int r = (lane >> 2) + 8 * half;
            const T *row = reinterpret_cast<const T *>(p.q) + b * p.q_seq + (head0 + (r < rows ? r : 0)) * p.q_head;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
                const uint32_t w0 = *reinterpret_cast<const uint32_t *>(row + 16 * ks + 2 * (lane & 3));
                const uint32_t w1 = *reinterpret_cast<const uint32_t *>(row + 16 * ks + 8 + 2 * (lane & 3));
                st.q[half][0][ks] = r < rows ? w0 : 0u;
                st.q[half][1][ks] = r < rows ? w1 : 0u;
            }
            st.m[half] = -INFINITY;
            st.l[half] = 0.f;
        }
#pragma unroll
        for (int d = 0; d < NT; ++d) st.o[d][0] = st.o[d][1] = st.o[d][2] = st.o[d][3] = 0.f;
    }

    __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[NR][2], uint32_t b0, uint32_t b1) {
        if constexpr (FULL) MmaTraits<T>::mma16(d, a[0][0], a[1][0], a[0][1], a[1][1], b0, b1);
        else MmaTraits<T>::mma(d, a[0][0], a[0][1], b0, b1);
    }

    __device__ __forceinline__ static void product(float (&d)[4], const uint32_t (&a)[NR][2], uint32_t b0, uint32_t b1) {
        if constexpr (FULL) MmaTraits<T>::product(d, a[0][0], a[1][0], a[0][1], a[1][1], b0, b1);
        else MmaTraits<T>::product(d, a[0][0], 0u, a[0][1], 0u, b0, b1);
    }

    __device__ __forceinline__ static void consume(State &st, const unsigned char *unit, uint32_t mask, int lane, float scale_log2) {
        const int qd = lane & 3, tile = lane >> 3, tr = lane & 7;
        // key tiles of a k-step: tokens 0..7 and 8..15, channels 0..7 and 8..15 of it
        const unsigned char *keys = unit + offset((tile >> 1) * 8 + tr) + (tile & 1) * 16;
        // value tiles of 16 channels, transposed by the load
        const unsigned char *values = unit + ROWB + offset((tile & 1) * 8 + tr) + (tile >> 1) * 16;

        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
        float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};   // odd k-steps: four chains instead of two
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            uint32_t b[4], a[NR][2];
            ldmatrix_x4(b, keys + ks * 32);
#pragma unroll
            for (int half = 0; half < NR; ++half) a[half][0] = st.q[half][0][ks], a[half][1] = st.q[half][1][ks];
            mma(ks & 1 ? t0 : s0, a, b[0], b[1]);
            mma(ks & 1 ? t1 : s1, a, b[2], b[3]);
        }
        // The weights take part in the second product as the sum of two 16-bit numbers, which leave 2^-16 of them in bfloat16 and
        // 2^-22 in float16: rounded to one, they alone put bfloat16 outputs 1.2 times as far from the 64-bit ones as their own
        // rounding does, and memory hides the products.
        uint32_t pa[NR][2], pb[NR][2];
        float alpha[NR];
#pragma unroll
        for (int half = 0; half < NR; ++half) {
            // this lane: row lane / 4 + 8 * half, tokens 2 qd, 2 qd + 1, 8 + 2 qd, 9 + 2 qd
            float v[4];
            v[0] = s0[2 * half] + t0[2 * half], v[1] = s0[2 * half + 1] + t0[2 * half + 1];
            v[2] = s1[2 * half] + t1[2 * half], v[3] = s1[2 * half + 1] + t1[2 * half + 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool there = (mask >> (2 * qd + (i & 1) + 8 * (i >> 1))) & 1;
                v[i] = there ? v[i] * scale_log2 : -INFINITY;
            }
            float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
            mx = fmaxf(mx, __shfl_xor_sync(DA_FULL_MASK, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(DA_FULL_MASK, mx, 2));
            const float m = fmaxf(st.m[half], mx);
            const float ms = m == -INFINITY ? 0.f : m;
            alpha[half] = fast_exp2(st.m[half] - ms);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = fast_exp2(v[i] - ms) * kWeight;
            st.l[half] = st.l[half] * alpha[half] + ((v[0] + v[1]) + (v[2] + v[3]));
            st.m[half] = m;
            if (!LONG && __any_sync(DA_FULL_MASK, alpha[half] != 1.f)) {   // once the maxima have settled there is nothing to rescale
#pragma unroll
                for (int d = 0; d < NT; ++d) {
                    st.o[d][2 * half] *= alpha[half];
                    st.o[d][2 * half + 1] *= alpha[half];
                }
            }
            pa[half][0] = MmaTraits<T>::pack(v[0], v[1]);
            pa[half][1] = MmaTraits<T>::pack(v[2], v[3]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float lo, hi;
                unpack2<T>(pa[half][i], lo, hi);
                pb[half][i] = MmaTraits<T>::pack(v[2 * i] - lo, v[2 * i + 1] - hi);
            }
        }
#pragma unroll
        for (int d = 0; d < NT / 2; ++d) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, values + d * 32);
            if constexpr (!LONG) {
                mma(st.o[2 * d], pa, b[0], b[1]);
                mma(st.o[2 * d + 1], pa, b[2], b[3]);
                mma(st.o[2 * d], pb, b[0], b[1]);
                mma(st.o[2 * d + 1], pb, b[2], b[3]);
            } else {
                float x[2][4];
                product(x[0], pa, b[0], b[1]);
                product(x[1], pa, b[2], b[3]);
                mma(x[0], pb, b[0], b[1]);
                mma(x[1], pb, b[2], b[3]);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 2 * NR; ++i) st.o[2 * d + t][i] = fmaf(st.o[2 * d + t][i], alpha[i / 2], x[t][i]);
            }
        }
    }

    __device__ __forceinline__ static float row_sum(float l) {
        l += __shfl_xor_sync(DA_FULL_MASK, l, 1);
        return l + __shfl_xor_sync(DA_FULL_MASK, l, 2);
    }

    __device__ __forceinline__ static void attended(State &st) {
#pragma unroll
        for (int half = 0; half < NR; ++half) st.m[half] = fmaxf(st.m[half], kLowest);
    }

    __device__ __forceinline__ static void publish(State &st, float *dst, int lane, int rows) {
        constexpr int PW = PagedRow<kD>::kWidth;
        const int qd = lane & 3;
#pragma unroll
        for (int half = 0; half < NR; ++half) {
            const float l = row_sum(st.l[half]) * (1.f / kWeight);
            const int r = (lane >> 2) + 8 * half;
            if (r >= rows) continue;
#pragma unroll
            for (int d = 0; d < NT; ++d)
                *reinterpret_cast<float2 *>(dst + r * PW + 8 * d + 2 * qd) =
                    make_float2(st.o[d][2 * half] * (1.f / kWeight), st.o[d][2 * half + 1] * (1.f / kWeight));
            if (qd == 0) *reinterpret_cast<float2 *>(dst + r * PW + kD) = make_float2(st.m[half], l);
        }
    }

    __device__ __forceinline__ static void write(State &st, const PagedParams &p, int item, int rows, int lane) {
        const int qd = lane & 3;
#pragma unroll
        for (int half = 0; half < NR; ++half) {
            const float l = row_sum(st.l[half]);
            const int r = (lane >> 2) + 8 * half;
            if (r >= rows) continue;
            size_t index;
            T *out = out_row<T>(p, item, r, kD, index);
            const float inv = st.m[half] == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
            for (int d = 0; d < NT; ++d)
                *reinterpret_cast<uint32_t *>(out + 8 * d + 2 * qd) =
                    MmaTraits<T>::pack(st.o[d][2 * half] * inv, st.o[d][2 * half + 1] * inv);
            if (qd == 0 && p.lse) p.lse[index] = natural_lse(st.m[half], l * (1.f / kWeight));
        }
    }
};

// As many stages as fit for the number of warps that is fastest, but two for 128 channels: 135 KB under way on every SM are enough
// (64 sequences of 5000 tokens, 1.3 GB: eight warps of three or two stages 206 us, seven of three 211, ten or twelve of two 211,
// whose threads have too few registers).  Smaller heads have units of fewer bytes, so more of them have to be worked on at a
// time: twelve (60 sequences of 3000 tokens with 64, 80, 96 channels: 61, 74, 86 us, with eight warps 80 to 100).  The
// accumulators of 256 channels leave registers for six (265 us; with four warps of three stages 289).
template <int D> struct PagedMmaShape {
    static constexpr int kStage = paged_mma_stage(D);
    static constexpr int kWarps = paged_mma_warps(D);
    static constexpr int kStages = D == 128 ? 2 : (220 * 1024) / (kWarps * kStage);
    static_assert(kStages >= 2, "");
};

// Whether a warp's stretch can hold more than kPagedRun units (65 536 tokens) of an item, by what the tables have room for.
constexpr long long kPagedRun = 4096;
static bool paged_long_runs(const PagedParams &p, int warps) {
    const long long room = p.window > 0 && p.window < p.capacity ? p.window : p.capacity, units = room / kPagedUnit + 2;
    return units > kPagedRun && units * p.n_sequences * p.n_kv_heads * p.groups > kPagedRun * kPagedCtas * warps;
}

template <typename T, int D, bool FULL>
static cudaError_t launch_paged_mma(const PagedParams &p, cudaStream_t stream) {
    using Shape = PagedMmaShape<D>;
    if (paged_long_runs(p, Shape::kWarps)) return launch_paged<PagedMma<T, D, FULL, true>, Shape::kWarps, Shape::kStages>(p, stream);
    return launch_paged<PagedMma<T, D, FULL, false>, Shape::kWarps, Shape::kStages>(p, stream);
}

template <typename T>
static cudaError_t paged_mma(const PagedParams &p, int head_dim, cudaStream_t stream) {
    const bool full = p.group_rows > 8;
    switch (head_dim) {
    case 64: return full ? launch_paged_mma<T, 64, true>(p, stream) : launch_paged_mma<T, 64, false>(p, stream);
    case 80: return full ? launch_paged_mma<T, 80, true>(p, stream) : launch_paged_mma<T, 80, false>(p, stream);
    case 96: return full ? launch_paged_mma<T, 96, true>(p, stream) : launch_paged_mma<T, 96, false>(p, stream);
    case 128: return full ? launch_paged_mma<T, 128, true>(p, stream) : launch_paged_mma<T, 128, false>(p, stream);
    default: return full ? launch_paged_mma<T, 256, true>(p, stream) : launch_paged_mma<T, 256, false>(p, stream);
    }
}

}  // namespace da
