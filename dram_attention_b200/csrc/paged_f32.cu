// Attention over a paged cache: float32, on CUDA cores.

#include "paged_attn.cuh"

namespace da {

// Eight lanes share a token (lane j has the 16-byte pieces j, j + 8, ... of its rows, which a quarter of a warp reads without
// bank conflicts), four tokens at a time, up to R query rows at once.  The four token groups of a warp keep a running
// softmax each and meet when the item is done.
template <int D_, int R>
struct PagedSimt {
    using Elem = float;
    static constexpr int kD = D_, kRows = R;
    static constexpr int ROWB = kD * 4, kPitch = 2 * ROWB;
    static constexpr int PIECES = kD / 4, NC = (PIECES + 7) / 8;

    struct State {
        float4 q[R][NC], o[R][NC];
        float m[R], l[R];
    };

    __device__ __forceinline__ static bool has(int j, int i) { return PIECES % 8 == 0 || j + 8 * i < PIECES; }

    __device__ __forceinline__ static void begin(State &st, const PagedParams &p, int b, int head, int group, int rows, int lane) {
        const int j = lane & 7;
        const int head0 = head * p.rep + group * p.group_rows;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float *row = reinterpret_cast<const float *>(p.q) + b * p.q_seq + (head0 + (r < rows ? r : 0)) * p.q_head;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                st.q[r][i] = has(j, i) && r < rows ? *reinterpret_cast<const float4 *>(row + 4 * (j + 8 * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                st.o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            st.m[r] = -INFINITY;
            st.l[r] = 0.f;
        }
    }

    __device__ __forceinline__ static void consume(State &st, const unsigned char *unit, uint32_t mask, int lane, float scale_log2) {
        const int g = lane >> 3, j = lane & 7;
        float s[4][R];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const unsigned char *key = unit + (g + 4 * t) * kPitch + 16 * j;
#pragma unroll
            for (int r = 0; r < R; ++r) s[t][r] = 0.f;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (!has(j, i)) continue;
                const float4 k = *reinterpret_cast<const float4 *>(key + 128 * i);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float4 q = st.q[r][i];
                    s[t][r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[t][r]))));
                }
            }
        }
#pragma unroll
        for (int off = 1; off <= 4; off <<= 1)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < R; ++r) s[t][r] += __shfl_xor_sync(DA_FULL_MASK, s[t][r], off);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = st.m[r];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                s[t][r] = (mask >> (g + 4 * t)) & 1 ? s[t][r] * scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[t][r]);
            }
            const float ms = mx == -INFINITY ? 0.f : mx;
            const float alpha = fast_exp2(st.m[r] - ms);
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                s[t][r] = fast_exp2(s[t][r] - ms);
                sum += s[t][r];
            }
            st.l[r] = st.l[r] * alpha + sum;
            st.m[r] = mx;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                st.o[r][i].x *= alpha;
                st.o[r][i].y *= alpha;
                st.o[r][i].z *= alpha;
                st.o[r][i].w *= alpha;
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const unsigned char *value = unit + (g + 4 * t) * kPitch + ROWB + 16 * j;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (!has(j, i)) continue;
                const float4 v = *reinterpret_cast<const float4 *>(value + 128 * i);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    st.o[r][i].x = fmaf(s[t][r], v.x, st.o[r][i].x);
                    st.o[r][i].y = fmaf(s[t][r], v.y, st.o[r][i].y);
                    st.o[r][i].z = fmaf(s[t][r], v.z, st.o[r][i].z);
                    st.o[r][i].w = fmaf(s[t][r], v.w, st.o[r][i].w);
                }
            }
        }
    }

    // the four token groups of the warp in one
    __device__ __forceinline__ static float sum_groups(float x) {
        x += __shfl_xor_sync(DA_FULL_MASK, x, 8);
        return x + __shfl_xor_sync(DA_FULL_MASK, x, 16);
    }
    __device__ __forceinline__ static void join(State &st) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float m = fmaxf(st.m[r], __shfl_xor_sync(DA_FULL_MASK, st.m[r], 8));
            m = fmaxf(m, __shfl_xor_sync(DA_FULL_MASK, m, 16));
            const float w = fast_exp2(st.m[r] - (m == -INFINITY ? 0.f : m));
            st.m[r] = m;
            st.l[r] = sum_groups(st.l[r] * w);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                st.o[r][i].x = sum_groups(st.o[r][i].x * w);
                st.o[r][i].y = sum_groups(st.o[r][i].y * w);
                st.o[r][i].z = sum_groups(st.o[r][i].z * w);
                st.o[r][i].w = sum_groups(st.o[r][i].w * w);
            }
        }
    }

    __device__ __forceinline__ static void publish(State &st, float *dst, int lane, int rows) {
        constexpr int PW = PagedRow<kD>::kWidth;
        const int j = lane & 7;
        join(st);
        if (lane >= 8) return;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= rows) continue;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (has(j, i)) *reinterpret_cast<float4 *>(dst + r * PW + 4 * (j + 8 * i)) = st.o[r][i];
            if (j == 0) *reinterpret_cast<float2 *>(dst + r * PW + kD) = make_float2(st.m[r], st.l[r]);
        }
    }

    __device__ __forceinline__ static void write(State &st, const PagedParams &p, int item, int rows, int lane) {
        const int j = lane & 7;
        join(st);
        if (lane >= 8) return;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= rows) continue;
            size_t index;
            float *out = out_row<float>(p, item, r, kD, index);
            const float l = st.l[r];
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const float4 o = st.o[r][i];
                if (has(j, i))
                    *reinterpret_cast<float4 *>(out + 4 * (j + 8 * i)) =
                        l > 0.f ? make_float4(o.x / l, o.y / l, o.z / l, o.w / l) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (j == 0 && p.lse) p.lse[index] = natural_lse(st.m[r], l);
        }
    }
};

// As few rows as the group has: fewer instructions per unit, and less code, which a short call fetches from memory.
// (warps x stages x 16 tokens of 8 D bytes: 160 to 197 KB; more than 8 warps would have 168 registers)
template <int D, int STAGES> static cudaError_t paged_simt(const PagedParams &p, cudaStream_t stream) {
    constexpr int MOST = paged_f32_rows(D), WARPS = paged_f32_warps(D);
    if (p.group_rows <= 1) return launch_paged<PagedSimt<D, 1>, WARPS, STAGES>(p, stream);
    if constexpr (MOST > 2) {
        if (p.group_rows <= 2) return launch_paged<PagedSimt<D, 2>, WARPS, STAGES>(p, stream);
    }
    if constexpr (MOST > 4) {
        if (p.group_rows <= 4) return launch_paged<PagedSimt<D, 4>, WARPS, STAGES>(p, stream);
    }
    return launch_paged<PagedSimt<D, MOST>, WARPS, STAGES>(p, stream);
}

cudaError_t paged_attention_f32(const PagedParams &p, int head_dim, cudaStream_t stream) {
    switch (head_dim) {
    case 64: return paged_simt<64, 3>(p, stream);
    case 80: return paged_simt<80, 2>(p, stream);
    case 96: return paged_simt<96, 2>(p, stream);
    case 128: return paged_simt<128, 2>(p, stream);
    default: return paged_simt<256, 2>(p, stream);
    }
}

}  // namespace da
