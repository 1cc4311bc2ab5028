// Attention over a paged cache: float32, on CUDA cores.

#include "paged_attn.cuh"

namespace da {

// Eight lanes share a token (lane j has the 16-byte pieces j, j + 8, ... of its rows, which a quarter of a warp reads without
// bank conflicts), four tokens at a time, up to R query rows at once.  The eight lanes' shares of the logits are added up so that each
// lane ends with the logits of one row, whose softmax it keeps: halves are exchanged, not copies (28 shuffles for eight rows and
// four tokens instead of 96, and an eighth of the exponentials); the weights then go round by shuffles.  The four token groups
// of a warp keep a running softmax each and meet when the item is done.  Many query rows stay in shared memory, where a piece is read once for the warp's
// sixteen tokens (in registers there would be room for half as many, and the keys and values would be read twice as often: 256
// channels, four rows 147 us, so 97), few in registers (4096 tokens, 64 channels, four rows: 9.3 us, so 8.7).
template <int D_, int R>
struct PagedSimt {
    using Elem = float;
    static constexpr int kD = D_, kRows = R;
    static constexpr int ROWB = kD * 4, kPitch = 2 * ROWB, kTogether = kPagedUnit, kStageBytes = kPagedUnit * kPitch;
    __device__ __forceinline__ static constexpr int offset(int t) { return t * kPitch; }
    static constexpr int PIECES = kD / 4, NC = (PIECES + 7) / 8;

    static constexpr bool kInRegisters = R * NC <= 8;
    static constexpr int kScratch = kInRegisters ? 0 : R * ROWB;   // query rows of a warp

    struct State {
        float4 qr[kInRegisters ? R : 1][NC];
        const float4 *q;                           // or this lane's first piece of row 0, in shared memory
        float4 o[R][NC];
        float m, l;                                // of row (lane % 8) % R
    };

    __device__ __forceinline__ static bool has(int j, int i) { return PIECES % 8 == 0 || j + 8 * i < PIECES; }

    __device__ __forceinline__ static void begin(State &st, const PagedParams &p, int b, int head, int group, int rows, int lane, unsigned char *scratch) {
        const int head0 = head * p.rep + group * p.group_rows;
        const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
        const float *src = reinterpret_cast<const float *>(p.q) + b * p.q_seq + head0 * p.q_head;
        if constexpr (kInRegisters) {
            const int j = lane & 7;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < NC; ++i)
                    st.qr[r][i] = has(j, i) && r < rows ? *reinterpret_cast<const float4 *>(src + r * p.q_head + 4 * (j + 8 * i)) : none;
        } else {
            float4 *q = reinterpret_cast<float4 *>(scratch);
#pragma unroll
            for (int r = 0; r < R; ++r)
                for (int c = lane; c < PIECES; c += 32)
                    q[r * PIECES + c] = r < rows ? *reinterpret_cast<const float4 *>(src + r * p.q_head + 4 * c) : none;
            __syncwarp();
            st.q = q + (lane & 7);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < NC; ++i) st.o[r][i] = none;
        }
        st.m = -INFINITY;
        st.l = 0.f;
    }

    // the lane of this token group that has row r
    __device__ __forceinline__ static int keeper(int lane, int r) { return (lane & 24) | r; }

    __device__ __forceinline__ static void consume(State &st, const unsigned char *unit, uint32_t mask, int lane, float scale_log2) {
        const int g = lane >> 3, j = lane & 7;
        float s[4][R];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < R; ++r) s[t][r] = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (!has(j, i)) continue;
            float4 k[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) k[t] = *reinterpret_cast<const float4 *>(unit + (g + 4 * t) * kPitch + 16 * j + 128 * i);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float4 q;
                if constexpr (kInRegisters) q = st.qr[r][i];
                else q = st.q[r * PIECES + 8 * i];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    s[t][r] = fmaf(q.x, k[t].x, fmaf(q.y, k[t].y, fmaf(q.z, k[t].z, fmaf(q.w, k[t].w, s[t][r]))));
            }
        }
        // rows in halves: a lane keeps those whose lowest bit is its own, then those whose next bit is
        int left = R;
#pragma unroll
        for (int off = 1; off <= 4; off <<= 1) {
            if (off < R) {
                const bool odd = lane & off;
                left /= 2;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int r = 0; r < R / 2; ++r)
                        if (r < left) {
                            const float mine = odd ? s[t][2 * r + 1] : s[t][2 * r], other = odd ? s[t][2 * r] : s[t][2 * r + 1];
                            s[t][r] = mine + __shfl_xor_sync(DA_FULL_MASK, other, off);
                        }
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) s[t][0] += __shfl_xor_sync(DA_FULL_MASK, s[t][0], off);
            }
        }
        float w[4], m = st.m;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            w[t] = (mask >> (g + 4 * t)) & 1 ? s[t][0] * scale_log2 : -INFINITY;
            m = fmaxf(m, w[t]);
        }
        const float ms = m == -INFINITY ? 0.f : m;
        const float alpha = fast_exp2(st.m - ms);
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = fast_exp2(w[t] - ms);
        st.l = st.l * alpha + ((w[0] + w[1]) + (w[2] + w[3]));
        st.m = m;
        if (__any_sync(DA_FULL_MASK, alpha != 1.f)) {   // once the maxima have settled there is nothing to rescale
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float a = __shfl_sync(DA_FULL_MASK, alpha, keeper(lane, r));
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    st.o[r][i].x *= a;
                    st.o[r][i].y *= a;
                    st.o[r][i].z *= a;
                    st.o[r][i].w *= a;
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const unsigned char *value = unit + (g + 4 * t) * kPitch + ROWB + 16 * j;
            float4 v[NC];
#pragma unroll
            for (int i = 0; i < NC; ++i) v[i] = has(j, i) ? *reinterpret_cast<const float4 *>(value + 128 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float a = __shfl_sync(DA_FULL_MASK, w[t], keeper(lane, r));
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    st.o[r][i].x = fmaf(a, v[i].x, st.o[r][i].x);
                    st.o[r][i].y = fmaf(a, v[i].y, st.o[r][i].y);
                    st.o[r][i].z = fmaf(a, v[i].z, st.o[r][i].z);
                    st.o[r][i].w = fmaf(a, v[i].w, st.o[r][i].w);
                }
            }
        }
    }

    // the four token groups of the warp in one
    __device__ __forceinline__ static float sum_groups(float x) {
        x += __shfl_xor_sync(DA_FULL_MASK, x, 8);
        return x + __shfl_xor_sync(DA_FULL_MASK, x, 16);
    }
    __device__ __forceinline__ static void join(State &st, int lane) {
        float m = fmaxf(st.m, __shfl_xor_sync(DA_FULL_MASK, st.m, 8));
        m = fmaxf(m, __shfl_xor_sync(DA_FULL_MASK, m, 16));
        const float w = fast_exp2(st.m - (m == -INFINITY ? 0.f : m));
        st.m = m;
        st.l = sum_groups(st.l * w);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float a = __shfl_sync(DA_FULL_MASK, w, keeper(lane, r));
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                st.o[r][i].x = sum_groups(st.o[r][i].x * a);
                st.o[r][i].y = sum_groups(st.o[r][i].y * a);
                st.o[r][i].z = sum_groups(st.o[r][i].z * a);
                st.o[r][i].w = sum_groups(st.o[r][i].w * a);
            }
        }
    }

    __device__ __forceinline__ static void attended(State &st) { st.m = fmaxf(st.m, kLowest); }

    __device__ __forceinline__ static void publish(State &st, float *dst, int lane, int rows) {
        constexpr int PW = PagedRow<kD>::kWidth;
        const int j = lane & 7;
        join(st, lane);
        if (lane >= 8) return;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= rows) continue;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (has(j, i)) *reinterpret_cast<float4 *>(dst + r * PW + 4 * (j + 8 * i)) = st.o[r][i];
        }
        if (j < min(rows, R)) *reinterpret_cast<float2 *>(dst + j * PW + kD) = make_float2(st.m, st.l);
    }

    __device__ __forceinline__ static void write(State &st, const PagedParams &p, int item, int rows, int lane) {
        const int j = lane & 7;
        join(st, lane);
        size_t index;
        if (lane < min(rows, R) && p.lse) {
            out_row<float>(p, item, lane, kD, index);
            p.lse[index] = natural_lse(st.m, st.l);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float m = __shfl_sync(DA_FULL_MASK, st.m, keeper(lane, r)), l = __shfl_sync(DA_FULL_MASK, st.l, keeper(lane, r));
            if (r >= rows || lane >= 8) continue;
            float *out = out_row<float>(p, item, r, kD, index);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const float4 o = st.o[r][i];
                if (has(j, i))
                    *reinterpret_cast<float4 *>(out + 4 * (j + 8 * i)) =
                        m == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
            }
        }
    }
};

// As few rows as the group has: fewer instructions per unit, and less code, which a short call fetches from memory.
// (warps x stages x 16 tokens of 8 D bytes, and the query rows: 184 to 221 KB; more than 8 warps would have 168 registers)
template <int D, int STAGES, int ROWS> static cudaError_t paged_simt(const PagedParams &p, cudaStream_t stream) {
    constexpr int FEWER = ROWS / 2;
    if constexpr (ROWS > 1) {
        if (p.group_rows <= FEWER) return paged_simt<D, STAGES, FEWER>(p, stream);
    }
    return launch_paged<PagedSimt<D, ROWS>, paged_f32_warps(D), STAGES>(p, stream);
}

cudaError_t paged_attention_f32(const PagedParams &p, int head_dim, cudaStream_t stream) {
    switch (head_dim) {
    case 64: return paged_simt<64, 3, paged_f32_rows(64)>(p, stream);
    case 80: return paged_simt<80, 2, paged_f32_rows(80)>(p, stream);
    case 96: return paged_simt<96, 2, paged_f32_rows(96)>(p, stream);
    case 128: return paged_simt<128, 2, paged_f32_rows(128)>(p, stream);
    default: return paged_simt<256, 2, paged_f32_rows(256)>(p, stream);
    }
}

}  // namespace da
