// Attention over a paged cache: the join of the items that cross CTAs, and the host side.

#include "paged_attn.cuh"

namespace da {

// One CTA per item and block of query rows.  WARPS / rows per CTA warps share a row (each every so-many-th partial result):
// 32 of them when there are few rows and so, for a long line, many partial results of each (148 results of a row are one
// round trip to memory then); one per row when there are many.
template <typename T, int D, int WARPS, int SLICES>
__global__ void __launch_bounds__(WARPS * 32) paged_join_kernel(const PagedParams p) {
    constexpr int PW = PagedRow<D>::kWidth, COLS = D / 4;
    constexpr int NV = (COLS + 31) / 32;           // float4 columns per lane
    constexpr int ROWS = WARPS / SLICES, AHEAD = 5;
    __shared__ __align__(16) float sh_o[SLICES > 1 ? WARPS : 1][D];
    __shared__ float2 sh_ml[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int item = blockIdx.x;
    const int per = p.n_kv_heads * p.groups, b = item / per;
    const int row = blockIdx.y * ROWS + warp / SLICES, slice = warp % SLICES;
    const int rows = rows_of(p, item);

    // (the lengths were complete before the launch that this one follows let it in)
    const Totals units = total_units(p, b, lane);
    const int length = __ldg(p.lengths + b);
    const int mine = span_of(p, length).units;
    const long long begin = units.before * per + (long long)(item % per) * mine;
    const Deal deal(units.all * per);
    int c0 = 0, c1 = 0;
    if (mine) c0 = deal.cta_of(begin), c1 = deal.cta_of(begin + mine - 1);

    griddep_wait();
    griddep_launch_dependents();
    if (blockIdx.y == 0 && threadIdx.x == 0 && item % per == 0 && (length < 0 || length > p.capacity)) atomicOr(p.status, DA_STATUS_BAD_POSITION);
    size_t index = 0;
    T *out = out_row<T>(p, item, row < rows ? row : 0, D, index);
    if (mine == 0) {                               // nothing to attend to
        if (slice == 0 && row < rows) {
            for (int c = lane; c < D; c += 32) out[c] = from_float<T>(0.f);
            if (lane == 0 && p.lse) p.lse[index] = -INFINITY;
        }
        return;
    }
    if (c0 == c1) return;                          // one CTA had all of it

    PartialSum x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i].clear();
    if (row < rows) {
        for (int first = c0 + slice; first <= c1; first += SLICES * AHEAD) {
            float4 v[NV][AHEAD];
            float2 ml[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int c = min(first + a * SLICES, c1);
                const float *src = p.cta_partials + (((size_t)c * 2 + (c == c0 ? 1 : 0)) * p.group_rows + row) * PW;
                ml[a] = __ldcg(reinterpret_cast<const float2 *>(src + D));
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    v[i][a] = __ldcg(reinterpret_cast<const float4 *>(src) + min(lane + 32 * i, COLS - 1));
                if (first + a * SLICES > c1) ml[a] = make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i].add(ml, v[i]);
        }
    }
    if constexpr (SLICES == 1) {
        if (row >= rows) return;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < COLS) store_divided(out + 4 * (lane + 32 * i), x[i].o, x[i].l);
        if (lane == 0 && p.lse) p.lse[index] = natural_lse(x[0].m, x[0].l);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < COLS) reinterpret_cast<float4 *>(sh_o[warp])[lane + 32 * i] = x[i].o;
        if (lane == 0) sh_ml[warp] = make_float2(x[0].m, x[0].l);
        __syncthreads();
        // one row per CTA: a thread adds up one channel of all slices, a lane of each warp the weights of one
        static_assert(ROWS == 1 && SLICES == 32, "");
        const float2 w = sh_ml[lane];
        float m = w.x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(DA_FULL_MASK, m, off));
        const float k = fast_exp2(w.x - (m == -INFINITY ? 0.f : m));
        float l = w.y * k;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(DA_FULL_MASK, l, off);
        const int c = threadIdx.x;
        if (row >= rows || warp * 32 >= D) return;   // (whole warps: the weights travel by shuffles)
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < SLICES; ++i) sum = fmaf(sh_o[i][min(c, D - 1)], __shfl_sync(DA_FULL_MASK, k, i), sum);
        if (c < D) out[c] = from_float<T>(l > 0.f ? sum / l : 0.f);
        if (c == 0 && p.lse) p.lse[index] = natural_lse(m, l);
    }
}

template <typename T, int D> static cudaError_t launch_join(const PagedParams &p, cudaStream_t stream) {
    const long long items = (long long)p.n_sequences * p.n_kv_heads * p.groups;
    if (items * p.group_rows <= 2 * kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 32, 32>, dim3((unsigned)items, p.group_rows), dim3(1024), (size_t)0, stream, p);
    return launch_dependent(paged_join_kernel<T, D, 8, 1>, dim3((unsigned)items, (p.group_rows + 7) / 8), dim3(256), (size_t)0, stream, p);
}

template <typename T> static cudaError_t join(const PagedParams &p, int head_dim, cudaStream_t stream) {
    switch (head_dim) {
    case 64: return launch_join<T, 64>(p, stream);
    case 80: return launch_join<T, 80>(p, stream);
    case 96: return launch_join<T, 96>(p, stream);
    case 128: return launch_join<T, 128>(p, stream);
    default: return launch_join<T, 256>(p, stream);
    }
}

// Query rows of a KV head that share a pass over its keys and values: as equal groups as possible.
static int group_rows(int64_t rep, int64_t head_dim, int64_t dtype) {
    const int64_t most = dtype == DA_F32 ? paged_f32_rows((int)head_dim) : kPagedMmaRows;
    const int64_t groups = (rep + most - 1) / most;
    return (int)((rep + groups - 1) / groups);
}

static bool paged_head_dim(int64_t d) { return d == 64 || d == 80 || d == 96 || d == 128 || d == 256; }

static bool paged_shape(int64_t rep, int64_t head_dim, int64_t dtype) {
    return rep >= 1 && rep <= 256 && paged_head_dim(head_dim) && dtype >= DA_F32 && dtype <= DA_BF16;
}

}  // namespace da

extern "C" size_t da_paged_attention_workspace_bytes(int rep, int head_dim, int dtype) {
    using namespace da;
    if (!paged_shape(rep, head_dim, dtype)) return 0;
    return (size_t)kPagedCtas * (kPagedMaxWarps + 2) * group_rows(rep, head_dim, dtype) * (head_dim + 4) * sizeof(float);
}

extern "C" int da_paged_attention(const da_paged_attention_args *args) {
    using namespace da;
    if (!args) return DA_ERR_NULL;
    const da_paged_attention_args &a = *args;
    if (!a.q || !a.pages || !a.page_table || !a.lengths || !a.out || !a.workspace || !a.status) return DA_ERR_NULL;
    if (a.dtype < DA_F32 || a.dtype > DA_BF16) return DA_ERR_DTYPE;
    if (a.n_sequences < 1 || a.n_kv_heads < 1 || a.rep < 1 || a.page_size < 1 || a.n_pages < 1 || a.table_columns < 1 ||
        a.window < 0 || a.n_sequences > 0x7fffffff || a.n_kv_heads > 1 << 16 || a.page_size > 1 << 20 || a.n_pages > 0x7fffffff ||
        a.table_columns > 0x7fffffff || a.table_columns * a.page_size > 0x7fffff00 || a.window > 0x7fffffff)
        return DA_ERR_SHAPE;
    if (!paged_shape(a.rep, a.head_dim, a.dtype)) return DA_ERR_UNSUPPORTED;
    const int esize = a.dtype == DA_F32 ? 4 : 2;
    const uintptr_t rows = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.pages) | reinterpret_cast<uintptr_t>(a.out) |
                           reinterpret_cast<uintptr_t>(a.workspace);
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.page_table) | reinterpret_cast<uintptr_t>(a.lengths) |
                            reinterpret_cast<uintptr_t>(a.lse) | reinterpret_cast<uintptr_t>(a.status);
    if ((rows & 15) || (words & 3) ||
        (a.q_strides[0] | a.q_strides[1] | a.page_stride | a.page_head_stride) % (16 / esize))
        return DA_ERR_ALIGN;
    if (a.workspace_bytes < (int64_t)da_paged_attention_workspace_bytes((int)a.rep, (int)a.head_dim, (int)a.dtype)) return DA_ERR_WORKSPACE;

    PagedParams p = {};
    p.q = static_cast<const unsigned char *>(a.q), p.q_seq = a.q_strides[0], p.q_head = a.q_strides[1];
    p.pages = static_cast<const unsigned char *>(a.pages);
    p.page_stride = a.page_stride, p.page_head_stride = a.page_head_stride;
    p.n_pages = (int)a.n_pages, p.page_size = (int)a.page_size;
    p.table = a.page_table, p.table_stride = a.table_stride;
    p.capacity = (int)(a.table_columns * a.page_size);
    // t / page_size for 0 <= t < 2^31 by a multiplication (Granlund and Montgomery): floor(2^(31 + l) / d) + 1 with 2^l >= d
    int l = 0;
    while ((1 << l) < p.page_size) ++l;
    p.page_mul = (uint32_t)((1ull << (31 + l)) / (unsigned)p.page_size + 1);
    p.page_shift = 31 + l;
    p.whole = p.page_size % kPagedUnit == 0;
    p.lengths = a.lengths, p.n_sequences = (int)a.n_sequences, p.window = (int)a.window;
    p.out = static_cast<unsigned char *>(a.out), p.lse = a.lse, p.status = a.status;
    p.n_kv_heads = (int)a.n_kv_heads, p.rep = (int)a.rep;
    p.group_rows = group_rows(a.rep, a.head_dim, a.dtype);
    p.groups = (p.rep + p.group_rows - 1) / p.group_rows;
    if (a.n_sequences * a.n_kv_heads * p.groups > 0x7fffffff) return DA_ERR_SHAPE;
    p.cta_partials = static_cast<float *>(a.workspace);
    p.warp_partials = p.cta_partials + (size_t)kPagedCtas * 2 * p.group_rows * (a.head_dim + 4);
    p.scale_log2 = (float)(a.scale * 1.4426950408889634);
    cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
    cudaError_t e;
    switch (a.dtype) {
    case DA_F32: e = paged_attention_f32(p, (int)a.head_dim, stream); break;
    case DA_F16: e = paged_attention_f16(p, (int)a.head_dim, stream); break;
    default: e = paged_attention_bf16(p, (int)a.head_dim, stream); break;
    }
    if (e != cudaSuccess) return (int)e;
    switch (a.dtype) {
    case DA_F32: return (int)join<float>(p, (int)a.head_dim, stream);
    case DA_F16: return (int)join<__half>(p, (int)a.head_dim, stream);
    default: return (int)join<__nv_bfloat16>(p, (int)a.head_dim, stream);
    }
}
