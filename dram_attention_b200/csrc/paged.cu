// Attention over a paged cache: the join of the items that cross CTAs, and the host side.

#include "paged_attn.cuh"

namespace da {

// An item's partial results: n of them, one per warp, from warp `first` of all warps on.
struct JoinSpan {
    int n, first;
    // (the first one begins the item)
    __device__ __forceinline__ int slot(int k) const { return (first + k) * 2 + (k == 0); }
};

// Joins the partial results of an item's rows.  Most CTAs have nothing to do but find that out, so one warp does it.
// A row is shared by `SLICES` warps and, of narrow columns (COLS float4), by the 32 / COLS groups of lanes in each: every one takes
// every so-many-th partial result, several requested together, then they meet in shared memory.  The fewer rows the launch has,
// the more partial results each can have (a line of one head: one from every warp of the GPU), so the more warps share a row and
// the narrower the columns (launch_join).  SLICES 1: a warp per row, but all warps of the CTA row by row for an item of many
// partial results (one long sequence among many short ones).
template <typename T, int D, int WARPS, int SLICES, int COLS>
__global__ void __launch_bounds__(WARPS * 32) paged_join_kernel(const PagedParams p) {
    constexpr int PW = PagedRow<D>::kWidth;
    constexpr int GROUPS = COLS >= 32 ? 1 : 32 / COLS;      // of lanes
    constexpr int NV = (COLS + 31) / 32;                    // float4 columns per lane
    constexpr int ROWS = WARPS / SLICES, AHEAD = 5, FEW = 24;
    constexpr int MAIN_WARPS = sizeof(T) == 4 ? paged_f32_warps(D) : paged_mma_warps(D);
    static_assert((GROUPS & (GROUPS - 1)) == 0 && (GROUPS == 1 || 32 % COLS == 0) && (ROWS == 1 || SLICES == 1) && WARPS <= 32, "");
    __shared__ __align__(16) float sh_o[WARPS][COLS * 4];
    __shared__ float2 sh_ml[WARPS];
    __shared__ JoinSpan sh_span;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = min(lane / COLS, GROUPS - 1), col = COLS >= 32 ? lane : lane % COLS;
    const int item = blockIdx.x;
    const int rows = min(rows_of(p, item) - (int)blockIdx.y * ROWS, ROWS);   // of this CTA (not positive: none)

    if (warp == 0) {
        // (the lengths were complete before the launch that this one follows let it in)
        const int per = p.n_kv_heads * p.groups, b = item / per;
        const Totals units = total_units(p, b, lane);
        const int length = __ldg(p.lengths + b);
        const int mine = span_of(p, length).units;
        JoinSpan s = {0, 0};
        if (mine) {
            const long long begin = units.before * per + (long long)(item % per) * mine;
            const Deal deal(units.all * per);
            const int c0 = deal.cta_of(begin), c1 = deal.cta_of(begin + mine - 1);
            const int w0 = Deal::warp_of(deal.count(c0), (int)(begin - deal.begin(c0)), MAIN_WARPS);
            const int w1 = Deal::warp_of(deal.count(c1), (int)(begin + mine - 1 - deal.begin(c1)), MAIN_WARPS);
            s.first = c0 * MAIN_WARPS + w0;
            s.n = c1 * MAIN_WARPS + w1 - s.first + 1;
        }
        if (lane == 0) {
            sh_span = s;
            if (blockIdx.y == 0 && blockIdx.z == 0 && item % per == 0 && (length < 0 || length > p.capacity))
                atomicOr(p.status, DA_STATUS_BAD_POSITION);
        }
    }
    __syncthreads();
    const JoinSpan span = sh_span;
    griddep_wait();
    griddep_launch_dependents();
    if (span.n == 1 || rows <= 0) return;          // one warp had all of it, and wrote it

    size_t index = 0;
    T *out = out_row<T>(p, item, blockIdx.y * ROWS, D, index) + blockIdx.z * (COLS * 4);
    const bool writes_lse = p.lse != nullptr && blockIdx.z == 0;
    if (span.n == 0) {                             // nothing to attend to
        for (int i = threadIdx.x; i < rows * COLS * 4; i += WARPS * 32) out[i / (COLS * 4) * D + i % (COLS * 4)] = from_float<T>(0.f);
        if (writes_lse)
            for (int r = threadIdx.x; r < rows; r += WARPS * 32) p.lse[index + r] = -INFINITY;
        return;
    }

    PartialSum x[NV];
    // every step-th partial result of a row of this CTA, from one on
    auto gather = [&](int row, int from, int step) {
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i].clear();
        const float *base = p.partials + (size_t)(blockIdx.y * ROWS + row) * PW;
        const size_t slot = (size_t)p.group_rows * PW;
        for (int first = from * GROUPS + group; first < span.n; first += step * GROUPS * AHEAD) {
            float4 v[NV][AHEAD];
            float2 ml[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = first + a * step * GROUPS;
                const float *src = base + span.slot(min(k, span.n - 1)) * slot;
                ml[a] = __ldcg(reinterpret_cast<const float2 *>(src + D));
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    v[i][a] = __ldcg(reinterpret_cast<const float4 *>(src) + blockIdx.z * COLS + min(col + 32 * i, COLS - 1));
                if (k >= span.n) ml[a] = make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i].add(ml, v[i]);
        }
#pragma unroll
        for (int off = COLS; off < GROUPS * COLS; off <<= 1) {
            const float2 ml[1] = {make_float2(__shfl_xor_sync(DA_FULL_MASK, x[0].m, off), __shfl_xor_sync(DA_FULL_MASK, x[0].l, off))};
            const float4 v[1] = {make_float4(__shfl_xor_sync(DA_FULL_MASK, x[0].o.x, off), __shfl_xor_sync(DA_FULL_MASK, x[0].o.y, off),
                                             __shfl_xor_sync(DA_FULL_MASK, x[0].o.z, off), __shfl_xor_sync(DA_FULL_MASK, x[0].o.w, off))};
            x[0].add(ml, v);
        }
    };
    if (SLICES == 1 && span.n <= FEW) {
        if (warp >= rows) return;
        gather(warp, 0, 1);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < COLS) store_divided(out + (size_t)warp * D + 4 * (lane + 32 * i), x[i].o, x[i].l);
        if (lane == 0 && writes_lse) p.lse[index + warp] = natural_lse(x[0].m, x[0].l);
        return;
    }
    for (int row = 0; row < rows; ++row) {
        gather(row, warp, WARPS);
        if (row > 0) __syncthreads();              // the row before has been read
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < COLS) reinterpret_cast<float4 *>(sh_o[warp])[lane + 32 * i] = x[i].o;
        if (lane == 0) sh_ml[warp] = make_float2(x[0].m, x[0].l);
        __syncthreads();
        // a lane of each warp has the weight of one warp's sum, a thread adds up one channel of all
        const float2 w = lane < WARPS ? sh_ml[lane] : make_float2(-INFINITY, 0.f);
        float m = w.x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(DA_FULL_MASK, m, off));
        const float k = fast_exp2(w.x - (m == -INFINITY ? 0.f : m));
        float l = w.y * k;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(DA_FULL_MASK, l, off);
        if (warp * 32 < COLS * 4) {                // (whole warps: the weights travel by shuffles)
            const int c = threadIdx.x;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) sum = fmaf(sh_o[i][min(c, COLS * 4 - 1)], __shfl_sync(DA_FULL_MASK, k, i), sum);
            if (c < COLS * 4) out[(size_t)row * D + c] = from_float<T>(l > 0.f ? sum / l : 0.f);
            if (c == 0 && writes_lse) p.lse[index + row] = natural_lse(m, l);
        }
    }
}

template <typename T, int D> static cudaError_t launch_join(const PagedParams &p, cudaStream_t stream) {
    constexpr int ALL = D / 4, NARROW = D % 32 == 0 ? 8 : 4, BLOCKS = ALL / NARROW;
    const long long items = (long long)p.n_sequences * p.n_kv_heads * p.groups, rows = items * p.group_rows;
    const unsigned x = (unsigned)items;
    // 1024 threads a row as long as all CTAs are on the GPU at once, with narrow columns if even then; then 256, while an item
    // has more than a few partial results on average (60 sequences, 480 items: a CTA per row 124 us, per item 117)
    if (rows * BLOCKS <= 2 * kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 32, 32, NARROW>, dim3(x, p.group_rows, BLOCKS), dim3(1024), (size_t)0, stream, p);
    if (rows <= 2 * kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 32, 32, ALL>, dim3(x, p.group_rows), dim3(1024), (size_t)0, stream, p);
    if (items <= 2 * kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 8, 8, ALL>, dim3(x, p.group_rows), dim3(256), (size_t)0, stream, p);
    return launch_dependent(paged_join_kernel<T, D, 8, 1, ALL>, dim3(x, (p.group_rows + 7) / 8), dim3(256), (size_t)0, stream, p);
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
    const int warps = dtype == DA_F32 ? paged_f32_warps(head_dim) : paged_mma_warps(head_dim);
    return (size_t)kPagedCtas * warps * 2 * group_rows(rep, head_dim, dtype) * (head_dim + 4) * sizeof(float);
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
    p.partials = static_cast<float *>(a.workspace);
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
