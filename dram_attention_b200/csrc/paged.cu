// Attention over a paged cache: the join of the items that cross warps, and the host side.

#include "paged_attn.cuh"

namespace da {

// Sums the partial results of one row: part k (of n) is the one of warp first + k; the first one begins the item.  A thread has
// NV float4 columns of every step-th part, from one on, several requested together.
template <int NV> struct RowSum {
    PartialSum x[NV];
    // row: the row in slot 0 of warp 0; columns in float4, spaced 32
    template <int PW> __device__ __forceinline__ void gather(const float *row, size_t slot, int d, int first, int n, int from, int step, int col, int last_col) {
        constexpr int AHEAD = 5;
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i].clear();
        for (int k0 = from; k0 < n; k0 += step * AHEAD) {
            float4 v[NV][AHEAD];
            float2 ml[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = min(k0 + a * step, n - 1);
                const float *src = row + ((size_t)(first + k) * 2 + (k == 0)) * slot;
                ml[a] = __ldcg(reinterpret_cast<const float2 *>(src + d));
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i][a] = __ldcg(reinterpret_cast<const float4 *>(src) + min(col + 32 * i, last_col));
                if (k0 + a * step >= n) ml[a] = make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i].add(ml, v[i]);
        }
    }
};

// Joins the partial results of the items that cross warps, and writes the rows of sequences of length 0.
//
// MANY false: a CTA has one row of one item and COLS float4 columns of it.  Its warps and, of narrow columns, the 32 / COLS groups of
// lanes in each share the parts and meet in shared memory.  The fewer rows the launch has, the more parts each can have (a line
// of one head: one from every warp of the GPU), so the more warps share a row and the narrower the columns.
// Where the parts lie follows from the lengths, and is worked out while the first launch is at work.
// MANY true: a warp has one row of one item, of few parts; an item of more (one long sequence among many short ones) is
// taken by all warps of the CTA together.  Most of very many items have only one part, and what the warps noted says so in one read.
template <typename T, int D, int WARPS, int COLS, bool MANY>
__global__ void __launch_bounds__(WARPS * 32) paged_join_kernel(const PagedParams p) {
    constexpr int PW = PagedRow<D>::kWidth;
    constexpr int GROUPS = COLS >= 32 ? 1 : 32 / COLS;      // of lanes
    constexpr int NV = (COLS + 31) / 32;                    // float4 columns per lane
    constexpr int FEW = 24;
    constexpr int MAIN_WARPS = sizeof(T) == 4 ? paged_f32_warps(D) : paged_mma_warps(D);
    static_assert((GROUPS & (GROUPS - 1)) == 0 && (GROUPS == 1 || 32 % COLS == 0) && WARPS <= 32, "");
    __shared__ __align__(16) float sh_o[WARPS][COLS * 4];
    __shared__ float2 sh_ml[WARPS];
    __shared__ int2 sh_span[MANY ? WARPS : 1];
    __shared__ int sh_length;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = min(lane / COLS, GROUPS - 1), col = COLS >= 32 ? lane : lane % COLS;
    const int column0 = MANY ? 0 : blockIdx.z * COLS;
    const bool writes_lse = p.lse != nullptr && column0 == 0;
    const size_t slot = (size_t)p.group_rows * PW;
    // the row of this warp
    const long long task = MANY ? (long long)blockIdx.x * WARPS + warp : 0;
    const int item = MANY ? (int)(task / p.group_rows) : blockIdx.x;
    const int row = MANY ? (int)(task - (long long)item * p.group_rows) : blockIdx.y;
    const int per = p.n_kv_heads * p.groups, b = item / per;
    const bool there = b < p.n_sequences && row < rows_of(p, item);
    int2 span = make_int2(0, 0);                   // warps the item begins and ends in
    int length = 1;
    if constexpr (!MANY) {
        // (the lengths were complete before the launch that this one follows let it in)
        if (warp == 0) {
            const Survey survey(p, lane);
            length = __ldg(p.lengths + b);
            const int mine = span_of(p, length).units;
            if (mine) {
                const long long begin = survey.before(p, b, lane) * per + (long long)(item % per) * mine;
                const Deal deal(survey.total() * per, MAIN_WARPS);
                const int c0 = deal.cta_of(begin), c1 = deal.cta_of(begin + mine - 1);
                span.x = c0 * MAIN_WARPS + Deal::warp_of(deal.count(c0), (int)(begin - deal.begin(c0)), MAIN_WARPS);
                span.y = c1 * MAIN_WARPS + Deal::warp_of(deal.count(c1), (int)(begin + mine - 1 - deal.begin(c1)), MAIN_WARPS);
            }
            if (lane == 0) {
                sh_span[0] = span;
                sh_length = length;
            }
        }
        __syncthreads();
        span = sh_span[0], length = sh_length;
    }
    griddep_wait();
    griddep_launch_dependents();
    if (MANY && there) {
        span = __ldcg(p.spans + item);             // (of no meaning for a sequence of length 0)
        length = __ldg(p.lengths + b);
    }
    if (row == 0 && there && column0 == 0 && item % per == 0 && (MANY ? lane == 0 : threadIdx.x == 0) && (length < 0 || length > p.capacity))
        atomicOr(p.status, DA_STATUS_BAD_POSITION);
    size_t index = 0;
    T *out = out_row<T>(p, there ? item : 0, there ? row : 0, D, index) + column0 * 4;
    if (there && length <= 0 && (MANY || warp == 0)) {   // nothing to attend to
        for (int c = lane; c < COLS * 4; c += 32) out[c] = from_float<T>(0.f);
        if (lane == 0 && writes_lse) p.lse[index] = -INFINITY;
    }
    int n = there && length > 0 ? span.y - span.x + 1 : 1;
    if (n < 1 || span.x < 0 || span.y >= kPagedCtas * MAIN_WARPS) n = 1;   // (a launch that gave up)
    RowSum<NV> sum;

    if constexpr (MANY) {
        if (n > 1 && n <= FEW) {
            sum.template gather<PW>(p.partials + (size_t)row * PW, slot, D, span.x, n, group, GROUPS, col, COLS - 1);
        }
        sh_span[warp] = make_int2(span.x, n);
        if (n > 1 && n <= FEW) {
#pragma unroll
            for (int off = COLS; off < GROUPS * COLS; off <<= 1) sum.x[0].add_lane(off);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (lane + 32 * i < COLS) store_divided(out + 4 * (lane + 32 * i), sum.x[i].o, sum.x[i].m, sum.x[i].l);
            if (lane == 0 && writes_lse) p.lse[index] = natural_lse(sum.x[0].m, sum.x[0].l);
        }
        if (!__syncthreads_or(n > FEW)) return;
    } else {
        if (n == 1) return;                        // one warp had all of it, and wrote it
    }
    for (int w = 0; w < (MANY ? WARPS : 1); ++w) {
        int r = row, i0 = item;
        if constexpr (MANY) {
            span.x = sh_span[w].x, n = sh_span[w].y;
            if (n <= FEW) continue;
            const long long t = (long long)blockIdx.x * WARPS + w;
            i0 = (int)(t / p.group_rows), r = (int)(t - (long long)i0 * p.group_rows);
            out = out_row<T>(p, i0, r, D, index);
        }
        sum.template gather<PW>(p.partials + (size_t)r * PW + column0 * 4, slot, D - column0 * 4, span.x, n, warp * GROUPS + group, WARPS * GROUPS, col, COLS - 1);
#pragma unroll
        for (int off = COLS; off < GROUPS * COLS; off <<= 1) sum.x[0].add_lane(off);
        if (MANY) __syncthreads();                 // the row before has been read
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < COLS) reinterpret_cast<float4 *>(sh_o[warp])[lane + 32 * i] = sum.x[i].o;
        if (lane == 0) sh_ml[warp] = make_float2(sum.x[0].m, sum.x[0].l);
        __syncthreads();
        // a lane of each warp has the weight of one warp's sum, a thread adds up one channel of all
        const float2 ml = lane < WARPS ? sh_ml[lane] : make_float2(-INFINITY, 0.f);
        float m = ml.x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(DA_FULL_MASK, m, off));
        const float k = fast_exp2(ml.x - (m == -INFINITY ? 0.f : m));
        float l = ml.y * k;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(DA_FULL_MASK, l, off);
        if (warp * 32 < COLS * 4) {                // (whole warps: the weights travel by shuffles)
            const int c = threadIdx.x;
            float o = 0.f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) o = fmaf(sh_o[i][min(c, COLS * 4 - 1)], __shfl_sync(DA_FULL_MASK, k, i), o);
            if (c < COLS * 4) out[c] = from_float<T>(m == -INFINITY ? 0.f : o / l);
            if (c == 0 && writes_lse) p.lse[index] = natural_lse(m, l);
        }
    }
}

template <typename T, int D> static cudaError_t launch_join(const PagedParams &p, cudaStream_t stream) {
    constexpr int ALL = D / 4, NARROW = D % 32 == 0 ? 8 : 4, BLOCKS = ALL / NARROW;
    const long long items = (long long)p.n_sequences * p.n_kv_heads * p.groups, rows = items * p.group_rows;
    const unsigned x = (unsigned)items;
    // CTAs of 1024 threads, narrow columns, while no SM gets two of them: few rows are of many parts (100 000 tokens of one head,
    // sixteen rows: 19.5 us, with 256 threads 24.8).  Up to a row for every SM CTAs of 256 with narrow columns (two of 2000 with 8
    // heads, 64 rows: 10.5, with 1024 threads 14.9), then with all columns while four lie on an SM (6 of 2000, 192 rows: 15.2,
    // narrow 18.4), then a warp per row (32 of 1000 with 8 heads, 768 to 1024 rows: 2 to 3 us less than a CTA per row; 512 rows 1 to 2 more).
    if (rows * BLOCKS <= kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 32, NARROW, false>, dim3(x, p.group_rows, BLOCKS), dim3(1024), (size_t)0, stream, p);
    if (rows <= kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 8, NARROW, false>, dim3(x, p.group_rows, BLOCKS), dim3(256), (size_t)0, stream, p);
    if (rows <= 4 * kPagedCtas)
        return launch_dependent(paged_join_kernel<T, D, 8, ALL, false>, dim3(x, p.group_rows), dim3(256), (size_t)0, stream, p);
    return launch_dependent(paged_join_kernel<T, D, 8, ALL, true>, dim3((unsigned)((rows + 7) / 8)), dim3(256), (size_t)0, stream, p);
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

extern "C" size_t da_paged_attention_workspace_bytes(int n_sequences, int n_kv_heads, int rep, int head_dim, int dtype) {
    using namespace da;
    if (n_sequences < 1 || n_kv_heads < 1 || !paged_shape(rep, head_dim, dtype)) return 0;
    const int warps = dtype == DA_F32 ? paged_f32_warps(head_dim) : paged_mma_warps(head_dim);
    const int rows = group_rows(rep, head_dim, dtype);
    return (size_t)kPagedCtas * warps * 2 * rows * (head_dim + 4) * sizeof(float) +
           (size_t)n_sequences * n_kv_heads * ((rep + rows - 1) / rows) * sizeof(int2);
}

extern "C" int da_paged_attention(const da_paged_attention_args *args) {
    using namespace da;
    if (!args) return DA_ERR_NULL;
    const da_paged_attention_args &a = *args;
    if (!a.q || !a.pages || !a.page_table || !a.lengths || !a.out || !a.workspace || !a.status) return DA_ERR_NULL;
    if (a.dtype < DA_F32 || a.dtype > DA_BF16) return DA_ERR_DTYPE;
    if (a.n_sequences < 1 || a.n_kv_heads < 1 || a.rep < 1 || a.page_size < 1 || a.n_pages < 1 || a.table_columns < 1 ||
        a.window < 0 || a.n_sequences > 0x7fffffff || a.n_kv_heads > 1 << 16 || a.page_size > 1 << 30 || a.n_pages > 0x7fffffff ||
        a.table_columns > 0x7fffffff || a.table_columns * a.page_size > 0x7fffff00 || a.window > 0x7fffffff)
        return DA_ERR_SHAPE;
    if (!paged_shape(a.rep, a.head_dim, a.dtype)) return DA_ERR_UNSUPPORTED;
    if (a.n_sequences * a.n_kv_heads * a.rep > 0x7fffffff) return DA_ERR_SHAPE;
    const int esize = a.dtype == DA_F32 ? 4 : 2;
    const uintptr_t rows = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.pages) | reinterpret_cast<uintptr_t>(a.out) |
                           reinterpret_cast<uintptr_t>(a.workspace);
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.page_table) | reinterpret_cast<uintptr_t>(a.lengths) |
                            reinterpret_cast<uintptr_t>(a.lse) | reinterpret_cast<uintptr_t>(a.status);
    if ((rows & 15) || (words & 3) ||
        (a.q_strides[0] | a.q_strides[1] | a.page_stride | a.page_head_stride) % (16 / esize))
        return DA_ERR_ALIGN;
    if (a.workspace_bytes < (int64_t)da_paged_attention_workspace_bytes((int)a.n_sequences, (int)a.n_kv_heads, (int)a.rep, (int)a.head_dim, (int)a.dtype))
        return DA_ERR_WORKSPACE;

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
    const int warps = a.dtype == DA_F32 ? paged_f32_warps((int)a.head_dim) : paged_mma_warps((int)a.head_dim);
    p.partials = static_cast<float *>(a.workspace);
    p.spans = reinterpret_cast<int2 *>(p.partials + (size_t)kPagedCtas * warps * 2 * p.group_rows * (a.head_dim + 4));
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
