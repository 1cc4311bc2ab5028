// Rotary positions of queries and keys, and the append of new tokens to a paged cache with that rotation on the way.
//
//   y = factor * R(p * w_i) x   on the channel pairs i < rot / 2 of a head (adjacent channels, or channel i of either half
//   of the rotated part); the channels behind the rotated part are copied.  The gradient of x is the rotation back,
//   factor * R(-p * w_i) dy: the same kernel with the sign of the angle turned.
//
// The angle p * w_i is taken in turns and in 64 bits, reduced there to an eighth of a turn either way, and only then
// rounded: at position 1 000 000 a 32-bit product is off by up to 0.03 rad, this one by 3e-8 at any position.  Products and
// sums are 32-bit, the result is rounded once to the element type.
//
// Bound by memory: a token of 32 + 8 heads of 128 bf16 channels is 10 KB in and 10 KB out against 64 angles.  One CTA per
// token (few tokens: several, each with some of the heads): the angles are made once per CTA and kept in shared memory, while
// the rows, already requested, are on their way; a thread keeps its place in the head and goes from row to row.

#include "da_common.cuh"

namespace da {

constexpr int kRotateThreads = 256;   // about; the block is a whole number of rows
constexpr int kRotateUnroll = 2;      // rows a thread has under way

struct RotateParams {
    // sources: queries, keys and (append) values; strides in elements
    const void *src[3];
    long long src_batch[3], src_token[3], src_head[3];
    int heads[3];
    void *dst[2];                     // rotated queries and keys, contiguous (append: queries only)
    int n_tokens;                     // per batch entry (append: rows of the ragged batch)
    int head_dim, rot_half;
    const float *inv_freq;
    float factor, sign;
    const void *positions;
    int positions_64;
    long long position_batch, position_token;
    int rows_per_cta;
    // append
    void *pages;
    long long page_stride, page_head_stride;
    int page_size, n_pages;
    const int32_t *table;
    long long table_stride;
    int table_cols;
    const int32_t *lengths, *starts;
    int n_sequences;
    int32_t *status;
};

// cos and sin of a fraction of `turns` full turns
__device__ __forceinline__ float2 cos_sin_turns(double turns) {
    const double quarters = 4.0 * turns;
    const double k = rint(quarters);
    float s, c;
    sincospif(0.5f * (float)(quarters - k), &s, &c);      // |argument| <= 1/4: nothing is lost in the conversion
    const int quadrant = (int)((long long)k & 3);
    const float a = (quadrant & 1) ? s : c, b = (quadrant & 1) ? c : s;
    return make_float2((quadrant == 1 || quadrant == 2) ? -a : a, quadrant >= 2 ? -b : b);
}

template <typename T, int V> struct Chunk {
    static_assert(V * sizeof(T) == 16, "vectors are 16 bytes");
    uint4 raw;
    __device__ __forceinline__ void load(const T *p) { raw = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = raw; }
    __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void unpack(float (&x)[V]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        Unpack<T, V>::run(w, x);
    }
    __device__ __forceinline__ void pack(const float (&x)[V]) {
        union { T t[V]; uint4 v; } u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.t[i] = from_float<T>(x[i]);
        raw = u.v;
    }
};
template <typename T> struct Chunk<T, 1> {
    T raw;
    __device__ __forceinline__ void load(const T *p) { raw = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = raw; }
    __device__ __forceinline__ void zero() { raw = from_float<T>(0.f); }
    __device__ __forceinline__ void unpack(float (&x)[1]) const { x[0] = to_float(raw); }
    __device__ __forceinline__ void pack(const float (&x)[1]) { raw = from_float<T>(x[0]); }
};

// (a, b) turned by (cos, sin)
__device__ __forceinline__ void turn(float &a, float &b, float2 cs) {
    const float x = a * cs.x - b * cs.y, y = b * cs.x + a * cs.y;
    a = x;
    b = y;
}

// Where a row of the ragged batch belongs.
struct Place {
    long long position;
    int page;                 // -1: nowhere
    int slot;
    bool used;                // the row belongs to a sequence and its position exists
    int status;
};
__device__ __forceinline__ Place find_place(const RotateParams &p, int row) {
    Place at = {0, -1, 0, false, 0};
    int b = row, first = row, n_new = 1;
    if (p.starts) {
        int lo = 0, hi = p.n_sequences + 1;     // how many starts are <= row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(p.starts + mid) <= row) lo = mid + 1;
            else hi = mid;
        }
        b = lo - 1;
        if (b < 0 || b >= p.n_sequences) return at;          // a row in front of or behind the sequences
        first = __ldg(p.starts + b);
        n_new = __ldg(p.starts + b + 1) - first;
    }
    const int length = __ldg(p.lengths + b);
    if (length == 0) return at;                              // an entry of the batch that is not in use
    at.position = (long long)length - n_new + (row - first);
    if (length < 0 || at.position < 0 || at.position >= (long long)p.table_cols * p.page_size) {
        at.status = DA_STATUS_BAD_POSITION;
        return at;
    }
    at.used = true;
    const int column = (int)at.position / p.page_size;
    at.slot = (int)at.position - column * p.page_size;
    at.page = __ldg(p.table + (long long)b * p.table_stride + column);
    if (at.page < 0 || at.page >= p.n_pages) {
        at.page = -1;
        at.status = DA_STATUS_BAD_PAGE_ID;
    }
    return at;
}

// HALF: channel i is paired with channel i + rot / 2; otherwise with its neighbour.  A thread's task is its column of the
// block: in front the tasks that rotate (both members' chunks of V channels; neighbours: one chunk that holds whole pairs, or
// the two channels of a pair when V is 1), then those that copy a chunk behind the rotated part.
template <typename T, int V, bool HALF, bool PAGED>
__global__ void __launch_bounds__(kRotateThreads * 2)
rotate_kernel(const RotateParams p) {
    constexpr bool kTwo = HALF || V == 1;         // a rotating task has two chunks
    extern __shared__ float2 cos_sin[];           // [rot_half]
    griddep_wait();
    griddep_launch_dependents();
    const int task = threadIdx.x, y = threadIdx.y;
    const int n_turn = kTwo ? p.rot_half / V : (2 * p.rot_half + V - 1) / V;
    const bool turns = task < n_turn;
    const int at0 = turns ? (V == 1 && !HALF ? 2 * task : task * V)
                          : (kTwo ? 2 * p.rot_half + (task - n_turn) * V : task * V);
    const int at1 = HALF ? p.rot_half + task * V : at0 + 1;
    const bool two = kTwo && turns;

    const int row0 = blockIdx.y * p.rows_per_cta;
    const int row_end = min(row0 + p.rows_per_cta, p.heads[0] + p.heads[1] + p.heads[2]);
    const int token = blockIdx.x % p.n_tokens, batch = blockIdx.x / p.n_tokens;

    Chunk<T, V> a[kRotateUnroll], b[kRotateUnroll];
    auto request = [&](int base) {
#pragma unroll
        for (int i = 0; i < kRotateUnroll; ++i) {
            const int r = base + i * blockDim.y;
            if (r >= row_end) continue;
            const int which = r < p.heads[0] ? 0 : (r < p.heads[0] + p.heads[1] ? 1 : 2);
            const int head = which == 0 ? r : (which == 1 ? r - p.heads[0] : r - p.heads[0] - p.heads[1]);
            const T *s = static_cast<const T *>(p.src[which]) + batch * p.src_batch[which] + token * p.src_token[which] +
                         head * p.src_head[which];
            a[i].load(s + at0);
            if (two) b[i].load(s + at1);
        }
    };
    request(row0 + y);

    // the token's position and its angles, while the rows are on their way
    Place at = {0, -1, 0, true, 0};
    if constexpr (PAGED) {
        at = find_place(p, token);
        if (at.status && blockIdx.y == 0 && task == 0 && y == 0) atomicOr(p.status, at.status);
    } else {
        const long long i = batch * p.position_batch + token * p.position_token;
        at.position = p.positions_64 ? __ldg(static_cast<const long long *>(p.positions) + i)
                                     : (long long)__ldg(static_cast<const int32_t *>(p.positions) + i);
    }
    for (int i = y * blockDim.x + task; i < p.rot_half; i += blockDim.x * blockDim.y) {
        const double per_turn = (double)__ldg(p.inv_freq + i) * 0.15915494309189535;   // 1 / 2 pi
        float2 cs = cos_sin_turns((double)at.position * per_turn);
        cos_sin[i] = make_float2(cs.x * p.factor, cs.y * p.factor * p.sign);
    }
    __syncthreads();

    for (int base = row0 + y; base < row_end; base += kRotateUnroll * blockDim.y) {
        if (base != row0 + y) request(base);
#pragma unroll
        for (int i = 0; i < kRotateUnroll; ++i) {
            const int r = base + i * blockDim.y;
            if (r >= row_end) continue;
            const int which = r < p.heads[0] ? 0 : (r < p.heads[0] + p.heads[1] ? 1 : 2);
            const int head = which == 0 ? r : (which == 1 ? r - p.heads[0] : r - p.heads[0] - p.heads[1]);
            if (turns && which != 2) {
                float x[V];
                a[i].unpack(x);
                if constexpr (kTwo) {
                    float z[V];
                    b[i].unpack(z);
#pragma unroll
                    for (int j = 0; j < V; ++j) turn(x[j], z[j], cos_sin[task * V + j]);
                    b[i].pack(z);
                } else {
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {
                        const int pair = task * (V / 2) + j;
                        if (pair < p.rot_half) turn(x[2 * j], x[2 * j + 1], cos_sin[pair]);
                    }
                }
                a[i].pack(x);
            }
            T *d;
            if (PAGED && which != 0) {
                if (at.page < 0) continue;
                d = static_cast<T *>(p.pages) + head * p.page_head_stride + at.page * p.page_stride +
                    (long long)at.slot * 2 * p.head_dim + (which == 2 ? p.head_dim : 0);
            } else {
                d = static_cast<T *>(p.dst[which]) + ((long long)blockIdx.x * p.heads[which] + head) * p.head_dim;
                if (PAGED && !at.used) {   // a row of no sequence
                    a[i].zero();
                    b[i].zero();
                }
            }
            a[i].store(d + at0);
            if (two) b[i].store(d + at1);
        }
    }
}

template <typename T, int V, bool HALF, bool PAGED>
static int launch_rotate(RotateParams p, int n_batch, cudaStream_t stream) {
    const int rot = 2 * p.rot_half, d = p.head_dim;
    const int tasks = (HALF || V == 1) ? p.rot_half / V + (d - rot) / V : d / V;
    const int rows = p.heads[0] + p.heads[1] + p.heads[2];
    const long long tokens = (long long)n_batch * p.n_tokens;
    // Few tokens: their rows are spread over as many CTAs as leave each at least two warps.
    int per_cta = rows;
    if (tokens < 148) {
        const int least = (64 + tasks - 1) / tasks;
        const int splits = (int)(148 / tokens);
        per_cta = (rows + splits - 1) / splits;
        if (per_cta < least) per_cta = least;
        if (per_cta > rows) per_cta = rows;
    }
    p.rows_per_cta = per_cta;
    const int splits = (rows + per_cta - 1) / per_cta;
    // as many rows at a time as fill the block, evenly over the passes
    int y = kRotateThreads / tasks;
    if (y < 1) y = 1;
    const int passes = (per_cta + y - 1) / y;
    y = (per_cta + passes - 1) / passes;
    const cudaError_t e = launch_dependent(rotate_kernel<T, V, HALF, PAGED>, dim3((unsigned)tokens, splits), dim3(tasks, y),
                                           p.rot_half * sizeof(float2), stream, p);
    return (int)e;
}

template <bool PAGED>
static int rotate(const RotateParams &p, int n_batch, int dtype, bool half, bool vectors, cudaStream_t stream) {
    switch (dtype) {
    case DA_F32:
        if (vectors) return half ? launch_rotate<float, 4, true, PAGED>(p, n_batch, stream) : launch_rotate<float, 4, false, PAGED>(p, n_batch, stream);
        return half ? launch_rotate<float, 1, true, PAGED>(p, n_batch, stream) : launch_rotate<float, 1, false, PAGED>(p, n_batch, stream);
    case DA_F16:
        if (vectors) return half ? launch_rotate<__half, 8, true, PAGED>(p, n_batch, stream) : launch_rotate<__half, 8, false, PAGED>(p, n_batch, stream);
        return half ? launch_rotate<__half, 1, true, PAGED>(p, n_batch, stream) : launch_rotate<__half, 1, false, PAGED>(p, n_batch, stream);
    default:
        if (vectors) return half ? launch_rotate<__nv_bfloat16, 8, true, PAGED>(p, n_batch, stream) : launch_rotate<__nv_bfloat16, 8, false, PAGED>(p, n_batch, stream);
        return half ? launch_rotate<__nv_bfloat16, 1, true, PAGED>(p, n_batch, stream) : launch_rotate<__nv_bfloat16, 1, false, PAGED>(p, n_batch, stream);
    }
}

static bool small(int64_t v, int64_t lo, int64_t hi) { return v >= lo && v <= hi; }

}  // namespace da

extern "C" int da_rotate(const da_rotate_args *args) {
    using namespace da;
    if (!args) return DA_ERR_NULL;
    const da_rotate_args &a = *args;
    if (!a.positions || !a.inv_freq || (!a.q && !a.k) || (a.q && !a.q_out) || (a.k && !a.k_out)) return DA_ERR_NULL;
    if (!small(a.dtype, DA_F32, DA_BF16)) return DA_ERR_DTYPE;
    if (!small(a.n_batch, 1, 1 << 24) || !small(a.n_tokens, 1, 1 << 30) || a.n_batch * a.n_tokens > 0x7fffffff ||
        !small(a.head_dim, 2, 512) || !small(a.rotary_dim, 2, a.head_dim) || (a.rotary_dim & 1) ||
        (a.q && !small(a.n_q_heads, 1, 1 << 16)) || (a.k && !small(a.n_kv_heads, 1, 1 << 16)))
        return DA_ERR_SHAPE;
    const int esize = a.dtype == DA_F32 ? 4 : 2;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                            reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k_out);
    if (bases & (esize - 1) || (reinterpret_cast<uintptr_t>(a.positions) & (a.positions_64 ? 7 : 3)) ||
        (reinterpret_cast<uintptr_t>(a.inv_freq) & 3))
        return DA_ERR_ALIGN;
    RotateParams p = {};
    int64_t strides = 0;
    const void *src[2] = {a.q, a.k};
    const int64_t heads[2] = {a.n_q_heads, a.n_kv_heads};
    for (int i = 0; i < 2; ++i) {
        if (!src[i]) continue;
        const int64_t *s = i == 0 ? a.q_strides : a.k_strides;
        p.src[i] = src[i];
        p.src_batch[i] = s[0], p.src_token[i] = s[1], p.src_head[i] = s[2];
        strides |= s[0] | s[1] | s[2];
        p.heads[i] = (int)heads[i];
    }
    p.dst[0] = a.q_out, p.dst[1] = a.k_out;
    p.n_tokens = (int)a.n_tokens;
    p.head_dim = (int)a.head_dim, p.rot_half = (int)a.rotary_dim / 2;
    p.inv_freq = a.inv_freq, p.factor = (float)a.factor, p.sign = a.transposed ? -1.f : 1.f;
    p.positions = a.positions, p.positions_64 = a.positions_64 != 0;
    p.position_batch = a.position_strides[0], p.position_token = a.position_strides[1];
    // 16-byte pieces, when every row and (halves) the second half start on such a boundary; otherwise channel by channel
    const int v = 16 / esize;
    const bool half = a.interleaved == 0;
    const bool vectors = !(bases & 15) && strides % v == 0 && a.head_dim % v == 0 && (!half || (a.rotary_dim / 2) % v == 0);
    return rotate<false>(p, (int)a.n_batch, (int)a.dtype, half, vectors, static_cast<cudaStream_t>(a.stream));
}

extern "C" int da_append_pages(const da_append_pages_args *args) {
    using namespace da;
    if (!args) return DA_ERR_NULL;
    const da_append_pages_args &a = *args;
    if (!a.k || !a.v || !a.pages || !a.page_table || !a.lengths || !a.status || (a.q && (!a.q_out || !a.inv_freq)))
        return DA_ERR_NULL;
    if (!small(a.dtype, DA_F32, DA_BF16)) return DA_ERR_DTYPE;
    if (!small(a.n_rows, 1, 1 << 30) || !small(a.n_sequences, 1, 1 << 30) || (!a.starts && a.n_rows != a.n_sequences) ||
        !small(a.head_dim, 2, 512) || (a.q && !small(a.n_q_heads, 1, 1 << 16)) || !small(a.n_kv_heads, 1, 1 << 16) ||
        !small(a.page_size, 1, 1 << 20) || !small(a.n_pages, 1, 0x7fffffff) || !small(a.table_columns, 1, 0x7fffffff) ||
        a.table_columns * a.page_size > 0x7fffff00 ||
        (a.inv_freq && (!small(a.rotary_dim, 2, a.head_dim) || (a.rotary_dim & 1))))
        return DA_ERR_SHAPE;
    const int esize = a.dtype == DA_F32 ? 4 : 2;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                            reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.q_out) |
                            reinterpret_cast<uintptr_t>(a.pages);
    if (bases & (esize - 1) || ((reinterpret_cast<uintptr_t>(a.page_table) | reinterpret_cast<uintptr_t>(a.lengths) |
                                 reinterpret_cast<uintptr_t>(a.starts) | reinterpret_cast<uintptr_t>(a.inv_freq) |
                                 reinterpret_cast<uintptr_t>(a.status)) & 3))
        return DA_ERR_ALIGN;
    RotateParams p = {};
    int64_t strides = a.page_stride | a.page_head_stride;
    const void *src[3] = {a.q, a.k, a.v};
    const int64_t *s[3] = {a.q_strides, a.k_strides, a.v_strides};
    for (int i = 0; i < 3; ++i) {
        if (!src[i]) continue;
        p.src[i] = src[i];
        p.src_token[i] = s[i][0], p.src_head[i] = s[i][1];
        strides |= s[i][0] | s[i][1];
        p.heads[i] = (int)(i == 0 ? a.n_q_heads : a.n_kv_heads);
    }
    p.dst[0] = a.q_out;
    p.n_tokens = (int)a.n_rows;
    p.head_dim = (int)a.head_dim, p.rot_half = a.inv_freq ? (int)a.rotary_dim / 2 : 0;
    p.inv_freq = a.inv_freq, p.factor = (float)a.factor, p.sign = 1.f;
    p.pages = a.pages, p.page_stride = a.page_stride, p.page_head_stride = a.page_head_stride;
    p.page_size = (int)a.page_size, p.n_pages = (int)a.n_pages;
    p.table = a.page_table, p.table_stride = a.table_stride, p.table_cols = (int)a.table_columns;
    p.lengths = a.lengths, p.starts = a.starts, p.n_sequences = (int)a.n_sequences;
    p.status = a.status;
    const int v = 16 / esize;
    const bool half = a.interleaved == 0;
    const bool vectors = !(bases & 15) && strides % v == 0 && a.head_dim % v == 0 && (!half || p.rot_half % v == 0);
    return rotate<true>(p, 1, (int)a.dtype, half, vectors, static_cast<cudaStream_t>(a.stream));
}
