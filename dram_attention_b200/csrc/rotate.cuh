// Rotary positions of queries and keys, and the append of new tokens to a paged cache with that rotation on the way.
//
//   y = factor * R(p * w_i) x   on the channel pairs i < rot / 2 of a head (adjacent channels, or channel i of either half
//   of the rotated part); the channels behind the rotated part are copied.  The gradient of x is the rotation back,
//   factor * R(-p * w_i) dy: the same kernel with the sign of the angle turned.
//
// The angle p * w_i is taken in quarter turns and in 64 bits, reduced there to an eighth of a turn either way, and only then
// rounded: at position 1 000 000 a 32-bit product is off by up to 0.03 rad, this one by 3e-8 up to position 10^8 (and by 5e-7 at
// 2^31, where 64 bits end).  Products and sums are 32-bit, the result is rounded once to the element type.
//
// Bound by memory: a token of 32 + 8 heads of 128 bf16 channels is 10 KB in and 10 KB out against 64 angles.  What stands in the
// way is the number of instructions, so a thread keeps its place: one column of up to four neighbouring heads, for several
// tokens in turn.  Addresses are then sums, the sines and cosines of a token are read once for four rows, and the
// angles, positions and (append) places in the pool are made once per token of the block, while the first rows are on their way.

#pragma once

#include "da_common.cuh"

namespace da {

constexpr int kRotateRows = 4;        // rows a thread has under way: heads of a token, or of several tokens
constexpr int kRotateTokens = 64;     // most tokens of a block

struct RotateParams {
    // sources: queries, keys and (append) values; strides in elements
    const void *src[3];
    long long src_batch[3], src_token[3], src_head[3];
    int heads[3];
    void *dst[2];                     // rotated queries and keys, contiguous (append: queries only)
    int n_tokens;                     // per batch entry, as the sources see it (append: rows of the ragged batch)
    int all_tokens;                   // of all batch entries
    int together;                     // tokens of a thread whose rows are under way at the same time (at most 4 / ROWS)
    int rounds;                       // ... and how often in turn
    int head_dim, rot_half;
    const float *inv_freq;
    float factor, sign;
    const void *positions;
    int positions_64;
    int position_tokens;              // per batch entry, as the positions see it
    long long position_batch, position_token;
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

// cos and sin of x quarter turns, |x| < 2^51.  x is split in 64 bits into its nearest whole number, whose low bits fall out of the
// sum with 1.5 * 2^52, and a rest of at most 1/2, which loses nothing when it is rounded to 32 bits; the rest goes through
// the Taylor series of sin and cos at (pi / 2) x, whose first left-out terms are below 2e-9 and 2e-10 there.
__device__ __forceinline__ float2 cos_sin_quarters(double x) {
    constexpr double kWhole = 6755399441055744.0, H = 1.5707963267948966;   // 1.5 * 2^52, pi / 2
    constexpr double H2 = H * H, H3 = H2 * H, H4 = H2 * H2, H5 = H4 * H, H6 = H4 * H2, H7 = H6 * H, H8 = H4 * H4, H9 = H8 * H, H10 = H8 * H2;
    const double shifted = x + kWhole;
    const int quadrant = __double2loint(shifted) & 3;
    const float f = (float)(x - (shifted - kWhole)), z = f * f;
    float s = fmaf(z, (float)(H9 / 362880), -(float)(H7 / 5040));
    s = fmaf(z, s, (float)(H5 / 120));
    s = fmaf(z, s, -(float)(H3 / 6));
    s = fmaf(z, s, (float)(H - (double)(float)H));          // (what pi / 2 loses in 32 bits)
    s = fmaf(f, (float)H, f * s);
    float c = fmaf(z, -(float)(H10 / 3628800), (float)(H8 / 40320));
    c = fmaf(z, c, -(float)(H6 / 720));
    c = fmaf(z, c, (float)(H4 / 24));
    c = fmaf(z, c, -(float)(H2 / 2));
    c = fmaf(z, c, 1.f);
    const float a = (quadrant & 1) ? s : c, b = (quadrant & 1) ? c : s;
    return make_float2((quadrant == 1 || quadrant == 2) ? -a : a, quadrant >= 2 ? -b : b);
}

template <int BYTES> struct Words;
template <> struct Words<16> { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = unsigned short; };

// V consecutive elements in one access.
template <typename T, int V> struct Chunk {
    using Raw = typename Words<V * (int)sizeof(T)>::type;
    Raw raw;
    __device__ __forceinline__ void load(const T *p) { raw = __ldcs(reinterpret_cast<const Raw *>(p)); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<Raw *>(p) = raw; }
    __device__ __forceinline__ void zero() { raw = Raw{}; }
    template <class At> __device__ __forceinline__ void gather(const T *p, At at) {
        union { Raw r; T t[V]; } u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.t[i] = p[at(i)];
        raw = u.r;
    }
    __device__ __forceinline__ void unpack(float (&x)[V]) const {
        union { Raw r; T t[V]; uint32_t w[V > 1 ? V * sizeof(T) / 4 : 1]; } u;
        u.r = raw;
        if constexpr (V == 1) {
            x[0] = to_float(u.t[0]);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = u.t[i];
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) unpack2<T>(u.w[i], x[2 * i], x[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void pack(const float (&x)[V]) {
        union { Raw r; T t[V]; uint32_t w[V > 1 ? V * sizeof(T) / 4 : 1]; } u;
        if constexpr (V == 1 || sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) u.t[i] = from_float<T>(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) u.w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
        }
        raw = u.r;
    }
};

// (a, b) turned by (cos, sin)
__device__ __forceinline__ void turn(float &a, float &b, float2 cs) {
    const float x = a * cs.x - b * cs.y, y = b * cs.x + a * cs.y;
    a = x;
    b = y;
}

// The last sequence that does not begin behind a row, or -1; by a warp, all starts at once.
__device__ __forceinline__ int find_near(const RotateParams &p, int row, int lane) {
    int count = 0;
    for (int i = lane; i <= p.n_sequences; i += 32) count += __ldg(p.starts + i) <= row;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) count += __shfl_xor_sync(DA_FULL_MASK, count, off);
    return count - 1;
}

// Where a row of the ragged batch belongs.
struct Place {
    long long position;
    int page;                 // -1: nowhere
    int slot;
    bool used;                // the row belongs to a sequence and its position exists
    int status;
};
// `near`: a sequence that does not begin behind the row (the one of the block's first row, or -1).
__device__ __forceinline__ Place find_place(const RotateParams &p, int row, int near) {
    Place at = {0, -1, 0, false, 0};
    int b = row, first = row, n_new = 1;
    if (p.starts) {
        b = near;
        int next = b < p.n_sequences ? __ldg(p.starts + b + 1) : 0;
        first = b >= 0 ? __ldg(p.starts + b) : 0;
        while (b < p.n_sequences && next <= row) {           // the row belongs to a sequence further on
            first = next;
            ++b;
            next = b < p.n_sequences ? __ldg(p.starts + b + 1) : 0;
        }
        if (b < 0 || b >= p.n_sequences) return at;          // a row in front of or behind the sequences
        n_new = next - first;
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

// Which channels a thread has: in front the columns that rotate, then those that copy a chunk behind the rotated part.
//   kNeighbours   channel 2 i is paired with 2 i + 1: one chunk of V channels, whole pairs (V 1: the two channels of a pair)
//   kHalves       channel i is paired with i + rot / 2, a multiple of V: the chunks of both members
//   kCrossed      the same where rot / 2 is no multiple of V: one chunk, the other members of its pairs read one by one
//                 (8000 tokens of 16 + 4 heads of 80, 17 pairs: channel by channel 44 us, so 28)
enum Pairing { kNeighbours, kHalves, kCrossed };

// ROWS: heads of a thread.
template <typename T, int V, Pairing PAIRING, bool PAGED, int ROWS>
__global__ void __launch_bounds__(V > 1 ? 256 : 512, V > 1 ? (PAIRING == kNeighbours ? 4 : 3) : 1)
rotate_kernel(const RotateParams p) {
    constexpr bool HALF = PAIRING == kHalves, CROSSED = PAIRING == kCrossed;
    constexpr bool kTwo = HALF || (V == 1 && !CROSSED);          // a rotating column has two chunks
    constexpr int kPairs = kTwo || CROSSED ? V : V / 2;          // pairs it takes part in
    extern __shared__ float2 cos_sin[];           // [tokens of the block][rot_half]
    __shared__ double sh_position[kRotateTokens];
    __shared__ int sh_near;
    __shared__ long long sh_place[PAGED ? kRotateTokens : 1];   // offset in the pool, -1: no page, -2: a row of no sequence
    griddep_wait();
    griddep_launch_dependents();
    const int column = threadIdx.x, z = threadIdx.z;
    const int linear = (z * blockDim.y + threadIdx.y) * blockDim.x + column, threads = blockDim.x * blockDim.y * blockDim.z;
    const int n_turn = kTwo ? p.rot_half / V : (2 * p.rot_half + V - 1) / V;
    const bool turns = column < n_turn, two = kTwo && turns;
    const int at0 = turns ? (V == 1 && !HALF ? 2 * column : column * V)
                          : (kTwo ? 2 * p.rot_half + (column - n_turn) * V : column * V);
    const int at1 = HALF ? p.rot_half + column * V : at0 + 1;

    // this thread's heads: `mine` of one kind from head0 on
    int kind = 0, head0 = (blockIdx.y * blockDim.y + threadIdx.y) * ROWS;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int all = (p.heads[i] + ROWS - 1) / ROWS * ROWS;
        if (kind == i && head0 >= all) head0 -= all, ++kind;
    }
    const int mine = min(ROWS, p.heads[kind] - head0);

    const int per_block = blockDim.z * p.together * p.rounds;
    const int first = blockIdx.x * per_block;
    const int here = min(per_block, p.all_tokens - first);      // tokens of this block

    const T *base = static_cast<const T *>(p.src[kind]) + head0 * p.src_head[kind];
    const long long src_head = p.src_head[kind];
    // crossed columns: where the partner of channel j stands, and which pair they are
    auto partner = [&](int j) { const int c = at0 + j; return c < p.rot_half ? c + p.rot_half : (c < 2 * p.rot_half ? c - p.rot_half : c); };
    auto pair_of = [&](int j) { const int c = at0 + j; return c < p.rot_half ? c : c - p.rot_half; };
    Chunk<T, V> a[kRotateRows], b[kRotateRows];
    // token t, and the thread's next ones: their rows of its heads
    auto request = [&](int t) {
#pragma unroll
        for (int g = 0; g < kRotateRows / ROWS; ++g) {
            if (g < p.together && t < here) {
                int batch = 0, token = first + t;
                if (!PAGED && p.n_tokens != p.all_tokens) batch = token / p.n_tokens, token -= batch * p.n_tokens;
                const T *s = base + (batch * p.src_batch[kind] + token * p.src_token[kind]);
#pragma unroll
                for (int i = g * ROWS; i < (g + 1) * ROWS; ++i) {
                    if (i - g * ROWS < mine) {
                        a[i].load(s + at0);
                        if (two) b[i].load(s + at1);
                        if constexpr (CROSSED) {
                            if (turns) b[i].gather(s, partner);
                        }
                    }
                    s += src_head;
                }
            }
            t += blockDim.z;
        }
    };
    request(z);

    // the tokens' positions and places, while the first rows are on their way
    if constexpr (PAGED) {
        if (p.starts) {
            if (linear < 32 && threads >= 32) {
                const int near = find_near(p, first, linear);
                if (linear == 0) sh_near = near;
            } else if (threads < 32 && linear == 0) {
                sh_near = -1;                      // (a walk from the front)
            }
            __syncthreads();
        }
    }
    for (int j = linear; j < here; j += threads) {
        const int t = first + j;
        if constexpr (PAGED) {
            const Place at = find_place(p, t, p.starts ? sh_near : 0);
            if (at.status && blockIdx.y == 0) atomicOr(p.status, at.status);
            sh_position[j] = (double)at.position;
            sh_place[j] = !at.used ? -2 : (at.page < 0 ? -1 : at.page * p.page_stride + (long long)at.slot * 2 * p.head_dim);
        } else {
            const int n = t / p.position_tokens;
            const long long i = n * p.position_batch + (t - n * p.position_tokens) * p.position_token;
            sh_position[j] = p.positions_64 ? (double)__ldg(static_cast<const long long *>(p.positions) + i)
                                                 : (double)__ldg(static_cast<const int32_t *>(p.positions) + i);
        }
    }
    __syncthreads();
    for (int i = linear; i < here * p.rot_half; i += threads) {
        const int t = i / p.rot_half, pair = i - t * p.rot_half;
        const double quarters = (double)__ldg(p.inv_freq + pair) * 0.6366197723675814;   // 2 / pi
        const float2 cs = cos_sin_quarters(sh_position[t] * quarters);
        cos_sin[i] = make_float2(cs.x * p.factor, cs.y * p.factor * p.sign);
    }
    __syncthreads();

    // a chunk that ends behind the rotated part: its last pairs are copied, not multiplied by 1 and 0
    const int pairs = CROSSED ? 2 * p.rot_half - at0 : (kTwo ? V : min(V / 2, p.rot_half - column * (V / 2)));
    const bool rotates = turns && kind != 2;
    const bool to_pages = PAGED && kind != 0;
    T *const out = to_pages ? static_cast<T *>(p.pages) + head0 * p.page_head_stride + (kind == 2 ? p.head_dim : 0)
                            : static_cast<T *>(p.dst[kind < 2 ? kind : 0]) + ((long long)first * p.heads[kind] + head0) * p.head_dim;
    const long long out_head = to_pages ? p.page_head_stride : p.head_dim;
    const int stride = blockDim.z * p.together;
    for (int start = z; start < here; start += stride) {
#pragma unroll
        for (int g = 0; g < kRotateRows / ROWS; ++g) {
            const int t = start + g * blockDim.z;
            if (g >= p.together || t >= here) continue;
            const float2 *cs = cos_sin + t * p.rot_half + (CROSSED ? 0 : column * kPairs);
            const long long place = PAGED ? sh_place[t] : 0;
            T *d = out + (to_pages ? place : (long long)t * p.heads[kind] * p.head_dim);
            if (rotates) {
                float2 w[kPairs];
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    if constexpr (CROSSED) {
                        w[j] = j < pairs ? cs[pair_of(j)] : make_float2(1.f, 0.f);
                        if (at0 + j < p.rot_half) w[j].y = -w[j].y;      // the first member of its pair
                    } else {
                        w[j] = kTwo || j < pairs ? cs[j] : make_float2(1.f, 0.f);
                    }
                }
#pragma unroll
                for (int i = g * ROWS; i < (g + 1) * ROWS; ++i) {
                    if (i - g * ROWS >= mine) continue;
                    float x[V];
                    a[i].unpack(x);
                    if constexpr (kTwo) {
                        float u[V];
                        b[i].unpack(u);
#pragma unroll
                        for (int j = 0; j < V; ++j) turn(x[j], u[j], w[j]);
                        b[i].pack(u);
                    } else if constexpr (CROSSED) {
                        float u[V];
                        b[i].unpack(u);
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            if (j < pairs) x[j] = x[j] * w[j].x + u[j] * w[j].y;
                    } else {
#pragma unroll
                        for (int j = 0; j < V / 2; ++j)
                            if (j < pairs) turn(x[2 * j], x[2 * j + 1], w[j]);
                    }
                    a[i].pack(x);
                }
            }
            if (PAGED && kind == 0 && place == -2) {
#pragma unroll
                for (int i = g * ROWS; i < (g + 1) * ROWS; ++i) a[i].zero(), b[i].zero();
            }
            if (!to_pages || place >= 0) {
#pragma unroll
                for (int i = g * ROWS; i < (g + 1) * ROWS; ++i) {
                    if (i - g * ROWS < mine) {
                        a[i].store(d + at0);
                        if (two) b[i].store(d + at1);
                    }
                    d += out_head;
                }
            }
        }
        request(start + stride);
    }
}

// Places for heads that threads of `each` heads have.
static int rotate_threads(const RotateParams &p, int each) {
    int y = 0;
    for (int h : p.heads) y += (h + each - 1) / each;
    return y;
}

template <typename T, int V, Pairing PAIRING, bool PAGED, int ROWS>
static int launch_rotate(RotateParams p, int columns, cudaStream_t stream) {
    // Whole tokens up to the size of a block; small blocks are fastest (32 768 tokens of 32 + 8 heads in halves: 105 us with 96 to
    // 192 threads, 115 with 384).  Then a few tokens in turn, which share the look-ups and angles of a block (append of 32 768
    // tokens of 32 + 8 heads in neighbours: 143 us with one, 131 with four), unless a thread has eight chunks under way
    // already (19 000 tokens of 32 + 8 heads in halves: 82 us with one, 95 with four).
    constexpr int THREADS = 128, CHUNKS = PAIRING == kNeighbours && V > 1 ? 1 : 2;
    const int all_y = rotate_threads(p, ROWS);
    int y = columns * all_y <= 192 ? all_y : THREADS / columns;   // (the angles of a token are made once, then)
    if (y < 1) y = 1;
    const int blocks_y = (all_y + y - 1) / y;
    y = (all_y + blocks_y - 1) / blocks_y;
    int z = THREADS / (columns * y);
    if (z > kRotateTokens / 4) z = kRotateTokens / 4;
    while (z > 1 && p.all_tokens / z < 148) z >>= 1;
    if (z < 1) z = 1;
    int tokens = p.all_tokens / (z * 16 * 148);    // of a thread, while sixteen blocks are left for every SM
    if (tokens > 4) tokens = 4;
    if (tokens < 1) tokens = 1;
    p.together = tokens < kRotateRows / ROWS ? tokens : kRotateRows / ROWS;
    p.rounds = ROWS * p.together * CHUNKS <= 4 ? tokens / p.together : 1;
    const int per_block = z * p.together * p.rounds;
    return (int)launch_dependent(rotate_kernel<T, V, PAIRING, PAGED, ROWS>, dim3((unsigned)(((long long)p.all_tokens + per_block - 1) / per_block), blocks_y),
                                 dim3(columns, y, z), (size_t)per_block * p.rot_half * sizeof(float2), stream, p);
}

template <typename T, int V, Pairing PAIRING, bool PAGED>
static int rotate_heads(RotateParams p, int n_batch, cudaStream_t stream) {
    const int rot = 2 * p.rot_half, d = p.head_dim;
    const int columns = PAIRING == kHalves || (V == 1 && PAIRING == kNeighbours) ? p.rot_half / V + (d - rot) / V : d / V;
    p.all_tokens = n_batch * p.n_tokens;
    // Many tokens: as many heads to a thread as leave fewest places empty, the larger number of two that do; few: one, so that
    // every row sets out at once.
    int rows = 1;
    if ((long long)p.all_tokens * rotate_threads(p, 1) * columns > 148 * 1024) {
        long long best = -1;
        for (int each = kRotateRows; each >= 1; --each) {
            if (V * sizeof(T) < 16 && (each == 2 || each == 3)) continue;   // (rare, and the kernel has forms enough)
            const long long places = (long long)rotate_threads(p, each) * each;
            if (best < 0 || places * 8 < best * 7) best = places, rows = each;
        }
    }
    if (rows == 4) return launch_rotate<T, V, PAIRING, PAGED, 4>(p, columns, stream);
    if constexpr (V * sizeof(T) == 16) {
        if (rows == 3) return launch_rotate<T, V, PAIRING, PAGED, 3>(p, columns, stream);
        if (rows == 2) return launch_rotate<T, V, PAIRING, PAGED, 2>(p, columns, stream);
    }
    return launch_rotate<T, V, PAIRING, PAGED, 1>(p, columns, stream);
}

// V: the longest access that every row starts on a multiple of, up to 16 bytes
template <typename T, int V, bool PAGED>
static int rotate_rows(const RotateParams &p, int n_batch, bool half, cudaStream_t stream) {
    if (!half) return rotate_heads<T, V, kNeighbours, PAGED>(p, n_batch, stream);
    if (p.rot_half % V == 0) return rotate_heads<T, V, kHalves, PAGED>(p, n_batch, stream);
    if constexpr (V > 1) return rotate_heads<T, V, kCrossed, PAGED>(p, n_batch, stream);
    return DA_ERR_UNSUPPORTED;   // (every size is a multiple of 1)
}
template <typename T, bool PAGED>
static int rotate_by(const RotateParams &p, int n_batch, bool half, int v, cudaStream_t stream) {
    constexpr int MOST = 16 / (int)sizeof(T);
    if (v >= MOST) return rotate_rows<T, MOST, PAGED>(p, n_batch, half, stream);
    if (v >= 2) return rotate_rows<T, 2, PAGED>(p, n_batch, half, stream);
    return rotate_rows<T, 1, PAGED>(p, n_batch, half, stream);
}

// One file per element type (rotate_f32.cu and so on) has all forms of its kernel.
template <typename T> static int rotate_any(const RotateParams &p, bool paged, int n_batch, bool half, int v, cudaStream_t stream) {
    return paged ? rotate_by<T, true>(p, n_batch, half, v, stream) : rotate_by<T, false>(p, n_batch, half, v, stream);
}
int rotate_f32(const RotateParams &p, bool paged, int n_batch, bool half, int v, cudaStream_t stream);
int rotate_f16(const RotateParams &p, bool paged, int n_batch, bool half, int v, cudaStream_t stream);
int rotate_bf16(const RotateParams &p, bool paged, int n_batch, bool half, int v, cudaStream_t stream);

}  // namespace da
