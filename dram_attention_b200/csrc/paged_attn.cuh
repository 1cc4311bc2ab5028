// Attention of one new token per sequence over a paged cache: what the kernels of the element types share.
//
//   out[b, hq] = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q.k_t),  t in [max(0, n_b - window), n_b)
//
// Bound by memory: a cached token of a KV head is read once, for all query rows of the head, and used for 4 rows x D
// operations per channel pair.  So everything serves one thing: bytes in flight on every SM from the first moment to the last.
//
// Work is counted in units of 16 tokens (aligned in the sequence) of one item = (sequence, KV head, group of query
// rows).  All units of the launch form one line, item by item; a CTA takes a contiguous stretch of it, and a warp of the CTA
// a contiguous stretch of that.  Whatever the lengths are, no warp has more than one unit more than another, and
// nothing about them has to be known on the host: every warp finds its place from the lengths itself, so a captured launch
// stays right while the sequences grow.  A warp walks its stretch with a private ring of stages (one mbarrier each) that
// bulk copies (TMA) fill, one per token: its key and value rows are contiguous in the page.  The ring runs on across the
// borders of items; there is no barrier of the CTA until its stretch is done.
//
// An item that lies in one warp's stretch is written by the warp.  One that crosses warps is put together by the CTA from the
// warps' partial results (row maximum, weight sum, accumulator: float32), and one that crosses CTAs by a second,
// dependent launch from the CTAs' partial results: a CTA leaves at most two, for the item it begins in and the one it ends
// in.  The joins go in the order of the line, so the same lengths give the same bits.
#pragma once

#include "da_common.cuh"

namespace da {

constexpr int kPagedUnit = 16;        // tokens
constexpr int kPagedCtas = 148;       // one per SM

struct PagedParams {
    const unsigned char *q;
    long long q_seq, q_head;          // elements
    const unsigned char *pages;
    long long page_stride, page_head_stride;   // elements
    int n_pages, page_size;
    const int32_t *table;
    long long table_stride;
    int capacity;                     // tokens a row of the table has room for
    const int32_t *lengths;
    int n_sequences, window;
    unsigned char *out;
    float *lse;
    float *warp_partials;             // [CTA][warp][group_rows][D + 4]
    float *cta_partials;              // [CTA][2][group_rows][D + 4]
    int32_t *status;
    int n_kv_heads, rep, groups, group_rows;   // query rows of a KV head, in groups of at most group_rows
    int min_units;                    // fewer units than this are not worth a CTA of their own
    float scale_log2;
};

// The part of a sequence that is attended to.
struct Span {
    int first, n;                     // tokens [first, n)
    int u0, units;                    // first unit and number of units
};
__device__ __forceinline__ Span span_of(const PagedParams &p, int length) {
    Span s;
    s.n = min(max(length, 0), p.capacity);
    s.first = p.window > 0 && s.n > p.window ? s.n - p.window : 0;
    s.u0 = s.first / kPagedUnit;
    s.units = s.n > 0 ? (s.n + kPagedUnit - 1) / kPagedUnit - s.u0 : 0;
    return s;
}

__device__ __forceinline__ long long shfl_up_64(long long v, int by) {
    const int lo = __shfl_up_sync(DA_FULL_MASK, (int)(v & 0xffffffff), by);
    const int hi = __shfl_up_sync(DA_FULL_MASK, (int)(v >> 32), by);
    return ((long long)hi << 32) | (unsigned)lo;
}
__device__ __forceinline__ long long shfl_64(long long v, int from) {
    const int lo = __shfl_sync(DA_FULL_MASK, (int)(v & 0xffffffff), from);
    const int hi = __shfl_sync(DA_FULL_MASK, (int)(v >> 32), from);
    return ((long long)hi << 32) | (unsigned)lo;
}

// Units of the whole launch, and of the sequences in front of `before` (all warps of a CTA compute the same).
struct Totals {
    long long all, before;
};
__device__ __forceinline__ Totals total_units(const PagedParams &p, int before, int lane) {
    long long all = 0, front = 0;
    for (int b = lane; b < p.n_sequences; b += 32) {
        const int u = span_of(p, __ldg(p.lengths + b)).units;
        all += u;
        if (b < before) front += u;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        all += __shfl_xor_sync(DA_FULL_MASK, all, off);
        front += __shfl_xor_sync(DA_FULL_MASK, front, off);
    }
    const int per = p.n_kv_heads * p.groups;
    return {all * per, front * per};
}

// Sequence that unit `at` of the line lies in, and the line's position of its first unit.
__device__ __forceinline__ void find_sequence(const PagedParams &p, long long at, int lane, int &b, long long &start) {
    const int per = p.n_kv_heads * p.groups;
    long long front = 0;
    for (int b0 = 0; b0 < p.n_sequences; b0 += 32) {
        const long long mine = b0 + lane < p.n_sequences ? (long long)span_of(p, __ldg(p.lengths + b0 + lane)).units * per : 0;
        long long sum = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long v = shfl_up_64(sum, off);
            if (lane >= off) sum += v;
        }
        const unsigned past = __ballot_sync(DA_FULL_MASK, front + sum > at);
        if (past) {
            const int l = __ffs(past) - 1;
            b = b0 + l;
            start = front + shfl_64(sum - mine, l);
            return;
        }
        front += shfl_64(sum, 31);
    }
    b = p.n_sequences - 1;   // (not reached: `at` is below the total)
    start = front;
}

// How the line is dealt out.  CTA c has the units [c * total / ctas, (c + 1) * total / ctas).
__device__ __forceinline__ int paged_ctas(const PagedParams &p, long long total, int most) {
    const long long want = (total + p.min_units - 1) / p.min_units;
    return (int)(want < most ? want : most);
}
__device__ __forceinline__ long long cta_begin(long long total, int ctas, int c) { return total * c / ctas; }
__device__ __forceinline__ int cta_of(long long total, int ctas, long long unit) {
    return (int)(((unit + 1) * ctas - 1) / total);
}

template <int D> struct PagedRow { static constexpr int kWidth = D + 4; };   // accumulator, maximum, weight sum, padding

// A place in the line.
struct Cursor {
    int b, item;                      // item: (head, group) inside the sequence
    int u;                            // unit inside the sequence
    Span s;
};
__device__ __forceinline__ void cursor_next(const PagedParams &p, Cursor &c) {
    if (++c.u < c.s.u0 + c.s.units) return;
    if (++c.item < p.n_kv_heads * p.groups) {
        c.u = c.s.u0;
        return;
    }
    c.item = 0;
    while (c.b + 1 < p.n_sequences) {
        ++c.b;
        c.s = span_of(p, __ldg(p.lengths + c.b));
        if (c.s.units) break;
    }
    c.u = c.s.u0;
}

// What a warp leaves to its CTA: a partial result of an item, and whether the item begins and ends in the warp's stretch.
struct WarpPart {
    int item;                         // (sequence, head, group), -1: none
    bool begins, ends;
    const float *rows;
};

template <typename T> __device__ __forceinline__ T *out_row(const PagedParams &p, int item, int row, int D, size_t &index) {
    const int g = item % p.groups, bh = item / p.groups;
    index = (size_t)bh * p.rep + (size_t)g * p.group_rows + row;
    return reinterpret_cast<T *>(p.out) + index * D;
}
__device__ __forceinline__ int rows_of(const PagedParams &p, int item) {
    return min(p.group_rows, p.rep - (item % p.groups) * p.group_rows);
}
__device__ __forceinline__ float natural_lse(float m, float l) { return (m + log2f(l)) * 0.6931471805599453f; }

// Math: the arithmetic of a unit.  kD, kPitch (bytes of a token in shared memory), State, begin (query rows),
// consume (one unit), publish (a partial result), write (a complete one).
template <class Math, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) paged_attention_kernel(const PagedParams p) {
    using T = typename Math::Elem;
    constexpr int D = Math::kD, PW = PagedRow<D>::kWidth;
    constexpr int ROWB = D * (int)sizeof(T), TOKB = 2 * ROWB;
    constexpr int STAGEB = kPagedUnit * Math::kPitch;
    static_assert(STAGES * STAGEB >= Math::kRows * PW * 4, "a warp's ring holds its last partial result");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bars[WARPS][STAGES];
    __shared__ uint32_t masks[WARPS][STAGES];      // tokens of the unit that are there
    __shared__ WarpPart parts[WARPS][2];           // in the order of the line
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) mbar_init(&bars[warp][s], 1);
        parts[warp][0].item = parts[warp][1].item = -1;
    }
    mbar_fence_init();
    __syncwarp();
    griddep_wait();
    griddep_launch_dependents();

    // ---- this warp's stretch ------------------------------------------------------------
    const long long total = total_units(p, 0, lane).all;
    const int ctas = paged_ctas(p, total, gridDim.x);
    if ((int)blockIdx.x >= ctas) return;
    const long long lo = cta_begin(total, ctas, blockIdx.x), hi = cta_begin(total, ctas, blockIdx.x + 1);
    const long long begin = lo + (hi - lo) * warp / WARPS;
    const int count = (int)(lo + (hi - lo) * (warp + 1) / WARPS - begin);
    unsigned char *ring = smem + (size_t)warp * STAGES * STAGEB;

    if (count > 0) {
        Cursor ahead;
        long long start;
        find_sequence(p, begin, lane, ahead.b, start);
        ahead.s = span_of(p, __ldg(p.lengths + ahead.b));
        ahead.item = (int)((begin - start) / ahead.s.units);
        ahead.u = ahead.s.u0 + (int)((begin - start) % ahead.s.units);
        Cursor at = ahead;
        bool begins = at.u == at.s.u0;

        // a lane's token of the unit: the page it lies in, and its place there
        int page, slot;
        auto look_up = [&](const Cursor &c) {
            const int t = c.u * kPagedUnit + lane;
            page = -2;                             // no such token
            slot = 0;
            if (lane < kPagedUnit && t >= c.s.first && t < c.s.n) {
                const int column = t / p.page_size;
                slot = t - column * p.page_size;
                page = __ldg(p.table + c.b * p.table_stride + column);
                if (page < 0 || page >= p.n_pages) page = -1;
            }
        };
        auto issue = [&](const Cursor &c, int s) {
            if (page == -1) atomicOr(p.status, DA_STATUS_BAD_PAGE_ID);   // the token is left out
            const unsigned mask = __ballot_sync(DA_FULL_MASK, page >= 0);
            if (lane == 0) {
                masks[warp][s] = mask;
                mbar_arrive_expect_tx(&bars[warp][s], (uint32_t)__popc(mask) * TOKB);
            }
            __syncwarp();
            if (page >= 0) {
                const unsigned char *src = p.pages + ((c.item / p.groups) * p.page_head_stride + page * p.page_stride +
                                                      (long long)slot * 2 * D) * (long long)sizeof(T);
                bulk_copy_g2s(ring + s * STAGEB + lane * Math::kPitch, src, TOKB, &bars[warp][s]);
            }
        };

        int issued = 0;
        look_up(ahead);
        for (; issued < STAGES && issued < count; ++issued) {
            issue(ahead, issued);
            if (issued + 1 < count) {
                cursor_next(p, ahead);
                look_up(ahead);
            }
        }

        typename Math::State st;
        int id = at.b * (p.n_kv_heads * p.groups) + at.item;
        int rows = rows_of(p, id);
        Math::begin(st, p, at.b, at.item, rows, lane);
        int in_flight_from = 0;
        bool dead = false;
        for (int i = 0; i < count; ++i) {
            const int s = i % STAGES;
            const bool arrived = mbar_wait_bounded(&bars[warp][s], (uint32_t)((i / STAGES) & 1));
            if (!__all_sync(DA_FULL_MASK, arrived)) {
                if (lane == 0) atomicOr(p.status, DA_STATUS_WAIT_TIMEOUT);
                dead = true;
                in_flight_from = i;
                break;
            }
            unsigned char *unit = ring + s * STAGEB;
            const uint32_t mask = masks[warp][s];
            if (mask != 0xffffu) {
                // value rows that no token filled hold stale bytes: a weight of zero times one of them must be zero
                for (int k = lane; k < kPagedUnit * (ROWB / 16); k += 32) {
                    const int t = k / (ROWB / 16);
                    if (!((mask >> t) & 1))
                        *reinterpret_cast<uint4 *>(unit + t * Math::kPitch + ROWB + (k % (ROWB / 16)) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the stage's next copies come after
                __syncwarp();
            }
            Math::consume(st, unit, mask, lane, p.scale_log2);
            __syncwarp();
            if (issued < count) {
                issue(ahead, issued % STAGES);
                if (++issued < count) {
                    cursor_next(p, ahead);
                    look_up(ahead);
                }
            }
            const bool ends = at.u + 1 == at.s.u0 + at.s.units;
            if (!ends && i + 1 < count) {
                ++at.u;
                continue;
            }
            // ---- the item, or this warp's part of it, is done ------------------------------
            if (begins && ends) {
                Math::write(st, p, id, rows, lane);
            } else {
                const bool last = i + 1 == count;
                float *dst = last ? reinterpret_cast<float *>(ring)
                                  : p.warp_partials + ((size_t)blockIdx.x * WARPS + warp) * p.group_rows * PW;
                Math::publish(st, dst, lane, rows);
                if (lane == 0) parts[warp][last ? 1 : 0] = {id, begins, ends, dst};
            }
            if (i + 1 < count) {
                cursor_next(p, at);
                id = at.b * (p.n_kv_heads * p.groups) + at.item;
                rows = rows_of(p, id);
                begins = true;
                Math::begin(st, p, at.b, at.item, rows, lane);
            }
        }
        if (dead)   // the copies under way end before the shared memory is given up, or the wait for them does
            for (int i = in_flight_from; i < issued; ++i) mbar_wait_bounded(&bars[warp][i % STAGES], (uint32_t)((i / STAGES) & 1));
    }
    __syncthreads();

    // ---- items that cross warps -------------------------------------------------------------
    int k = 0;
    while (k < 2 * WARPS) {
        const WarpPart lead = parts[k >> 1][k & 1];
        if (lead.item < 0) {
            ++k;
            continue;
        }
        int end = k + 1;
        bool ends = lead.ends;
        for (int j = k + 1; j < 2 * WARPS; ++j) {
            const WarpPart &x = parts[j >> 1][j & 1];
            if (x.item < 0) continue;
            if (x.item != lead.item) break;
            end = j + 1;
            ends = x.ends;
        }
        const bool complete = lead.begins && ends;
        const int rows = rows_of(p, lead.item);
        float *dst = p.cta_partials + ((size_t)blockIdx.x * 2 + (lead.begins ? 1 : 0)) * p.group_rows * PW;
        for (int e = tid; e < rows * PW; e += WARPS * 32) {
            const int r = e / PW, c = e % PW;
            float m = -INFINITY;
            for (int j = k; j < end; ++j) {
                const WarpPart &x = parts[j >> 1][j & 1];
                if (x.item >= 0) m = fmaxf(m, x.rows[r * PW + D]);
            }
            const float ms = m == -INFINITY ? 0.f : m;
            float sum = 0.f, l = 0.f;
            for (int j = k; j < end; ++j) {
                const WarpPart &x = parts[j >> 1][j & 1];
                if (x.item < 0) continue;
                const float w = fast_exp2(x.rows[r * PW + D] - ms);
                sum = fmaf(x.rows[r * PW + min(c, D + 1)], w, sum);
                l = fmaf(x.rows[r * PW + D + 1], w, l);
            }
            if (!complete) {
                dst[e] = c == D ? m : sum;
            } else if (c < D) {
                size_t index;
                out_row<T>(p, lead.item, r, D, index)[c] = from_float<T>(l > 0.f ? sum / l : 0.f);
            } else if (c == D && p.lse) {
                size_t index;
                out_row<T>(p, lead.item, r, D, index);
                p.lse[index] = natural_lse(m, l);
            }
        }
        k = end;
    }
}

template <class Math, int WARPS, int STAGES>
static cudaError_t launch_paged(const PagedParams &p, cudaStream_t stream) {
    constexpr int SMEM = WARPS * STAGES * kPagedUnit * Math::kPitch;
    static_assert(SMEM <= 224 * 1024, "");
    auto kernel = paged_attention_kernel<Math, WARPS, STAGES>;
    static bool ready[64] = {};
    int dev;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return e;
        ready[dev] = true;
    }
    return launch_dependent(kernel, dim3(kPagedCtas), dim3(WARPS * 32), (size_t)SMEM, stream, p);
}

constexpr int kPagedMaxWarps = 12;
// query rows that share a pass over the keys and values, float32: what the registers of a warp hold
constexpr int paged_f32_rows(int head_dim) { return head_dim <= 64 ? 8 : (head_dim <= 128 ? 4 : 2); }
constexpr int kPagedMmaRows = 16;

cudaError_t paged_attention_f32(const PagedParams &p, int head_dim, cudaStream_t stream);
cudaError_t paged_attention_f16(const PagedParams &p, int head_dim, cudaStream_t stream);
cudaError_t paged_attention_bf16(const PagedParams &p, int head_dim, cudaStream_t stream);

}  // namespace da
