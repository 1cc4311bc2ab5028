// Attention of one new token per sequence over a paged cache: what the kernels of the element types share.
//
//   out[b, hq] = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q.k_t),  t in [max(0, n_b - window), n_b)
//
// Bound by memory: a cached token of a KV head is read once, for all query rows of the head, and used for four operations per
// channel and row.  So everything serves one thing: bytes in flight on every SM from the first moment to the last.
//
// Work is counted in units of 16 tokens (aligned in the sequence) of one item = (sequence, KV head, group of query
// rows).  All units of the launch form one line, item by item; a CTA takes a contiguous stretch of it, and a warp of the CTA
// a contiguous stretch of that.  Whatever the lengths are, no warp has more than one unit more than another, and
// nothing about them has to be known on the host: every warp finds its place from the lengths itself, so a captured launch
// stays right while the sequences grow.  A warp walks its stretch with a private ring of stages (one mbarrier each) that
// bulk copies (TMA) fill, one for one or more tokens: key and value rows of a token, and tokens, are contiguous in the page.  The ring runs on across the
// borders of items; there is no barrier of the CTA.  Where a unit lies in one page a single elected lane
// issues its copies: a bulk copy takes its operands from the warp, so one per lane is a loop over the lanes (60 sequences of 3000
// tokens, 64 channels: 76 us, elected 64, two tokens to a copy 61).  16-byte asynchronous copies of all lanes need fewer instructions still but
// bring in less (64 sequences of 5000 tokens, 128 channels: 221 us against 197).
//
// An item that lies in one warp's stretch is written by the warp.  Of one that does not, every warp leaves its partial result (row
// maximum, weight sum, accumulator: float32) in the workspace; the warps an item begins and ends in note their numbers there;
// and a second, dependent launch joins the parts, in the order of the line: the same lengths give the same bits.  (Joining the
// warps of a CTA in shared memory first leaves the second launch an eighth of the rows, but its code, fetched when the stream has
// just ended, took 3 to 6 us.)
//
// What 64 sequences of 5000 tokens (8 heads of 128 bf16 channels, four rows: 1.31 GB) take: 202 us, 6.5 TB/s; one of 131 072 (0.54
// GB) 87, of which some 4 before the first unit is there and 4 from the last one to the last joined row.
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
    uint32_t page_mul;                // t / page_size = (t * page_mul) >> page_shift
    int page_shift;
    int whole;                        // a unit lies in one page: page_size is a multiple of 16
    const int32_t *lengths;
    int n_sequences, window;
    unsigned char *out;
    float *lse;
    float *partials;                  // [CTA][warp][2][group_rows][D + 4]: of the item that had begun before the warp's stretch,
                                      // and of the one that begins in it and does not end there
    int2 *spans;                      // [item]: the warps (numbered through all CTAs) it begins and ends in
    int32_t *status;
    int n_kv_heads, rep, groups, group_rows;   // query rows of a KV head, in groups of at most group_rows
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

// (a 64-bit division takes some hundred instructions; nearly every line is shorter than 2^32 units)
__device__ __forceinline__ long long divide(long long n, long long d) {
    if (((n | d) >> 32) == 0) return (long long)((uint32_t)n / (uint32_t)d);
    return n / d;
}

__device__ __forceinline__ long long shfl_64(long long v, int from) {
    const int lo = __shfl_sync(DA_FULL_MASK, (int)(v & 0xffffffff), from);
    const int hi = __shfl_sync(DA_FULL_MASK, (int)(v >> 32), from);
    return ((long long)hi << 32) | (unsigned)lo;
}

// Units per (head, group) of the sequences, a lane for a run of `each` consecutive ones, and their sums up to the lane's run.
struct Survey {
    int each;
    long long mine, sum;
    __device__ __forceinline__ Survey(const PagedParams &p, int lane) {
        each = (p.n_sequences + 31) >> 5;
        if (each == 1) {                           // (below 2^32: 32 times 2^27)
            const uint32_t u = lane < p.n_sequences ? span_of(p, __ldg(p.lengths + lane)).units : 0;
            uint32_t v = u;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t w = __shfl_up_sync(DA_FULL_MASK, v, off);
                if (lane >= off) v += w;
            }
            mine = u, sum = v;
            return;
        }
        mine = 0;
        const int end = min((lane + 1) * each, p.n_sequences);
#pragma unroll 4
        for (int b = lane * each; b < end; ++b) mine += span_of(p, __ldg(p.lengths + b)).units;
        sum = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int lo = __shfl_up_sync(DA_FULL_MASK, (int)(sum & 0xffffffff), off);
            const int hi = __shfl_up_sync(DA_FULL_MASK, (int)(sum >> 32), off);
            if (lane >= off) sum += ((long long)hi << 32) | (unsigned)lo;
        }
    }
    __device__ __forceinline__ long long total() const { return shfl_64(sum, 31); }
    // of the sequences in front of `b`
    __device__ __forceinline__ long long before(const PagedParams &p, int b, int lane) const {
        const int l = b / each;
        long long front = shfl_64(sum - mine, l);
        if (each > 1) {
            long long u = 0;
            for (int i = l * each + lane; i < b; i += 32) u += span_of(p, __ldg(p.lengths + i)).units;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) u += __shfl_xor_sync(DA_FULL_MASK, u, off);
            front += u;
        }
        return front;
    }
};

// How the line is dealt out: to as many CTAs as have a unit for each of their `warps`, up to kPagedCtas, the first `more` of them
// one unit more; inside a CTA to its warps in the same way.
struct Deal {
    int ctas, more;
    long long each;
    __device__ __forceinline__ Deal(long long total, int warps) {
        const long long most = divide(total, warps);
        ctas = total <= 0 ? 0 : (most < 1 ? 1 : (most < kPagedCtas ? (int)most : kPagedCtas));
        each = ctas ? divide(total, ctas) : 0;
        more = (int)(total - each * ctas);
    }
    __device__ __forceinline__ long long begin(int c) const { return each * c + min(c, more); }
    __device__ __forceinline__ int count(int c) const { return (int)each + (c < more); }
    __device__ __forceinline__ int cta_of(long long unit) const {
        const long long long_part = (each + 1) * more;
        if (unit < long_part) return (int)divide(unit, each + 1);
        return more + (int)divide(unit - long_part, each);
    }
    // warp of the CTA's unit `at` among `warps`
    static __device__ __forceinline__ int warp_of(int count, int at, int warps) {
        const int e = count / warps, m = count - e * warps;
        if (at < (e + 1) * m) return at / (e + 1);
        return m + (at - (e + 1) * m) / e;
    }
};

template <int D> struct PagedRow { static constexpr int kWidth = D + 4; };   // accumulator, maximum, weight sum, padding

// A place in the line.
struct Cursor {
    int b, head, group;               // the item
    int u, end;                       // unit inside the sequence, and the first behind its last
    Span s;
    const int32_t *row;               // the sequence's pages
    __device__ __forceinline__ int id(const PagedParams &p) const { return (b * p.n_kv_heads + head) * p.groups + group; }
    __device__ __forceinline__ void enter(const PagedParams &p, int sequence) {
        b = sequence;
        s = span_of(p, __ldg(p.lengths + b));
        end = s.u0 + s.units;
        row = p.table + b * p.table_stride;
    }
    // to the next unit of the line (there is one)
    __device__ __forceinline__ void next(const PagedParams &p) {
        if (++u < end) return;
        if (++group == p.groups) {
            group = 0;
            if (++head == p.n_kv_heads) {
                head = 0;
                do enter(p, b + 1);
                while (s.units == 0 && b + 1 < p.n_sequences);
            }
        }
        u = s.u0;
    }
    // to unit `at` of the line
    __device__ __forceinline__ void seek(const PagedParams &p, long long at, int lane, const Survey &survey) {
        const int per = p.n_kv_heads * p.groups;
        const unsigned past = __ballot_sync(DA_FULL_MASK, survey.sum * per > at);
        const int l = past ? __ffs(past) - 1 : 31;
        long long front = shfl_64(survey.sum - survey.mine, l);
        int sequence = l * survey.each;
        if (survey.each > 1) {
            // inside the lane's run, 32 sequences at a time (their sums below 2^32)
            for (int b0 = sequence;; b0 += 32) {
                const int b = b0 + lane;
                const uint32_t u = b < min(sequence + survey.each, p.n_sequences) ? span_of(p, __ldg(p.lengths + b)).units : 0;
                uint32_t v = u;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t w = __shfl_up_sync(DA_FULL_MASK, v, off);
                    if (lane >= off) v += w;
                }
                const unsigned here = __ballot_sync(DA_FULL_MASK, (front + v) * per > at);
                if (here || b0 + 32 >= sequence + survey.each) {
                    const int i = here ? __ffs(here) - 1 : 0;
                    front += __shfl_sync(DA_FULL_MASK, v - u, i);
                    sequence = b0 + i;
                    break;
                }
                front += __shfl_sync(DA_FULL_MASK, v, 31);
            }
        }
        enter(p, min(sequence, p.n_sequences - 1));
        const long long inside = at - front * per;
        const int item = (int)divide(inside, max(s.units, 1));
        head = item / p.groups;
        group = item - head * p.groups;
        u = s.u0 + (int)(inside - (long long)item * s.units);
    }
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
// A row's maximum is -inf as long as it has no token, and at least kLowest from then on, were all its logits -inf.  So only a row
// without tokens is zeros; a weight sum of 0 (every logit -inf) or NaN (a query, or a logit, that is no number) makes the quotient NaN.
constexpr float kLowest = -3.402823466e38f;

// Running sum of partial results (max, weight sum, four accumulator columns), several at a time so that their loads and
// exponentials do not wait for one another.
struct PartialSum {
    float m, l;
    float4 o;
    __device__ __forceinline__ void clear() { m = -INFINITY, l = 0.f, o = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void add_lane(int off);     // what the lane `off` across has
    template <int N> __device__ __forceinline__ void add(const float2 (&ml)[N], const float4 (&v)[N]) {
        float mx = m;
#pragma unroll
        for (int i = 0; i < N; ++i) mx = fmaxf(mx, ml[i].x);
        const float ms = mx == -INFINITY ? 0.f : mx;
        const float old = fast_exp2(m - ms);
        m = mx;
        l *= old;
        o.x *= old, o.y *= old, o.z *= old, o.w *= old;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float w = fast_exp2(ml[i].x - ms);     // (0 for one without tokens: its sums are zero)
            l = fmaf(ml[i].y, w, l);
            o.x = fmaf(v[i].x, w, o.x), o.y = fmaf(v[i].y, w, o.y), o.z = fmaf(v[i].z, w, o.z), o.w = fmaf(v[i].w, w, o.w);
        }
    }
};

__device__ __forceinline__ void PartialSum::add_lane(int off) {
    const float2 ml[1] = {make_float2(__shfl_xor_sync(DA_FULL_MASK, m, off), __shfl_xor_sync(DA_FULL_MASK, l, off))};
    const float4 v[1] = {make_float4(__shfl_xor_sync(DA_FULL_MASK, o.x, off), __shfl_xor_sync(DA_FULL_MASK, o.y, off),
                                     __shfl_xor_sync(DA_FULL_MASK, o.z, off), __shfl_xor_sync(DA_FULL_MASK, o.w, off))};
    add(ml, v);
}

// Four consecutive elements of a row, divided by its weight sum.
template <typename T> __device__ __forceinline__ void store_divided(T *dst, const float4 &o, float m, float l) {
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(dst) = m == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
    } else {
        union { T t[4]; uint2 w; } x;
        x.t[0] = from_float<T>(o.x * inv), x.t[1] = from_float<T>(o.y * inv);
        x.t[2] = from_float<T>(o.z * inv), x.t[3] = from_float<T>(o.w * inv);
        *reinterpret_cast<uint2 *>(dst) = x.w;
    }
}

// Math: the arithmetic of a unit.  kD, kStageBytes (of a unit in shared memory), offset (of a token in it), kTogether (tokens that
// follow one another there without a gap), kScratch (bytes of a warp's own), State, begin
// (query rows), consume (one unit), attended (there was a token), publish (a partial result), write (a complete one).
template <class Math, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) paged_attention_kernel(const PagedParams p) {
    using T = typename Math::Elem;
    constexpr int D = Math::kD, PW = PagedRow<D>::kWidth;
    constexpr int ROWB = D * (int)sizeof(T), TOKB = 2 * ROWB;
    constexpr int STAGEB = Math::kStageBytes;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bars[WARPS][STAGES];
    __shared__ uint32_t masks[WARPS][STAGES];      // tokens of the unit that are there
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) mbar_init(&bars[warp][s], 1);
    }
    mbar_fence_init();
    __syncwarp();
    griddep_wait();
    griddep_launch_dependents();

    // this warp's stretch
    const Survey survey(p, lane);
    const Deal deal(survey.total() * (p.n_kv_heads * p.groups), WARPS);
    if ((int)blockIdx.x >= deal.ctas) return;
    const long long lo = deal.begin(blockIdx.x);
    const int mine = deal.count(blockIdx.x), spare = mine % WARPS;
    const int skip = mine / WARPS * warp + min(warp, spare);
    const int count = mine / WARPS + (warp < spare);
    if (count == 0) return;
    unsigned char *ring = smem + (size_t)warp * STAGES * STAGEB;
    unsigned char *scratch = smem + (size_t)WARPS * STAGES * STAGEB + (size_t)warp * Math::kScratch;

    Cursor ahead;
    ahead.seek(p, lo + skip, lane, survey);
    Cursor at = ahead;
    bool begins = at.u == at.s.u0;

    // The unit to be requested next: its tokens that there are, and its page (pages not whole: each lane's token's), looked
    // up one unit ahead; then where it lies.
    int page, slot;
    uint32_t there;
    auto look_up = [&](const Cursor &c) {
        const int t0 = c.u * kPagedUnit, t = p.whole ? t0 : t0 + (lane & 15);
        const int from = max(c.s.first - t0, 0), to = min(c.s.n - t0, kPagedUnit);
        there = (0xffffu >> (kPagedUnit - to)) & (0xffffu << from);
        const int column = (int)(((unsigned long long)(unsigned)t * p.page_mul) >> p.page_shift);
        slot = t - column * p.page_size;
        page = 0;
        if (p.whole || ((there >> (lane & 15)) & 1)) page = __ldg(c.row + column);
    };
    // Read once per call: the stream must not push the code of the joins and the partial results out of L2 (1.3 GB:
    // 204 -> 200 us).
    const uint64_t policy = l2_policy_evict_first();
    const unsigned char *src;
    auto locate = [&](const Cursor &c) {
        const bool bad = (unsigned)page >= (unsigned)p.n_pages;
        if (bad) {                             // the tokens are left out
            atomicOr(p.status, DA_STATUS_BAD_PAGE_ID);
            page = 0;
        }
        there &= ~__ballot_sync(DA_FULL_MASK, bad);
        src = p.pages + (c.head * p.page_head_stride + page * p.page_stride + (long long)slot * (2 * D)) * (long long)sizeof(T);
    };
    auto request = [&](int s) {
        unsigned char *dst = ring + s * STAGEB;
        uint64_t *bar = &bars[warp][s];
        if (p.whole && there == 0xffffu) {
            if (elect_one()) {
                masks[warp][s] = 0xffffu;
                mbar_arrive_expect_tx(bar, kPagedUnit * TOKB);
#pragma unroll
                for (int t = 0; t < kPagedUnit; t += Math::kTogether)
                    bulk_copy_g2s_hint(dst + Math::offset(t), src + t * TOKB, Math::kTogether * TOKB, bar, policy);
            }
            __syncwarp();
        } else {
            if (lane == 0) {
                masks[warp][s] = there;
                mbar_arrive_expect_tx(bar, (uint32_t)__popc(there) * TOKB);
            }
            __syncwarp();
            if (p.whole) src += lane * TOKB;
            if (lane < kPagedUnit && ((there >> lane) & 1)) bulk_copy_g2s_hint(dst + Math::offset(lane), src, TOKB, bar, policy);
        }
    };

    int issued = 0;
    look_up(ahead);
    for (; issued < STAGES && issued < count; ++issued) {
        locate(ahead);
        request(issued);
        if (issued + 1 < count) {
            ahead.next(p);
            look_up(ahead);
        }
    }

    typename Math::State st;
    int id = at.id(p);
    int rows = rows_of(p, id);
    Math::begin(st, p, at.b, at.head, at.group, rows, lane, scratch);
    int s = 0;
    uint32_t parity = 0, seen = 0;                 // seen: tokens of the item this warp has had, by their place in a unit
    for (int i = 0; i < count; ++i) {
        if (issued < count) locate(ahead);
        const bool arrived = mbar_wait_bounded(&bars[warp][s], parity);
        if (!__all_sync(DA_FULL_MASK, arrived)) {
            if (lane == 0) atomicOr(p.status, DA_STATUS_WAIT_TIMEOUT);
            // the copies under way end before the shared memory is given up, or the wait for them does
            for (; i < issued; ++i) {
                mbar_wait_bounded(&bars[warp][s], parity);
                if (++s == STAGES) s = 0, parity ^= 1;
            }
            break;
        }
        unsigned char *unit = ring + s * STAGEB;
        const uint32_t mask = masks[warp][s];
        if (mask != 0xffffu) {
            // value rows that no token filled hold stale bytes: a weight of zero times one of them must be zero
            for (int k = lane; k < kPagedUnit * (ROWB / 16); k += 32) {
                const int t = k / (ROWB / 16);
                if (!((mask >> t) & 1))
                    *reinterpret_cast<uint4 *>(unit + Math::offset(t) + ROWB + (k % (ROWB / 16)) * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the stage's next copies come after
            __syncwarp();
        }
        seen |= mask;
        Math::consume(st, unit, mask, lane, p.scale_log2);
        __syncwarp();
        if (issued < count) {
            request(s);
            if (++issued < count) {
                ahead.next(p);
                look_up(ahead);
            }
        }
        if (++s == STAGES) s = 0, parity ^= 1;
        const bool ends = at.u + 1 == at.end;
        if (!ends && i + 1 < count) {
            ++at.u;
            continue;
        }
        // the item, or this warp's part of it, is done
        if (lane == 0) {
            if (begins) p.spans[id].x = blockIdx.x * WARPS + warp;
            if (ends) p.spans[id].y = blockIdx.x * WARPS + warp;
        }
        if (seen) Math::attended(st);
        if (begins && ends) {
            Math::write(st, p, id, rows, lane);
        } else {
            Math::publish(st, p.partials + (((size_t)blockIdx.x * WARPS + warp) * 2 + (begins ? 1 : 0)) * p.group_rows * PW, lane, rows);
        }
        if (i + 1 < count) {
            at.next(p);
            id = at.id(p);
            rows = rows_of(p, id);
            begins = true;
            seen = 0;
            Math::begin(st, p, at.b, at.head, at.group, rows, lane, scratch);
        }
    }
}

template <class Math, int WARPS, int STAGES>
static cudaError_t launch_paged(const PagedParams &p, cudaStream_t stream) {
    constexpr int SMEM = WARPS * (STAGES * Math::kStageBytes + Math::kScratch);
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

// query rows that share a pass over the keys and values, float32: what the registers of a warp hold
constexpr int paged_f32_rows(int head_dim) { return head_dim <= 128 ? 8 : 4; }
constexpr int kPagedMmaRows = 16;
// Warps of the CTAs of paged_attention_kernel.
__host__ __device__ constexpr int paged_mma_warps(int head_dim) { return head_dim > 128 ? 6 : head_dim > 96 ? 8 : 12; }
__host__ __device__ constexpr int paged_f32_warps(int head_dim) { return head_dim > 128 ? 3 : head_dim > 96 ? 6 : 8; }

cudaError_t paged_attention_f32(const PagedParams &p, int head_dim, cudaStream_t stream);
cudaError_t paged_attention_f16(const PagedParams &p, int head_dim, cudaStream_t stream);
cudaError_t paged_attention_bf16(const PagedParams &p, int head_dim, cudaStream_t stream);

}  // namespace da
