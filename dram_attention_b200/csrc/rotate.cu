// Rotary positions and the append to a paged cache: the host side (rotate.cuh has the kernel).

#include "rotate.cuh"

namespace da {

static int rotate(const RotateParams &p, bool paged, int n_batch, int dtype, bool half, int v, cudaStream_t stream) {
    switch (dtype) {
    case DA_F32: return rotate_f32(p, paged, n_batch, half, v, stream);
    case DA_F16: return rotate_f16(p, paged, n_batch, half, v, stream);
    default: return rotate_bf16(p, paged, n_batch, half, v, stream);
    }
}

// Elements of the longest power of two up to 16 bytes that divides all of them: the addresses (bytes), the strides and sizes (elements).
static int access_elements(uintptr_t bases, int64_t elements, int esize) {
    int v = 16 / esize;
    while (v > 1 && ((bases & (uintptr_t)(v * esize - 1)) || (elements & (v - 1)))) v >>= 1;
    return v;
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
        (a.q && !small(a.n_q_heads, 1, 1 << 14)) || (a.k && !small(a.n_kv_heads, 1, 1 << 14)))
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
    p.n_tokens = p.position_tokens = (int)a.n_tokens;
    int n_batch = (int)a.n_batch;
    // batch entries that follow one another as tokens do are one sequence of tokens
    bool joined = true;
    for (int i = 0; i < 2; ++i) joined = joined && (!src[i] || p.src_batch[i] == p.src_token[i] * a.n_tokens);
    if (joined) p.n_tokens *= n_batch, n_batch = 1;
    p.head_dim = (int)a.head_dim, p.rot_half = (int)a.rotary_dim / 2;
    p.inv_freq = a.inv_freq, p.factor = (float)a.factor, p.sign = a.transposed ? -1.f : 1.f;
    p.positions = a.positions, p.positions_64 = a.positions_64 != 0;
    p.position_batch = a.position_strides[0], p.position_token = a.position_strides[1];
    const bool half = a.interleaved == 0;
    const int v = access_elements(bases, strides | a.head_dim, esize);
    return rotate(p, false, n_batch, (int)a.dtype, half, v, static_cast<cudaStream_t>(a.stream));
}

extern "C" int da_append_pages(const da_append_pages_args *args) {
    using namespace da;
    if (!args) return DA_ERR_NULL;
    const da_append_pages_args &a = *args;
    if (!a.k || !a.v || !a.pages || !a.page_table || !a.lengths || !a.status || (a.q && (!a.q_out || !a.inv_freq)))
        return DA_ERR_NULL;
    if (!small(a.dtype, DA_F32, DA_BF16)) return DA_ERR_DTYPE;
    if (!small(a.n_rows, 1, 1 << 30) || !small(a.n_sequences, 1, 1 << 30) || (!a.starts && a.n_rows != a.n_sequences) ||
        !small(a.head_dim, 2, 512) || (a.q && !small(a.n_q_heads, 1, 1 << 14)) || !small(a.n_kv_heads, 1, 1 << 14) ||
        !small(a.page_size, 1, 1 << 30) || !small(a.n_pages, 1, 0x7fffffff) || !small(a.table_columns, 1, 0x7fffffff) ||
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
    const bool half = a.interleaved == 0;
    const int v = access_elements(bases, strides | a.head_dim, esize);
    return rotate(p, true, 1, (int)a.dtype, half, v, static_cast<cudaStream_t>(a.stream));
}
