// Host side of the page pool's row entry points (cqkv_paged_append, cqkv_paged_rope_append,
// cqkv_paged_dequantize): argument checks and the dispatch to the per-format kernels of paged_rows.h.
#include "paged_rows.h"

#include <algorithm>

namespace cqkv {

int check_pool(const char *who, const cqkv_side *k, const cqkv_side *v, const cqkv_pages *pages,
               int32_t total, PageTable *p) {
    for (int i = 0; i < (v ? 2 : 1); ++i) {
        const cqkv_side *s = i ? v : k;
        if (int rc = check_side(s, who)) return rc;
        if (s->format != CQKV_FMT_FP8 && s->format != CQKV_FMT_MXFP8 && s->format != CQKV_FMT_MXFP4)
            return fail(CQKV_ERR_ARG, "%s: page pools hold FP8, MXFP8 or MXFP4 rows, not format %d", who, s->format);
        if (side_rotates(s)) return fail(CQKV_ERR_ARG, "%s: page pools hold unrotated rows", who);
        if (s->capacity & (s->capacity - 1))
            return fail(CQKV_ERR_ARG, "%s: a page of %d tokens is not a power of two", who, s->capacity);
        // planes start on 16-byte boundaries: the kernels move whole 16-byte pieces
        if (((uintptr_t)s->codes | (uintptr_t)s->scales) % 16)
            return fail(CQKV_ERR_ARG, "%s: codes / scales are not 16-byte aligned", who);
    }
    if (v) {
        if (k->is_value != 0 || v->is_value != 1)
            return fail(CQKV_ERR_ARG, "%s: expected a key side and a value side", who);
        if (k->format != v->format || k->head_dim != v->head_dim || k->kv_heads != v->kv_heads ||
            k->capacity != v->capacity)
            return fail(CQKV_ERR_ARG, "%s: key / value sides differ in format, D, heads or page size", who);
    }
    if (!pages) return fail(CQKV_ERR_ARG, "%s: null pages", who);
    if (pages->batch < 0 || pages->max_pages < 0 || pages->n_pages < 0 || total < 0)
        return fail(CQKV_ERR_ARG, "%s: batch %d max_pages %d n_pages %d rows %d", who, pages->batch,
                    pages->max_pages, pages->n_pages, total);
    if (pages->batch > 0 && total > 0 && (!pages->cu_seqlens || (pages->max_pages > 0 && !pages->table)))
        return fail(CQKV_ERR_ARG, "%s: null page table or cu_seqlens", who);
    if (pages->table_stride < 0 || (pages->batch > 1 && pages->table_stride < pages->max_pages && pages->table_stride != 0))
        return fail(CQKV_ERR_ARG, "%s: table stride %lld below %d pages", who, (long long)pages->table_stride, pages->max_pages);
    if ((int64_t)pages->max_pages * k->capacity > 1 << 30)
        return fail(CQKV_ERR_ARG, "%s: %d pages of %d tokens per sequence are above 2^30", who, pages->max_pages, k->capacity);
    if (total > 1 << 28) return fail(CQKV_ERR_ARG, "%s: %d rows above 2^28", who, total);
    p->table = pages->table;
    p->stride = pages->table_stride;
    p->cu = pages->cu_seqlens;
    p->max_pages = pages->max_pages;
    p->n_pages = pages->n_pages;
    p->batch = pages->batch;
    p->total = total;
    p->shift = __builtin_ctz((unsigned)k->capacity);
    return CQKV_OK;
}

// Largest number of 8-token tiles of `total` rows in `batch` sequences: a sequence of n rows touches at
// most n tiles, and at most (n + 14) / 8.
static int64_t tiles_bound(int64_t total, int64_t batch) {
    return std::min<int64_t>(total, total / 8 + 2 * batch);
}

static bool whole16(const void *p, int64_t s0, int64_t s1, int v) {
    return (uintptr_t)p % 16 == 0 && s0 % v == 0 && s1 % v == 0;
}

// The launch of an append whose arguments but the grid are filled in.
static int append_run(const char *who, const cqkv_side *k, int rope, PagedRowsArgs &a, hipStream_t st) {
    const int dk = kernel_dim(k->head_dim), rpw = 64 / (dk / 8);
    a.k_units = a.v_units = (a.kv_heads + rpw - 1) / rpw;
    a.q_units = rope ? (a.q_heads + rpw - 1) / rpw : 0;
    const int64_t tiles = tiles_bound(a.pt.total, a.pt.batch);
    // with angles: half a tile for a wavefront, and two head groups where that leaves 4 wavefronts to every
    // SIMD (6333 tokens, FP8, 32 / 8 heads, D = 128: append and read-back 63 us with one group, 59 with two,
    // 60 with three, 68 with four, before the read-back's stores were nontemporal)
    const int64_t kq = a.k_units + a.q_units, parts = rope ? 2 : 1;
    a.per = rope && tiles * parts * kq >= 8192 ? 2 : 1;
    a.units = (int)(parts * ((kq + a.per - 1) / a.per) + a.v_units);
    const int64_t wgs = (tiles * a.units + 3) / 4;
    if (tiles * a.units > 0x7fffffffll / 64)
        return fail(CQKV_ERR_ARG, "%s: %d rows of %d head groups exceed one launch", who, a.pt.total, a.units);
    a.tiles = (int32_t)tiles;
    const dim3 grid((unsigned)wgs);
    if (k->format == CQKV_FMT_FP8) paged_append_launch_5(dk, rope, grid, st, a);
    else if (k->format == CQKV_FMT_MXFP8) paged_append_launch_4(dk, rope, grid, st, a);
    else paged_append_launch_2(dk, rope, grid, st, a);
    CQKV_HIP_CHECK(hipGetLastError());
    return CQKV_OK;
}

}  // namespace cqkv

using namespace cqkv;

extern "C" int cqkv_paged_append(const cqkv_side *k_side, const cqkv_side *v_side,
                                 const cqkv_pages *pages, const int32_t *positions, const void *k,
                                 const int64_t k_strides[2], const void *v,
                                 const int64_t v_strides[2], int32_t dtype, int32_t total,
                                 cqkv_stream_t stream) {
    clear_error();
    static const char *who = "cqkv_paged_append";
    PagedRowsArgs a = {};
    if (!k_side || !v_side) return fail(CQKV_ERR_ARG, "%s: null side", who);
    if (int rc = check_pool(who, k_side, v_side, pages, total, &a.pt)) return rc;
    if (dtype < CQKV_BF16 || dtype > CQKV_F32) return fail(CQKV_ERR_ARG, "%s: dtype %d", who, dtype);
    if (total == 0 || pages->batch == 0) return CQKV_OK;
    if (!k || !v || !k_strides || !v_strides || !positions)
        return fail(CQKV_ERR_ARG, "%s: null pointer argument", who);
    a.positions = positions;
    a.k = pool_side(k_side);
    a.v = pool_side(v_side);
    a.kx = k;
    a.vx = v;
    a.k_st = k_strides[0];
    a.k_sh = k_strides[1];
    a.v_st = v_strides[0];
    a.v_sh = v_strides[1];
    a.dim = k_side->head_dim;
    a.dtype = dtype;
    a.kv_heads = k_side->kv_heads;
    a.vec = dtype != CQKV_F32 && a.dim % 8 == 0 && whole16(k, a.k_st, a.k_sh, 8) && whole16(v, a.v_st, a.v_sh, 8);
    return append_run(who, k_side, 0, a, (hipStream_t)stream);
}

extern "C" int cqkv_paged_rope_append(const cqkv_side *k_side, const cqkv_side *v_side,
                                      const cqkv_pages *pages, const int32_t *positions,
                                      const void *q, const int64_t q_strides[2], const void *k,
                                      const int64_t k_strides[2], const void *v,
                                      const int64_t v_strides[2], int32_t dtype, int32_t total,
                                      int32_t q_heads, const void *cos, const void *sin,
                                      int32_t cs_rows, int32_t rope_kind, int32_t axes,
                                      const int32_t *rope_positions, int64_t rope_stride,
                                      const uint8_t *pair_axis, void *q_out,
                                      const int64_t q_out_strides[2], cqkv_stream_t stream) {
    clear_error();
    static const char *who = "cqkv_paged_rope_append";
    PagedRowsArgs a = {};
    if (!k_side || !v_side) return fail(CQKV_ERR_ARG, "%s: null side", who);
    if (int rc = check_pool(who, k_side, v_side, pages, total, &a.pt)) return rc;
    if (dtype < CQKV_BF16 || dtype > CQKV_F32) return fail(CQKV_ERR_ARG, "%s: dtype %d", who, dtype);
    if (rope_kind != CQKV_ROPE_HALVES && rope_kind != CQKV_ROPE_INTERLEAVED)
        return fail(CQKV_ERR_ARG, "%s: rope kind %d", who, rope_kind);
    const int dim = k_side->head_dim;
    if (dim % 2 != 0) return fail(CQKV_ERR_ARG, "%s: rotary embedding of an odd head_dim %d", who, dim);
    if (q_heads <= 0) return fail(CQKV_ERR_ARG, "%s: q_heads %d", who, q_heads);
    if (cs_rows <= 0) return fail(CQKV_ERR_ARG, "%s: cos / sin rows %d", who, cs_rows);
    if (axes < 1 || axes > 4) return fail(CQKV_ERR_ARG, "%s: %d rotary axes (1-4)", who, axes);
    if (!pair_axis) return fail(CQKV_ERR_ARG, "%s: null pair_axis", who);
    for (int j = 0; j < dim / 2; ++j) {
        if (pair_axis[j] >= axes)
            return fail(CQKV_ERR_ARG, "%s: pair %d has axis %d of %d", who, j, pair_axis[j], axes);
        a.axis[j >> 4] |= (uint32_t)pair_axis[j] << (2 * (j & 15));
        if (j % 8 && pair_axis[j] != pair_axis[j - 1]) a.mixed = 1;
    }
    if (total == 0 || pages->batch == 0) return CQKV_OK;
    if (!q || !k || !v || !q_out || !q_strides || !k_strides || !v_strides || !q_out_strides || !cos ||
        !sin || !rope_positions || !positions)
        return fail(CQKV_ERR_ARG, "%s: null pointer argument", who);
    if (axes > 1 && rope_stride < total)
        return fail(CQKV_ERR_ARG, "%s: rope position stride %lld below %d rows", who, (long long)rope_stride, total);
    a.positions = positions;
    a.k = pool_side(k_side);
    a.v = pool_side(v_side);
    a.q = q;
    a.kx = k;
    a.vx = v;
    a.q_out = q_out;
    a.q_st = q_strides[0];
    a.q_sh = q_strides[1];
    a.k_st = k_strides[0];
    a.k_sh = k_strides[1];
    a.v_st = v_strides[0];
    a.v_sh = v_strides[1];
    a.o_st = q_out_strides[0];
    a.o_sh = q_out_strides[1];
    a.cos = cos;
    a.sin = sin;
    a.cs_rows = cs_rows;
    a.axes = axes;
    a.rope_pos = rope_positions;
    a.rope_stride = rope_stride;
    a.dim = dim;
    a.dtype = dtype;
    a.kv_heads = k_side->kv_heads;
    a.q_heads = q_heads;
    // table rows of dim / 2 elements: whole 16-byte pieces (halves), as the chunks' partners
    a.vec = dtype != CQKV_F32 && dim % 16 == 0 && whole16(k, a.k_st, a.k_sh, 8) && whole16(v, a.v_st, a.v_sh, 8) &&
            whole16(q, a.q_st, a.q_sh, 8) && whole16(q_out, a.o_st, a.o_sh, 8) && (uintptr_t)cos % 16 == 0 &&
            (uintptr_t)sin % 16 == 0;
    return append_run(who, k_side, rope_kind, a, (hipStream_t)stream);
}

extern "C" int cqkv_paged_dequantize(const cqkv_side *side, const cqkv_pages *pages,
                                     const int32_t *positions, int32_t total, void *out,
                                     int32_t out_dtype, const int64_t out_strides[2],
                                     cqkv_stream_t stream) {
    clear_error();
    static const char *who = "cqkv_paged_dequantize";
    PagedRowsArgs a = {};
    if (!side) return fail(CQKV_ERR_ARG, "%s: null side", who);
    if (int rc = check_pool(who, side, nullptr, pages, total, &a.pt)) return rc;
    if (out_dtype < CQKV_BF16 || out_dtype > CQKV_F32) return fail(CQKV_ERR_ARG, "%s: dtype %d", who, out_dtype);
    if (total == 0 || pages->batch == 0) return CQKV_OK;
    if (!out || !out_strides || !positions) return fail(CQKV_ERR_ARG, "%s: null pointer argument", who);
    a.positions = positions;
    a.k = pool_side(side);
    a.side_is_value = side->is_value;
    a.out = out;
    a.out_st = out_strides[0];
    a.out_sh = out_strides[1];
    a.out_dtype = out_dtype;
    a.dim = side->head_dim;
    a.kv_heads = side->kv_heads;
    a.out_vec = a.dim % 8 == 0 && whole16(out, a.out_st, a.out_sh, out_dtype == CQKV_F32 ? 4 : 8);
    const int dk = kernel_dim(a.dim), rpw = 64 / (dk / 8);
    a.units = (a.kv_heads + rpw - 1) / rpw;
    const int64_t tiles = tiles_bound(total, pages->batch);
    if (tiles * a.units > 0x7fffffffll / 64)
        return fail(CQKV_ERR_ARG, "%s: %d rows of %d head groups exceed one launch", who, total, a.units);
    a.tiles = (int32_t)tiles;
    const dim3 grid((unsigned)((tiles * a.units + 3) / 4));
    hipStream_t st = (hipStream_t)stream;
    if (side->format == CQKV_FMT_FP8) paged_dequant_launch_5(dk, grid, st, a);
    else if (side->format == CQKV_FMT_MXFP8) paged_dequant_launch_4(dk, grid, st, a);
    else paged_dequant_launch_2(dk, grid, st, a);
    CQKV_HIP_CHECK(hipGetLastError());
    return CQKV_OK;
}
