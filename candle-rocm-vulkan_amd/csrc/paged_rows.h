// Rows of a page pool (included by paged_inst.hip, one object per format, and by paged_rows.hip for the
// arguments): quantize-and-append into pages (cqkv_paged_append), the same with rotary
// positions of several axes applied to q and k (cqkv_paged_rope_append), and the read-back
// (cqkv_paged_dequantize). The codes are those of the dense appends (RowCodec::quantize_row,
// candle-core/src/accel/turbo.rs:324-374): FP8 code = E4M3(x / s) with s = absmax / 448 of the row;
// MX scale 2^e with e = floor(log2 absmax) - emax of 32 elements, code = E4M3 / E2M1(x / 2^e).
//
// Work split: a wavefront takes one 8-token tile of one sequence (tiles of positions, so a value
// tile and a page belong to one wavefront) and the heads that fill its lanes. D / 8 lanes hold a row,
// 8 elements each, so every load and store of a row is whole 16-byte pieces of one contiguous range
// and the eight tokens' loads are in flight together. A lane then holds the 8 x 8 block of codes that
// is 64 (or 32) contiguous bytes of a value tile: the transpose is byte permutes in registers, with no
// LDS and no barrier. Bound by HBM; single tokens by the latency of the chain sequence -> page -> row. 8192 tokens into MXFP4, 8 kv heads of
// 128: 13 us (3.3 TB/s of rows and codes); 6333 tokens rotated on three axes into FP8, 32 / 8 heads: 39 us
// (3.9 TB/s); 48769 rows of one FP8 side read back: 24 us (6.2 TB/s); 64 single tokens: 4.9 us.
#pragma once

#include <type_traits>

#include "paged.h"

namespace cqkv {

struct PagedRowsArgs {
    PageTable pt;
    const int32_t *positions;  // first position of every sequence's rows
    PoolSide k, v;
    const void *q, *kx, *vx;   // rows (total, heads, dim); element strides token, head
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    void *q_out;
    int64_t o_st, o_sh;
    const void *cos, *sin;     // (cs_rows, dim / 2) tables of the dtype
    const int32_t *rope_pos;   // (axes, total)
    int64_t rope_stride;
    uint32_t axis[8];          // 2 bits per rotary pair: its axis
    uint32_t mixed;            // the pairs of some 8 neighbours have different axes
    int32_t cs_rows, axes;
    int32_t dim, dtype, kv_heads, q_heads;
    int32_t vec;               // rows, tables and strides are whole 16-byte pieces (16-bit dtypes)
    int32_t q_units, k_units, v_units;  // head groups of a tile's q, k and v
    int32_t per;               // groups of k and q that a wavefront takes (append)
    int32_t units;             // wavefronts of a tile
    // read-back
    void *out;
    int64_t out_st, out_sh;
    int32_t out_dtype, out_vec, side_is_value, tiles;
};

// Sequence and tile of linear tile index `idx`: the tiles of sequence b cover positions
// [positions[b], positions[b] + len). Lane l looks at sequence base + l, 64 at a time, so the search
// costs the latency of one load and one scan whatever the batch. False past the last tile.
struct TileAt {
    int b, first, len, pos, tile;
};
__device__ inline bool find_tile(const PageTable &p, const int32_t *positions, int idx, int lane,
                                 TileAt &t) {
    for (int base = 0; base < p.batch; base += 64) {
        const int b = base + lane;
        int first = 0, len = 0, pos = 0, n = 0;
        if (b < p.batch) {
            first = min(max(p.cu[b], 0), p.total);
            len = min(max(p.cu[b + 1], first), p.total) - first;
            pos = positions[b];
            // positions below zero, and rows past the largest one, have no place
            len = pos < 0 ? 0 : min(len, 0x7fffffc0 - min(pos, 0x7fffffc0));
            n = len > 0 ? (pos + len - 1) / 8 - pos / 8 + 1 : 0;
        }
        int sum = n;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(sum, m);
            if (lane >= m) sum += o;
        }
        const uint64_t past = __ballot(sum > idx);
        if (past) {
            const int w = __builtin_ctzll(past);
            t.b = base + w;
            t.first = __builtin_amdgcn_readlane(first, w);
            t.len = __builtin_amdgcn_readlane(len, w);
            t.pos = __builtin_amdgcn_readlane(pos, w);
            t.tile = t.pos / 8 + idx - __builtin_amdgcn_readlane(sum - n, w);
            return true;
        }
        idx -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// Maximum over the LPR lanes (8, 16 or 32, aligned) of a row, over quads by DPP (maxima within a quad,
// then mirrored halves and rows: every lane of a group already holds its maximum).
template <int CTRL>
__device__ inline float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true)));
}
__device__ inline float quad_max(float v) { return dpp_max<0x4E>(dpp_max<0xB1>(v)); }
template <int LPR>
__device__ inline float row_max_lanes(float v) {
    v = dpp_max<0x141>(quad_max(v));            // row_half_mirror: 8 lanes
    if constexpr (LPR >= 16) v = dpp_max<0x140>(v);  // row_mirror: 16
    if constexpr (LPR == 32) v = xor16_max(v);
    return v;
}

// 8 elements from `p` (the row's elements j0 .. j0 + 7; elements from `dim` on are zero)
__device__ inline void raw_to_f32x8(const u32x4 &w, bool bf, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = w[i] & 0xffffu, hi = w[i] >> 16;
        x[2 * i] = bf ? bf16_bits_to_f32(lo) : f16_bits_to_f32(lo);
        x[2 * i + 1] = bf ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi);
    }
}
__device__ inline void load_any8(const void *x, int64_t row, int j0, int dim, int dtype, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = j0 + e < dim ? load_elem(x, row + j0 + e, dtype) : 0.0f;
}

// Axis of rotary pair j.
__device__ inline int pair_axis(const PagedRowsArgs &a, int j) { return (a.axis[j >> 4] >> (2 * (j & 15))) & 3; }

__device__ inline int axis_row(const int (&row)[4], int ax) {
    return ax == 0 ? row[0] : ax == 1 ? row[1] : ax == 2 ? row[2] : row[3];
}

// cos and sin of the pairs of elements e0 .. e0 + 7, as they are in the tables (16-bit): halves the 8 pairs
// e0 .. modulo dim / 2, interleaved the 4 pairs e0 / 2 .. in two words.
template <int ROPE, bool MIXED>
__device__ inline void load_angles(const PagedRowsArgs &a, const int (&row)[4], int e0, u32x4 &c, u32x4 &s) {
    const int half = a.dim / 2, j0 = ROPE == CQKV_ROPE_INTERLEAVED ? e0 >> 1 : e0 >= half ? e0 - half : e0;
    const uint16_t *ct = (const uint16_t *)a.cos + j0, *st = (const uint16_t *)a.sin + j0;
    if constexpr (!MIXED) {  // one axis for them
        const int64_t at = (int64_t)axis_row(row, pair_axis(a, j0)) * half;
        if constexpr (ROPE == CQKV_ROPE_INTERLEAVED) {
            const u32x2 cw = *(const u32x2 *)(ct + at), sw = *(const u32x2 *)(st + at);
            c = u32x4{cw.x, cw.y, 0u, 0u};
            s = u32x4{sw.x, sw.y, 0u, 0u};
        } else {
            c = *(const u32x4 *)(ct + at);
            s = *(const u32x4 *)(st + at);
        }
        return;
    }
    c = s = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < (ROPE == CQKV_ROPE_INTERLEAVED ? 4 : 8); ++i) {
        const int64_t at = (int64_t)axis_row(row, pair_axis(a, j0 + i)) * half + i;
        c[i / 2] |= (uint32_t)ct[at] << (16 * (i & 1));
        s[i / 2] |= (uint32_t)st[at] << (16 * (i & 1));
    }
}
// The same of any dtype, as f32 (interleaved: element e's pair is entry e & ~1).
template <int ROPE>
__device__ inline void load_angles_any(const PagedRowsArgs &a, const int (&row)[4], int e0, bool live,
                                       float (&c)[8], float (&s)[8]) {
    const int half = a.dim / 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int j = ROPE == CQKV_ROPE_HALVES ? (e0 + e >= half ? e0 + e - half : e0 + e) : (e0 + e) >> 1;
        c[e] = s[e] = 0.0f;
        if (!live || e0 + e >= a.dim || (ROPE == CQKV_ROPE_INTERLEAVED && (e & 1))) continue;
        const int64_t at = (int64_t)axis_row(row, pair_axis(a, j)) * half + j;
        c[e] = load_elem(a.cos, at, a.dtype);
        s[e] = load_elem(a.sin, at, a.dtype);
    }
}

// The 8 elements dim / 2 away from the lane's, which another lane of the row holds.
template <int LPR>
__device__ inline u32x4 partner8(const u32x4 &w, const PagedRowsArgs &a, int e0, int lane) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = (int)w[i];
        if (a.dim != 8 * LPR) {
            r[i] = (uint32_t)__shfl(v, lane + (e0 >= a.dim / 2 ? -(a.dim / 16) : a.dim / 16));
        } else if constexpr (LPR == 8) {  // lane ^ 7, then ^ 3
            const int m = __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true);
            r[i] = (uint32_t)__builtin_amdgcn_mov_dpp(m, 0x1B, 0xF, 0xF, true);
        } else if constexpr (LPR == 16) {  // row_ror:8
            r[i] = (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);
        } else {
            const auto x = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
            r[i] = lane & 16 ? x[0] : x[1];
        }
    }
    return r;
}

// x rotated: y0 = x0 c - x1 s, y1 = x0 s + x1 c of every pair, products rounded before the sum as in
// the dense rotary kernels, then rounded to the dtype (a rotated row is a row of the dtype; the codes
// of the pages are those of that row). px: the partners of a halves pair; interleaved: entries 0, 2, 4, 6
// of c and s are the pairs'.
template <int ROPE>
__device__ inline void rotate8(float (&x)[8], const float (&px)[8], const float (&c)[8],
                               const float (&s)[8], int e0, int half, int dtype) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (ROPE == CQKV_ROPE_HALVES) {
            x[e] = e0 + e >= half ? px[e] * s[e] + x[e] * c[e] : x[e] * c[e] - px[e] * s[e];
        } else if (!(e & 1)) {
            const float x0 = x[e], x1 = x[e + 1];
            x[e] = x0 * c[e] - x1 * s[e];
            x[e + 1] = x0 * s[e] + x1 * c[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (dtype == CQKV_BF16) x[e] = bf16_bits_to_f32(f32_to_bf16_bits(x[e]));
        else if (dtype == CQKV_F16) x[e] = (float)(_Float16)x[e];
    }
}

// Codes of a lane's 8 elements (8-bit: two words; 4-bit: one) and the scale: FP8 the row's f32, MX the
// block's E8M0 byte (a block is the 8-element chunks of four lanes). False where the lane needs the
// software encoders (an element that is not finite, an FP8 row of extreme magnitude) and ANY is not set.
template <int FMT, int LPR, bool ANY>
__device__ inline bool encode8(const float (&x)[8], u32x2 &cw, float &tok, uint32_t &blk) {
    float m = 0.0f, chk = 0.0f;  // chk: NaN iff an element is not finite
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        m = fmaxf(m, __builtin_fabsf(x[e]));
        chk = __builtin_fmaf(x[e], 0.0f, chk);
    }
    cw = u32x2{0u, 0u};
    if constexpr (FMT == CQKV_FMT_FP8) {
        const float amax = row_max_lanes<LPR>(m);
        const float sc = amax > 0.0f ? amax / 448.0f : 1.0f, rc = 1.0f / sc;
        tok = sc;
        // (a row of zeros too: s = 1, every quotient the zero of its element)
        const bool plain = chk == chk && amax <= 3.0e38f && (amax >= kFp8FastRowMin || amax == 0.0f);
        if (!ANY || plain) {
#pragma unroll
            for (int w = 0; w < 2; ++w)
                cw[w] = fp8_row_codes_fast(x[4 * w], x[4 * w + 1], sc, rc) |
                        (fp8_row_codes_fast(x[4 * w + 2], x[4 * w + 3], sc, rc) << 16);
        } else {
#pragma unroll
            for (int w = 0; w < 2; ++w)
                cw[w] = fp8_row_codes(x[4 * w], x[4 * w + 1], sc, rc) |
                        (fp8_row_codes(x[4 * w + 2], x[4 * w + 3], sc, rc) << 16);
        }
        return ANY || plain;
    } else {
        constexpr bool kFp4 = FMT == CQKV_FMT_MXFP4;
        blk = mx_scale_code(quad_max(m), kFp4 ? 2 : 8);
        if (blk == 0) return true;
        const float scale = e8m0_to_f32(blk), rs = 1.0f / scale;  // a power of two: exact
        // a NaN in any of the block's lanes is encoded by the software encoders, of the whole chunk
        if (!ANY || chk == chk) {
            if constexpr (kFp4) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    cw[0] |= fp4_encode_hw(x[2 * i] * rs, x[2 * i + 1] * rs) << (8 * i);
            } else {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fminf(fmaxf(x[e] * rs, -448.0f), 448.0f);
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    cw[w] = e4m3_encode2(y[4 * w], y[4 * w + 1]) | (e4m3_encode2(y[4 * w + 2], y[4 * w + 3]) << 16);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t c = kFp4 ? fp4_encode(x[e] / scale) : e4m3_encode(x[e] / scale);
                cw[kFp4 ? 0 : e / 4] |= c << (kFp4 ? 4 * e : 8 * (e % 4));
            }
        }
        return ANY || chk == chk;
    }
}

// Transposes the 8 x 8 bytes r[s] (row s, bytes 0-7) into r[j] byte s, by byte permutes: 2 x 2 blocks
// of bytes, then of byte pairs, then of words.
__device__ inline void transpose8x8(u32x2 (&r)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // word h of every row: a 4 x 4 transpose of rows 0-3 and of rows 4-7
#pragma unroll
        for (int b = 0; b < 8; b += 4) {
            const uint32_t a0 = r[b][h], a1 = r[b + 1][h], a2 = r[b + 2][h], a3 = r[b + 3][h];
            // v_perm_b32 selector bytes: 0-3 the second operand's bytes, 4-7 the first's
            const uint32_t lo01 = __builtin_amdgcn_perm(a1, a0, 0x05010400u), hi01 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);
            const uint32_t lo23 = __builtin_amdgcn_perm(a3, a2, 0x05010400u), hi23 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
            r[b][h] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
            r[b + 1][h] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
            r[b + 2][h] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
            r[b + 3][h] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // the off-diagonal 4 x 4 blocks change places
        const uint32_t t = r[j][1];
        r[j][1] = r[j + 4][0];
        r[j + 4][0] = t;
    }
}

// Transposes the 8 x 8 nibbles r[s] (row s, nibbles 0-7) into r[j] nibble s: single nibbles, pairs, then
// halves exchanged between rows 1, 2 and 4 apart.
__device__ inline void transpose8x8_nibbles(uint32_t (&r)[8]) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const int d = 1 << k;
        const uint32_t mask = k == 0 ? 0x0f0f0f0fu : k == 1 ? 0x00ff00ffu : 0x0000ffffu;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            if (s & d) continue;
            const uint32_t lo = r[s], hi = r[s + d];
            r[s] = (lo & mask) | ((hi & mask) << (4 * d));
            r[s + d] = ((lo >> (4 * d)) & mask) | (hi & ~mask);
        }
    }
}

// The plane of (page, head h) of a side; false for a hole.
__device__ inline bool page_of(const PageTable &p, int b, int tile, int &page) {
    const int at = tile >> (p.shift - 3);
    if (at >= p.max_pages) return false;
    page = ((const scalar_i32 *)p.table)[(int64_t)b * p.stride + at];
    return (uint32_t)page < (uint32_t)p.n_pages;
}

// Rotary table rows of the axes of packed row i (axes the call does not have: row 0); false when one
// lies outside the tables.
__device__ inline bool angle_rows(const PagedRowsArgs &a, int64_t i, int (&r)[4]) {
    bool in = true;
#pragma unroll
    for (int ax = 0; ax < 4; ++ax) {
        r[ax] = ax < a.axes ? ((const scalar_i32 *)a.rope_pos)[ax * a.rope_stride + i] : 0;
        in = in && (uint32_t)r[ax] < (uint32_t)a.cs_rows;
    }
    return in;
}

// Values: the 8 elements' codes of all 8 tokens are 64 (32) contiguous bytes of the tile; slots this call
// does not write keep their codes.
template <int FMT, int D>
__device__ inline void store_values(uint8_t *codes, int in_page, int c, uint32_t live, u32x2 (&cw)[8]) {
    if constexpr (FMT != CQKV_FMT_MXFP4) {
        uint8_t *dst = codes + (int64_t)in_page * 8 * D + 64 * c;
        transpose8x8(cw);
        if (live == 0xffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(u32x4 *)(dst + 16 * i) = u32x4{cw[2 * i].x, cw[2 * i].y, cw[2 * i + 1].x, cw[2 * i + 1].y};
        } else {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                if (!((live >> s) & 1)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[8 * j + s] = (uint8_t)(cw[j][s >> 2] >> (8 * (s & 3)));
            }
        }
    } else {
        uint32_t w[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) w[s] = cw[s].x;
        transpose8x8_nibbles(w);
        u32x4 *dst = (u32x4 *)(codes + (int64_t)in_page * 4 * D + 32 * c);
        u32x4 lo = {w[0], w[1], w[2], w[3]}, hi = {w[4], w[5], w[6], w[7]};
        if (live != 0xffu) {
            uint32_t keep = 0;
#pragma unroll
            for (int s = 0; s < 8; ++s) keep |= ((live >> s) & 1) ? 0u : 0xfu << (4 * s);
            const u32x4 olo = dst[0], ohi = dst[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo[i] = (lo[i] & ~keep) | (olo[i] & keep);
                hi[i] = (hi[i] & ~keep) | (ohi[i] & keep);
            }
        }
        dst[0] = lo;
        dst[1] = hi;
    }
}

// One head group of a tile.
struct RowsUnit {
    int kind, h;  // keys, values or queries; the lane's head
    bool mine;
    const void *x;
    int64_t st, sh;
};
template <int D>
__device__ inline RowsUnit rows_unit(const PagedRowsArgs &a, bool values, int u, int lane) {
    constexpr int LPR = D / 8, RPW = 64 / LPR;
    RowsUnit r;
    r.kind = values ? 1 : u < a.k_units ? 0 : 2;
    r.h = (r.kind == 2 ? u - a.k_units : u) * RPW + lane / LPR;
    r.mine = r.h < (r.kind == 2 ? a.q_heads : a.kv_heads);
    r.x = r.kind == 0 ? a.kx : r.kind == 1 ? a.vx : a.q;
    r.st = r.kind == 0 ? a.k_st : r.kind == 1 ? a.v_st : a.q_st;
    r.sh = r.kind == 0 ? a.k_sh : r.kind == 1 ? a.v_sh : a.q_sh;
    return r;
}

// Slots that a wavefront takes: values all 8 of a tile; with angles 4, whose registers leave room for 4
// wavefronts on a SIMD while the angles stay in them.
template <int ROPE, bool VALUES>
constexpr int rows_slots() { return ROPE != 0 && !VALUES ? 4 : 8; }

// Slots sb .. sb + SL - 1 of a tile, for head groups [u0, u1): those of k (first) and q, or one of v.
template <int FMT, int D, int ROPE, int VEC, bool VALUES>
__device__ inline void rows_run(const PagedRowsArgs &a, const TileAt &t, int sb, int u0, int u1, int lane) {
    constexpr int LPR = D / 8, SL = rows_slots<ROPE, VALUES>();
    constexpr bool kRope = ROPE != 0 && !VALUES;
    constexpr bool kB8 = FMT != CQKV_FMT_MXFP4;
    const int c = lane % LPR, e0 = 8 * c, half = a.dim / 2;
    const int s_lo = max(t.pos - 8 * t.tile - sb, 0), s_hi = min(t.pos + t.len - 8 * t.tile - sb, SL);
    const int64_t row0 = t.first + (int64_t)8 * t.tile + sb - t.pos;  // packed row of slot sb

    // the rows are requested before what has to be looked up for them (angles, the page)
    u32x4 ca[SL], sa[SL], raw[SL], next[SL];
    const auto load = [&](u32x4 (&w)[SL], const RowsUnit &r) {
        const uint16_t *base = (const uint16_t *)r.x + r.h * r.sh + e0;
#pragma unroll
        for (int s = 0; s < SL; ++s) {
            w[s] = u32x4{0u, 0u, 0u, 0u};
            if (r.mine && e0 < a.dim && s >= s_lo && s < s_hi) w[s] = *(const u32x4 *)(base + (row0 + s) * r.st);
        }
    };
    RowsUnit r = rows_unit<D>(a, VALUES, u0, lane);
    if constexpr (VEC) {
        load(raw, r);
        __builtin_amdgcn_sched_barrier(0);
    }
    int page = 0;
    const bool hole = (VALUES || u0 < a.k_units) && !page_of(a.pt, t.b, t.tile, page);
    // the slots written: those of the call's rows, without the ones whose angles lie outside the tables
    uint32_t live = 0;
    int rows[SL][4];
#pragma unroll
    for (int s = 0; s < SL; ++s) {
        if (s < s_lo || s >= s_hi) continue;
        if (ROPE != 0 && !angle_rows(a, row0 + s, rows[s])) continue;
        live |= 1u << s;
    }
    if (!live) return;
    const int in_page = t.tile & ((1 << (a.pt.shift - 3)) - 1);  // the tile's place in its page
    if (hole && (VALUES || u1 <= a.k_units)) return;  // (only queries are left)
    const int64_t plane0 = (int64_t)(hole ? 0 : page) * a.kv_heads;

    if constexpr (VEC) {
        if constexpr (kRope) {
#pragma unroll
            for (int s = 0; s < SL; ++s) {
                ca[s] = sa[s] = u32x4{0u, 0u, 0u, 0u};
                if (!a.mixed && e0 < a.dim && ((live >> s) & 1)) load_angles<ROPE, false>(a, rows[s], e0, ca[s], sa[s]);
            }
            if (a.mixed) {  // element by element
#pragma unroll 1
                for (int s = 0; s < SL; ++s) {
                    if (!((live >> s) & 1)) continue;
                    int at[4];
                    u32x4 cm = {0u, 0u, 0u, 0u}, sm = cm;
                    angle_rows(a, row0 + s, at);
                    if (e0 < a.dim) load_angles<ROPE, true>(a, at, e0, cm, sm);
#pragma unroll
                    for (int i = 0; i < SL; ++i)  // (selects: the slot is not a constant here)
                        if (i == s) {
                            ca[i] = cm;
                            sa[i] = sm;
                        }
                }
            }
        }
    }
#pragma unroll 1
    for (int u = u0; u < u1; ++u) {
        RowsUnit rn = r;
        if (kRope && u + 1 < u1) {
            rn = rows_unit<D>(a, VALUES, u + 1, lane);
            if constexpr (VEC) load(next, rn);
        }
        const int kind = r.kind, h = r.h;
        const bool mine = r.mine && !(hole && kind != 2);
        const PoolSide &side = VALUES ? a.v : a.k;
        const int64_t plane = plane0 + (mine && kind != 2 ? h : 0);
        uint8_t *codes = side.codes + plane * side.codes_plane, *scales = side.scales + plane * side.scales_plane;

        // slot s's elements: the queries go out, keys and values are encoded
        const auto finish = [&](int s, const float (&y)[8], auto any, bool &plain) {
            u32x2 w = {0u, 0u};
            if (!VALUES && kind == 2) {
                if (!mine) return w;
                const int64_t o = (row0 + s) * a.o_st + h * a.o_sh + e0;
                if (VEC && e0 < a.dim) {
                    u32x4 ow;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        ow[i] = VEC == 1 ? pack_bf16x2(y[2 * i], y[2 * i + 1]) : pack_f16x2(y[2 * i], y[2 * i + 1]);
                    *(u32x4 *)((uint16_t *)a.q_out + o) = ow;
                } else if (!VEC) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e0 + e < a.dim) store_elem(a.q_out, o + e, a.dtype, y[e]);
                }
                return w;
            }
            float tok = 0.0f;
            uint32_t blk = 0;
            plain = encode8<FMT, LPR, any.value>(y, w, tok, blk);
            if (!mine) return w;
            const int row = 8 * in_page + sb + s;
            if constexpr (FMT == CQKV_FMT_FP8) {
                if (c == 0) ((float *)scales)[row] = tok;
            } else if ((c & 3) == 0) {
                scales[row * (D / 32) + c / 4] = (uint8_t)blk;
            }
            if (!VALUES) {
                if constexpr (kB8) *(u32x2 *)(codes + (int64_t)row * D + e0) = w;
                else *(uint32_t *)(codes + (int64_t)row * (D / 2) + 4 * c) = w.x;
            }
            return w;
        };

        u32x2 cw[SL];
        bool plain = true;
        if constexpr (VEC) {
            const auto row = [&](u32x4 w, u32x4 &cv, u32x4 &sv, float (&y)[8]) {
                constexpr bool bf = VEC == 1;
                raw_to_f32x8(w, bf, y);
                if constexpr (kRope) {
                    float px[8], cc[8], ss[8];
                    // (converted here for every head group: as f32 across the loop they would take twice the registers)
#pragma unroll
                    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(cv[i]), "+v"(sv[i]));
                    if constexpr (ROPE == CQKV_ROPE_HALVES) {
                        raw_to_f32x8(partner8<LPR>(w, a, e0, lane), bf, px);
                        raw_to_f32x8(cv, bf, cc);
                        raw_to_f32x8(sv, bf, ss);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const uint32_t cb = (cv[e / 4] >> (8 * (e & 2))) & 0xffffu, sb = (sv[e / 4] >> (8 * (e & 2))) & 0xffffu;
                            cc[e] = bf ? bf16_bits_to_f32(cb) : f16_bits_to_f32(cb);
                            ss[e] = bf ? bf16_bits_to_f32(sb) : f16_bits_to_f32(sb);
                        }
                    }
                    rotate8<ROPE>(y, px, cc, ss, e0, half, bf ? CQKV_BF16 : CQKV_F16);
                }
            };
            uint32_t again = 0;  // slots with a lane that needs the software encoders
#pragma unroll
            for (int s = 0; s < SL; ++s) {
                cw[s] = u32x2{0u, 0u};
                if (!((live >> s) & 1)) continue;
                float y[8];
                row(raw[s], ca[s], sa[s], y);
                cw[s] = finish(s, y, std::false_type{}, plain);
                if (__any(!plain)) again |= 1u << s;
            }
            if (__builtin_expect(again != 0, 0)) {
                // (one copy of the encoders, which are long, for all slots: skipping a copy per slot costs an
                // instruction fetch each, 4 us of a single token's 9)
#pragma unroll 1
                for (int s = 0; s < SL; ++s) {
                    if (!((again >> s) & 1)) continue;
                    u32x4 w = raw[0], cv = ca[0], sv = sa[0];
#pragma unroll
                    for (int i = 1; i < SL; ++i)
                        if (i == s) {
                            w = raw[i];
                            cv = ca[i];
                            sv = sa[i];
                        }
                    float y[8];
                    row(w, cv, sv, y);
                    const u32x2 r2 = finish(s, y, std::true_type{}, plain);
#pragma unroll
                    for (int i = 0; i < SL; ++i)
                        if (i == s) cw[i] = r2;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < SL; ++s) cw[s] = u32x2{0u, 0u};
#pragma unroll 1
            for (int s = 0; s < SL; ++s) {
                if (!((live >> s) & 1)) continue;
                const int64_t row = (row0 + s) * r.st + h * r.sh;
                float y[8];
                load_any8(r.x, row, e0, mine ? a.dim : 0, a.dtype, y);
                if constexpr (kRope) {
                    int at[4];
                    float px[8] = {}, cc[8], ss[8];
                    angle_rows(a, row0 + s, at);
                    if (ROPE == CQKV_ROPE_HALVES && mine) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (e0 + e < a.dim)
                                px[e] = load_elem(r.x, row + (e0 + e >= half ? e0 + e - half : e0 + e + half), a.dtype);
                    }
                    load_angles_any<ROPE>(a, at, e0, mine, cc, ss);
                    rotate8<ROPE>(y, px, cc, ss, e0, half, a.dtype);
                }
                const u32x2 w = finish(s, y, std::true_type{}, plain);
#pragma unroll
                for (int i = 0; i < SL; ++i)  // (selects: the slot is not a constant here)
                    if (i == s) cw[i] = w;
            }
        }
        if constexpr (VALUES) {
            if (mine) store_values<FMT, D>(codes, in_page, c, live, cw);
        }
        if constexpr (!kRope) return;
        r = rn;
        if constexpr (VEC) {
#pragma unroll
            for (int s = 0; s < SL; ++s) raw[s] = next[s];
        }
    }
}

// 4 wavefronts, one run of head groups each; runs of a tile are neighbours, so the wavefronts in flight
// together read whole token rows.
// VEC: rows of whole 16-byte pieces of bf16 (1) or f16 (2); 0: any dtype and strides.
template <int FMT, int D, int ROPE, int VEC>
__global__ __launch_bounds__(256, (VEC ? 4 : 1)) void paged_append_kernel(PagedRowsArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = (int)blockIdx.x * 4 + wave;
    const int idx = at / a.units;
    TileAt t;
    if (idx >= a.tiles || !find_tile(a.pt, a.positions, idx, lane, t)) return;
    // runs: of k and q for each part of the tile's slots, then of v
    constexpr int SL = rows_slots<ROPE, false>(), PARTS = 8 / SL;
    const int kq = a.k_units + a.q_units, kq_runs = (kq + a.per - 1) / a.per, run = at - idx * a.units;
    if (run >= PARTS * kq_runs) {
        const int u = run - PARTS * kq_runs;
        rows_run<FMT, D, ROPE, VEC, true>(a, t, 0, u, u + 1, lane);
    } else {
        const int part = run / kq_runs, u0 = (run - part * kq_runs) * a.per;
        rows_run<FMT, D, ROPE, VEC, false>(a, t, SL * part, u0, min(u0 + a.per, kq), lane);
    }
}

// Read-back of one side: y = scale * value(code) in f32, rounded to the output dtype; rows of holes
// are zeros. The inverse of the append's split.
// OUT: rows of whole 16-byte pieces of bf16 (1), f16 (2) or f32 (3); 0: any dtype and strides (all in one
// kernel, their stores for every slot made a short call's instruction fetches its longest part).
template <int FMT, int D, int OUT>
__global__ __launch_bounds__(256) void paged_dequant_kernel(PagedRowsArgs a) {
    constexpr int LPR = D / 8, RPW = 64 / LPR;
    constexpr bool kB8 = FMT != CQKV_FMT_MXFP4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = (int)blockIdx.x * 4 + wave;
    const int idx = at / a.units;
    TileAt t;
    if (idx >= a.tiles || !find_tile(a.pt, a.positions, idx, lane, t)) return;
    const int c = lane % LPR, e0 = 8 * c, h = (at - idx * a.units) * RPW + lane / LPR;
    if (h >= a.kv_heads || e0 >= a.dim) return;
    const int s_lo = max(t.pos - 8 * t.tile, 0), s_hi = min(t.pos + t.len - 8 * t.tile, 8);
    const int64_t row0 = t.first + (int64_t)8 * t.tile - t.pos;
    int page = 0;
    const bool hole = !page_of(a.pt, t.b, t.tile, page);
    const int64_t plane = (int64_t)(hole ? 0 : page) * a.kv_heads + h;
    const int in_page = t.tile & ((1 << (a.pt.shift - 3)) - 1);
    const uint8_t *codes = a.k.codes + plane * a.k.codes_plane;
    const uint8_t *scales = a.k.scales + plane * a.k.scales_plane;
    u32x2 cw[8];
    uint32_t sw[8];  // the rows' scales as they are in the pool (a conversion here would wait for each load)
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        cw[s] = u32x2{0u, 0u};
        sw[s] = 0u;
    }
    if (!hole) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            if (s < s_lo || s >= s_hi) continue;
            const int row = 8 * in_page + s;
            if constexpr (FMT == CQKV_FMT_FP8) sw[s] = ((const uint32_t *)scales)[row];
            else sw[s] = scales[(int64_t)row * (D / 32) + c / 4];
            if (!a.side_is_value) {
                if constexpr (kB8) cw[s] = *(const u32x2 *)(codes + (int64_t)row * D + e0);
                else cw[s].x = *(const uint32_t *)(codes + (int64_t)row * (D / 2) + 4 * c);
            }
        }
        if (a.side_is_value) {
            if constexpr (kB8) {
                const u32x4 *src = (const u32x4 *)(codes + (int64_t)in_page * 8 * D + 64 * c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x4 w = src[i];
                    cw[2 * i] = u32x2{w.x, w.y};
                    cw[2 * i + 1] = u32x2{w.z, w.w};
                }
                transpose8x8(cw);
            } else {
                const u32x4 *src = (const u32x4 *)(codes + (int64_t)in_page * 4 * D + 32 * c);
                const u32x4 lo = src[0], hi = src[1];
                uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                transpose8x8_nibbles(w);
#pragma unroll
                for (int s = 0; s < 8; ++s) cw[s].x = w[s];
            }
        }
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        if (s < s_lo || s >= s_hi) continue;
        const float sc = FMT == CQKV_FMT_FP8 ? __uint_as_float(sw[s]) : sw[s] == 0 ? 0.0f : __uint_as_float(sw[s] << 23);
        float y[8];
        if constexpr (kB8) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const f32x2 p0 = __builtin_amdgcn_cvt_pk_f32_fp8(cw[s][w], false);
                const f32x2 p1 = __builtin_amdgcn_cvt_pk_f32_fp8(cw[s][w], true);
                y[4 * w] = p0.x * sc;
                y[4 * w + 1] = p0.y * sc;
                y[4 * w + 2] = p1.x * sc;
                y[4 * w + 3] = p1.y * sc;
            }
        } else {
            const uint32_t w = cw[s].x;
            const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
            const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
            const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
            const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
            y[0] = p0.x * sc; y[1] = p0.y * sc; y[2] = p1.x * sc; y[3] = p1.y * sc;
            y[4] = p2.x * sc; y[5] = p2.y * sc; y[6] = p3.x * sc; y[7] = p3.y * sc;
        }
        const int64_t o = (row0 + s) * a.out_st + h * a.out_sh + e0;
        // (nontemporal: 48769 rows of two FP8 sides 62 us, 66 with cached stores)
        if constexpr (OUT == 3) {
            __builtin_nontemporal_store(f32x4{y[0], y[1], y[2], y[3]}, (f32x4 *)((float *)a.out + o));
            __builtin_nontemporal_store(f32x4{y[4], y[5], y[6], y[7]}, (f32x4 *)((float *)a.out + o + 4));
        } else if constexpr (OUT != 0) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = OUT == 1 ? pack_bf16x2(y[2 * i], y[2 * i + 1]) : pack_f16x2(y[2 * i], y[2 * i + 1]);
            __builtin_nontemporal_store(w, (u32x4 *)((uint16_t *)a.out + o));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e0 + e < a.dim) store_elem(a.out, o + e, a.out_dtype, y[e]);
        }
    }
}

template <int FMT, int D, int ROPE>
inline void launch_append(dim3 grid, hipStream_t st, const PagedRowsArgs &a) {
    if (!a.vec) hipLaunchKernelGGL((paged_append_kernel<FMT, D, ROPE, 0>), grid, dim3(256), 0, st, a);
    else if (a.dtype == CQKV_BF16) hipLaunchKernelGGL((paged_append_kernel<FMT, D, ROPE, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<FMT, D, ROPE, 2>), grid, dim3(256), 0, st, a);
}
template <int FMT, int D>
inline void launch_append_rope(int rope, dim3 grid, hipStream_t st, const PagedRowsArgs &a) {
    if (rope == CQKV_ROPE_HALVES) launch_append<FMT, D, CQKV_ROPE_HALVES>(grid, st, a);
    else if (rope == CQKV_ROPE_INTERLEAVED) launch_append<FMT, D, CQKV_ROPE_INTERLEAVED>(grid, st, a);
    else launch_append<FMT, D, 0>(grid, st, a);
}
template <int FMT>
inline void launch_append_dim(int dk, int rope, dim3 grid, hipStream_t st, const PagedRowsArgs &a) {
    if (dk == 64) launch_append_rope<FMT, 64>(rope, grid, st, a);
    else if (dk == 128) launch_append_rope<FMT, 128>(rope, grid, st, a);
    else launch_append_rope<FMT, 256>(rope, grid, st, a);
}
template <int FMT, int D>
inline void launch_dequant_out(dim3 grid, hipStream_t st, const PagedRowsArgs &a) {
    if (!a.out_vec) hipLaunchKernelGGL((paged_dequant_kernel<FMT, D, 0>), grid, dim3(256), 0, st, a);
    else if (a.out_dtype == CQKV_BF16) hipLaunchKernelGGL((paged_dequant_kernel<FMT, D, 1>), grid, dim3(256), 0, st, a);
    else if (a.out_dtype == CQKV_F16) hipLaunchKernelGGL((paged_dequant_kernel<FMT, D, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_dequant_kernel<FMT, D, 3>), grid, dim3(256), 0, st, a);
}
template <int FMT>
inline void launch_dequant(int dk, dim3 grid, hipStream_t st, const PagedRowsArgs &a) {
    if (dk == 64) launch_dequant_out<FMT, 64>(grid, st, a);
    else if (dk == 128) launch_dequant_out<FMT, 128>(grid, st, a);
    else launch_dequant_out<FMT, 256>(grid, st, a);
}

// Per-format launchers, defined in paged_inst.hip.
#define CQKV_PAGED_ROWS_LAUNCHERS(F)                                                              \
    void paged_append_launch_##F(int dk, int rope, dim3 grid, hipStream_t st, const PagedRowsArgs &a); \
    void paged_dequant_launch_##F(int dk, dim3 grid, hipStream_t st, const PagedRowsArgs &a);
CQKV_PAGED_ROWS_LAUNCHERS(2)
CQKV_PAGED_ROWS_LAUNCHERS(4)
CQKV_PAGED_ROWS_LAUNCHERS(5)

}  // namespace cqkv
