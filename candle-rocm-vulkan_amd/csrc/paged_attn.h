// Attention over a page pool, few columns per kv head (single tokens, drafted tokens): split-K
// flash-decode in one pass over the pages (included by paged_inst.hip, one object per format, and by
// paged_attn.hip for the arguments).
//
// Mathematics: o_i = sum_j p_ij v_j / sum_j p_ij over the keys j that query i sees, with
// p_ij = 2^(x_ij - m_i), x = scale log2(e) q k and m_i the running maximum. Keys and values enter the
// products as exact bf16 operands: E4M3 codes as they are, MX codes times their power of two. The f32
// scale of an FP8 row multiplies the score after the product (keys) or the weight before it (values),
// so quantization is the pool's only rounding of K and V.
//
// A workgroup takes one piece of a (sequence, kv head) plane: a range of its 32-key tiles, its wavefronts
// taking tiles in turn. A tile lies in one page, so a page change is a new set of buffer resources in
// scalar registers. Operand layouts are those of the dense decode kernel: lane (n, g) of
// v_mfma_f32_16x16x32_bf16 holds column n = a (query, head of the group) pair, keys 8 g .. 8 g + 7 of a
// tile. More than 16 columns (drafted tokens) are blocks of 16 in wavefronts of their own, 2 or 4 on the
// same tile, whose bytes come from HBM once and from L1 or L2 after that: a wavefront then keeps the
// registers of one block, and two fit a SIMD.
//
// Bound by HBM for single tokens over 8-bit codes (64 sequences of up to 8K keys, FP8, 32 / 8 heads, D = 128:
// 119 us, 5.7 TB/s), by the decoding VALU work for MXFP4 (4 sequences of up to 128K keys, 64 / 8 heads: 85 us,
// 5.4 TB/s), by the latency of a tile for drafted tokens (16 sequences of 5: 40 us, 3.1 TB/s), by the chain
// length -> page -> tile -> merge for a short sequence (7.6 us at 500 keys, D = 64).
#pragma once

#include <type_traits>

#include "paged.h"
#include "prefill_split.h"

namespace cqkv {

struct PagedAttnArgs {
    PageTable pt;
    PoolSide k, v;
    const void *q;
    void *out;
    int64_t q_st, q_sh, o_st, o_sh;  // element strides: token, head
    const int32_t *kv_lens;
    int32_t max_q, max_kv;
    int32_t kv_heads, q_heads, group, dim, q_vec, o_vec;
    uint32_t group_m;
    int32_t wl, wr;
    float scale_log2, cap2;  // cap2: softcap * log2(e), 0: off
    const float *alibi;
    int32_t alibi_bs;
    int32_t parts;           // pieces of the decode kernel's work (see piece_tiles); 0: one per plane
    int32_t slot_cols;       // columns of a slot of its partial outputs
    // sequences with more than chunk_from columns per kv head (if the call may have any: chunk_blocks
    // bounds their column blocks) are the chunk kernel's: splits of chunk_tps of its key tiles
    int32_t chunk_from, chunk_blocks, chunk_splits, chunk_tps, chunk_bk;
    // Partial outputs, normalised, and their log2-sum-exp: (2 parts, slot_cols) columns of the decode
    // kernel's pieces, (splits, total * q_heads) rows of the chunk kernel's splits
    float *part_o, *part_lse, *chunk_o, *chunk_lse;
};

// A sequence of the call: packed rows, keys, and the 32-key tiles that its queries see.
struct PagedSeq {
    int first, lq, lk, t0, t1;
};
__device__ inline PagedSeq paged_seq_of(const PagedAttnArgs &a, int cu0, int cu1, int len) {
    PagedSeq s;
    s.first = min(max(cu0, 0), a.pt.total);
    s.lq = min(max(cu1, s.first), a.pt.total) - s.first;
    const int reach = min(a.max_kv, a.pt.max_pages << a.pt.shift);
    s.lk = min(max(len, 0), reach);
    // queries past max_q are not computed: the sequence keeps its alignment, so they are its last ones
    int lo, hi, lo1;
    pf_key_range(0, s.lq, s.lk, a.wl, a.wr, lo, hi);
    pf_key_range(max(min(s.lq, a.max_q) - 1, 0), s.lq, s.lk, a.wl, a.wr, lo1, hi);
    s.t0 = lo / 32;
    s.t1 = (hi + 31) / 32;
    return s;
}
__device__ inline PagedSeq paged_seq(const PagedAttnArgs &a, int b) {  // b uniform
    const scalar_i32 *cu = (const scalar_i32 *)a.pt.cu;
    return paged_seq_of(a, cu[b], cu[b + 1], ((const scalar_i32 *)a.kv_lens)[b]);
}
__device__ inline PagedSeq paged_seq_lane(const PagedAttnArgs &a, int b) {  // a sequence per lane
    if (b >= a.pt.batch) return PagedSeq{0, 0, 0, 0, 0};
    return paged_seq_of(a, a.pt.cu[b], a.pt.cu[b + 1], a.kv_lens[b]);
}
// Splits of a sequence that the chunk kernel takes: at least one (its rows are written by someone), at
// most those that the workspace holds (the last one takes what lengths beyond the call's maxima leave).
__device__ inline int chunk_splits(const PagedAttnArgs &a, const PagedSeq &s) {
    const int per = a.chunk_bk / 32, tiles = (s.t1 + per - 1) / per - s.t0 / per;
    return min(max((tiles + a.chunk_tps - 1) / a.chunk_tps, 1), a.chunk_splits);
}
__device__ inline bool chunk_takes(const PagedAttnArgs &a, const PagedSeq &s) {
    return a.chunk_blocks > 0 && (int64_t)min(s.lq, a.max_q) * a.group > a.chunk_from;
}

// ---- pieces ----
// The launch is made without knowing the lengths, so the workgroups cut the call's planes themselves: into
// equal pieces of at most U tiles, U = all planes' tiles / parts. Lengths of any mixture then fill the chip
// (workgroups start as others end), and a captured graph whose lengths grow keeps its balance. At most
// parts + planes pieces come of it, and at most 2 parts of them belong to planes that are cut (ceil(n / U)
// <= 2 n / U): those write to their slots, which the combine kernel merges, the others to the output.
struct SeqWork {
    int n, pieces;  // tiles of a plane, its pieces (0: nothing for the decode kernel)
};
__device__ inline int seq_tiles(const PagedAttnArgs &a, const PagedSeq &s) {  // -1: not the decode kernel's
    return s.lq > 0 && !chunk_takes(a, s) ? max(s.t1 - s.t0, 0) : -1;
}
// Inclusive sum over the lanes (of a count, or of two in the halves of a word).
__device__ inline uint64_t wave_scan2(uint64_t v, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, m), hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), m);
        if (lane >= m) v += (uint64_t)hi << 32 | lo;
    }
    return v;
}
__device__ inline uint64_t readlane64(uint64_t v, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
// U: at least kPieceTiles tiles, so that a piece's start and merge (about 3 us) stay small beside it.
constexpr int kPieceTiles = 32;
__device__ inline uint32_t piece_tiles(const PagedAttnArgs &a, uint64_t lane_tiles, int lane) {
    const uint64_t total = readlane64(wave_scan2(lane_tiles, lane), 63);
    const uint64_t u = (total * (uint32_t)a.kv_heads + (uint32_t)a.parts - 1) / (uint32_t)a.parts;
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)min(max(u, (uint64_t)kPieceTiles), (uint64_t)0x40000000u));
}
__device__ inline SeqWork seq_work(const PagedAttnArgs &a, const PagedSeq &s, uint32_t u) {
    const int n = seq_tiles(a, s);
    return SeqWork{n, n < 0 ? 0 : max((int)(((uint32_t)n + u - 1) / u), 1)};
}
// Pieces of a sequence's planes in all, and (high half) those that go to slots.
__device__ inline uint64_t seq_pieces(const PagedAttnArgs &a, const SeqWork &w) {
    const uint32_t p = (uint32_t)(w.pieces * a.kv_heads);
    return (uint64_t)(w.pieces > 1 ? p : 0u) << 32 | p;
}

// Sequence of piece `idx` of the call (-1: past the last) and the pieces in front of that sequence. A lane
// sums a run of sequences, so the search costs two scans and a run's loads, which are independent, however
// many sequences there are.
__device__ inline int piece_sequence(const PagedAttnArgs &a, uint32_t idx, int lane, uint32_t &u, uint64_t &first) {
    const int run = (a.pt.batch + 63) >> 6;
    uint64_t mine = 0;
#pragma unroll 4
    for (int i = 0; i < run; ++i) mine += (uint32_t)max(seq_tiles(a, paged_seq_lane(a, lane * run + i)), 0);
    u = piece_tiles(a, mine, lane);
    mine = 0;
#pragma unroll 4
    for (int i = 0; i < run; ++i) mine += seq_pieces(a, seq_work(a, paged_seq_lane(a, lane * run + i), u));
    uint64_t sum = wave_scan2(mine, lane), past = __ballot((uint32_t)sum > idx);
    if (!past) return -1;
    const int l = __builtin_ctzll(past);
    first = readlane64(sum - mine, l);
    if (run == 1) return l;
    for (int base = l * run; base < (l + 1) * run; base += 64) {  // the lane's run, a sequence per lane
        const int b = base + lane;
        mine = b < (l + 1) * run ? seq_pieces(a, seq_work(a, paged_seq_lane(a, b), u)) : 0;
        sum = first + wave_scan2(mine, lane);
        past = __ballot((uint32_t)sum > idx);
        if (past) {
            const int k = __builtin_ctzll(past);
            first = readlane64(sum - mine, k);
            return base + k;
        }
        first = readlane64(sum, 63);
    }
    return -1;
}

// Head dim held in k-slot 0 of MFMA chunk j by lane group g (the same for K and Q operands).
template <int FMT, int D>
__device__ inline int paged_qdim(int j, int g) {
    return FMT == CQKV_FMT_MXFP4 ? (D / 4) * g + 8 * j : 64 * (j >> 1) + 16 * g + 8 * (j & 1);
}

// A 32-key tile in registers: code words of the two 16-key sub-tiles (lane (n, g): key
// 8 (n / 4) + 4 s + n % 4), value code words of head dims 32 u + 2 n, + 1 of keys 8 g .. 8 g + 7, and
// the scales of those 8 keys (FP8: f32; MX: their value block bytes, D / 32 a key) and of the lane's
// two key rows (MX: the block bytes of its head dims).
template <int FMT, int D>
struct PagedTile {
    static constexpr bool B8 = FMT != CQKV_FMT_MXFP4;
    static constexpr int VSW = FMT == CQKV_FMT_FP8 ? 8 : D / 16;  // words of 8 keys' value scales
    uint32_t k[2][B8 ? D / 16 : D / 32];
    uint32_t v[D / 32][B8 ? 4 : 2];
    uint32_t ks[FMT == CQKV_FMT_FP8 ? 8 : 2], ks2[2];
    uint32_t vs[VSW];
};

struct PageRsrc {
    rsrc_t k, ks, v, vs;
};
// Resources of page id `page`, kv head hk; a hole or a dead tile gets empty ones: loads return zeros.
__device__ inline PageRsrc page_rsrc(const PagedAttnArgs &a, int page, int hk, bool ok) {
    const int64_t plane = ok ? (int64_t)page * a.kv_heads + hk : 0;
    const uint32_t kb = ok ? a.k.codes_plane : 0u, sb = ok ? a.k.scales_plane : 0u;
    PageRsrc r;
    r.k = make_rsrc(a.k.codes + plane * a.k.codes_plane, kb);
    r.ks = make_rsrc(a.k.scales + plane * a.k.scales_plane, sb);
    r.v = make_rsrc(a.v.codes + plane * a.v.codes_plane, kb);
    r.vs = make_rsrc(a.v.scales + plane * a.v.scales_plane, sb);
    return r;
}

// Code loads: read once per call (nontemporal), or by other wavefronts on the same tile too (ONCE false:
// they then come from L2; nontemporal lines come from HBM again). 16 sequences of 5 drafted tokens, FP8: 47 us,
// 56 with ONCE; single tokens of 64 sequences: 128 with ONCE, 138 without or with a branch between the two.
template <bool ONCE>
__device__ inline u32x4 code128(rsrc_t r, uint32_t off) { return ONCE ? ld128_stream(r, off) : ld128(r, off); }
template <bool ONCE>
__device__ inline u32x2 code64(rsrc_t r, uint32_t off) { return ONCE ? ld64_stream(r, off) : ld64(r, off); }

// t0: the tile's first row in its page.
template <int FMT, int D, bool ONCE>
__device__ inline void paged_load(PagedTile<FMT, D> &r, const PageRsrc &p, uint32_t t0, int lane) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const uint32_t key = t0 + 8 * (n >> 2) + 4 * s + (n & 3);
        if constexpr (PagedTile<FMT, D>::B8) {
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const u32x4 w = code128<ONCE>(p.k, key * D + 16 * g + 64 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) r.k[s][4 * i + e] = w[e];
            }
        } else if constexpr (D == 64) {
            const u32x2 w = code64<ONCE>(p.k, key * 32 + 8 * g);
            r.k[s][0] = w.x;
            r.k[s][1] = w.y;
        } else {
#pragma unroll
            for (int i = 0; i < D / 128; ++i) {
                const u32x4 w = code128<ONCE>(p.k, key * (D / 2) + (D / 8) * g + 16 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) r.k[s][4 * i + e] = w[e];
            }
        }
        if constexpr (FMT == CQKV_FMT_MXFP8) {  // all the key's block bytes
            if constexpr (D == 256) {
                const u32x2 w = ld64(p.ks, key * 8);
                r.ks[s] = w.x;
                r.ks2[s] = w.y;
            } else if constexpr (D == 128) {
                r.ks[s] = ld32(p.ks, key * 4);
            } else {
                r.ks[s] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(p.ks, key * 2, 0, 0);
            }
        } else if constexpr (FMT == CQKV_FMT_MXFP4) {  // those of head dims (D / 4) g ..
            if constexpr (D == 256)
                r.ks[s] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(p.ks, key * 8 + 2 * g, 0, 0);
            else
                r.ks[s] = __builtin_amdgcn_raw_buffer_load_b8(p.ks, key * (D / 32) + (D == 128 ? g : g >> 1), 0, 0);
        }
    }
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
        const uint32_t at = (t0 / 8 + g) * D + 32 * u + 2 * n;
        if constexpr (PagedTile<FMT, D>::B8) {
            const u32x4 w = code128<ONCE>(p.v, at * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) r.v[u][e] = w[e];
        } else {
            const u32x2 w = code64<ONCE>(p.v, at * 4);
            r.v[u][0] = w.x;
            r.v[u][1] = w.y;
        }
    }
    const uint32_t kb = t0 + 8 * g;
    if constexpr (FMT == CQKV_FMT_FP8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4 w = ld128(p.ks, kb * 4 + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) r.ks[4 * i + e] = w[e];
        }
    }
#pragma unroll
    for (int i = 0; i < PagedTile<FMT, D>::VSW / 4; ++i) {
        const u32x4 w = ld128(p.vs, kb * (PagedTile<FMT, D>::VSW / 2) + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) r.vs[4 * i + e] = w[e];
    }
}

__device__ inline float e8m0_or_zero(uint32_t code) {  // code 0 marks an all-zero block
    return code == 0 ? 0.0f : __uint_as_float(code << 23);
}
__device__ inline bf16x8 fp4x8_bf16x8(uint32_t w, float scale) {
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return __builtin_bit_cast(bf16x8, r);
}

// Key operand of chunk j, sub-tile s: exact.
template <int FMT, int D>
__device__ inline bf16x8 paged_key(const PagedTile<FMT, D> &t, int s, int j, int g) {
    if constexpr (FMT == CQKV_FMT_FP8) {
        return fp8x8_to_bf16x8(t.k[s][2 * j], t.k[s][2 * j + 1]);
    } else if constexpr (FMT == CQKV_FMT_MXFP8) {
        const int bi = 2 * (j >> 1) + (g >> 1);
        const uint32_t w = bi < 4 ? t.ks[s] : t.ks2[s];
        return fp8x8_pow2_bf16x8(t.k[s][2 * j], t.k[s][2 * j + 1], e8m0_or_zero((w >> (8 * (bi & 3))) & 0xffu));
    } else {
        const uint32_t b = D == 256 ? (t.ks[s] >> (8 * (j >> 2))) & 0xffu : t.ks[s];
        return fp4x8_bf16x8(t.k[s][j], b ? __uint_as_float(b << 23) : 1.0f);
    }
}
// Value operand of head dims 32 u + 2 n + h, keys 8 g .. + 7: the bare codes, exact.
template <int FMT, int D>
__device__ inline bf16x8 paged_value(const PagedTile<FMT, D> &t, int u, int h) {
    if constexpr (FMT == CQKV_FMT_MXFP4) return fp4x8_bf16x8(t.v[u][h], 1.0f);
    else return fp8x8_to_bf16x8(t.v[u][2 * h], t.v[u][2 * h + 1]);
}
// Value block bytes (block u) of keys 2 i, 2 i + 1 of the lane's 8, in bytes 0 and 2.
template <int D>
__device__ inline uint32_t paged_block_pair(const uint32_t *vs, int i, int u) {
    if constexpr (D == 64) {
        const uint32_t sel = (uint32_t)u | 0x0c00u | ((uint32_t)(2 + u) << 16) | 0x0c000000u;
        return __builtin_amdgcn_perm(vs[i], vs[i], sel);
    } else {
        constexpr int W = D / 128;  // words a key
        const uint32_t sel = (uint32_t)(u & 3) | 0x0c00u | ((uint32_t)(4 + (u & 3)) << 16) | 0x0c000000u;
        return __builtin_amdgcn_perm(vs[W * (2 * i + 1) + (u >> 2)], vs[W * 2 * i + (u >> 2)], sel);
    }
}

// The weights of 8 keys as P operands: hi the bf16 part (truncated, so the rest is not negative), lo the
// rest (LO). FP8: the weight times the key's value scale.
template <bool LO>
__device__ inline void paged_split(const float (&p)[8], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (LO) {
            const uint32_t a = __float_as_uint(p[2 * i]), b = __float_as_uint(p[2 * i + 1]);
            hi[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            lo[i] = pack_bf16x2(p[2 * i] - __uint_as_float(a & 0xffff0000u), p[2 * i + 1] - __uint_as_float(b & 0xffff0000u));
        } else {
            hi[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
        }
    }
}
// bf16 weights times 2^(c - 127) of the keys' block bytes c: the codes are added to the exponent
// fields (a packed multiply-add and a clamp per pair), the bits of the exact product wherever it is a
// normal bf16 number; below that range it is zero or below 2^-126. A weight of zero gives at most
// 2^(c - 254): nothing beside another weight of its block, whose factor is 2^(c - 127).
__device__ inline uint32_t paged_scale_pair(uint32_t p, uint32_t c) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    const u16x2 pb = __builtin_bit_cast(u16x2, p) - u16x2{0x3f80, 0x3f80};
    uint32_t r;  // c * 128 + pb per half, one v_pk_mad_u16 (the compiler emits a shift and an add)
    asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(r) : "v"(c), "v"(0x00800080u), "v"(pb));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(i16x2, r), i16x2{0, 0}));
}

// The column of a lane: its keys [lo, hi).
struct PagedCol {
    int lo, hi, qpos;
    float slope2;
};

// F16: f16 queries and outputs. The queries enter as bf16 hi + lo parts (exact), the weights too.
template <int FMT, int D, bool F16>
__device__ inline void paged_compute(PagedTile<FMT, D> &t, const PagedAttnArgs &a, int key0, int lk,
                                     bool full, const bf16x8 *qhi, const bf16x8 *qlo, const PagedCol &col,
                                     int lane, float &m_run, float &l_run, f32x4 *acc) {
    constexpr int NCH = D / 32;
    constexpr bool kFp8 = FMT == CQKV_FMT_FP8;
    constexpr bool LO = F16 || FMT != CQKV_FMT_MXFP4;
    const int g = lane >> 4;
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const bf16x8 k0 = paged_key<FMT, D>(t, 0, j, g), k1 = paged_key<FMT, D>(t, 1, j, g);
        s0 = mfma16x16x32(k0, qhi[j], s0);
        s1 = mfma16x16x32(k1, qhi[j], s1);
        if constexpr (F16) {
            s0 = mfma16x16x32(k0, qlo[j], s0);
            s1 = mfma16x16x32(k1, qlo[j], s1);
        }
    }
    const int kb = key0 + 8 * g;  // the lane's first key
    const int nv = min(max(lk - kb, 0), 8);
    if (key0 + 32 > lk) {
        // the tile that holds the end of the keys: codes and scales past it may be any bytes
#pragma unroll
        for (int u = 0; u < NCH; ++u) {
            if constexpr (PagedTile<FMT, D>::B8) {
                const uint64_t keep = nv == 0 ? 0ull : (~0ull >> (64 - 8 * nv));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    t.v[u][2 * h] &= (uint32_t)keep;
                    t.v[u][2 * h + 1] &= (uint32_t)(keep >> 32);
                }
            } else {
                const uint32_t keep = nv == 0 ? 0u : (~0u >> (32 - 4 * nv));
                t.v[u][0] &= keep;
                t.v[u][1] &= keep;
            }
        }
        if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= nv) t.vs[e] = 0u;
        } else {
#pragma unroll
            for (int w = 0; w < PagedTile<FMT, D>::VSW; ++w) {
                constexpr int kBytes = D / 32;  // a key
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    if ((4 * w + y) / kBytes >= nv) t.vs[w] &= ~(0xffu << (8 * y));
            }
        }
    }
    // A value that is not finite, in a tile where some column does not see some key: its key must not
    // reach that column (0 times it is NaN)
    bool bad = false;
    if (!full && FMT != CQKV_FMT_MXFP4) {
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < NCH; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w) m |= (t.v[u][w] & 0x7f7f7f7fu) + 0x01010101u;  // NaN: 0x7f
        bad = (m & 0x80808080u) != 0;
        if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) bad |= (t.vs[e] & 0x7f800000u) == 0x7f800000u;
        }
        bad = __any(bad);
    }
    float x[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= kFp8 ? __uint_as_float(t.ks[e]) * a.scale_log2 : a.scale_log2;
    if (a.cap2 > 0.0f || a.alibi) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fa_logit2(x[e], a.cap2, col.slope2, col.qpos - (kb + e));
    }
    uint32_t see = 0xffu;
    if (!full) {
        see = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = kb + e >= col.lo && kb + e < col.hi;
            see |= in ? 1u << e : 0u;
            if (!in) x[e] = -__builtin_inff();
        }
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
    mx = group16_max(mx);
    const float m_new = fmaxf(m_run, mx);
    const bool none = m_new == -__builtin_inff();
    const float alpha = none ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
    const float m_sub = none ? 0.0f : m_new;  // scores of -inf then have weight 0, NaN stays NaN
    float p[8], psum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(x[e] - m_sub);
        psum += p[e];
    }
    l_run = l_run * alpha + psum;
    m_run = m_new;
    if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int i = 0; i < 2 * NCH; ++i) acc[i] *= alpha;
    }
    if constexpr (kFp8) {
        // (a key out of sight keeps weight zero whatever its scale)
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = (see >> e) & 1u ? p[e] * __uint_as_float(t.vs[e]) : 0.0f;
    }
    uint32_t hi[4], lo[4];
    paged_split<LO>(p, hi, lo);
    // MX: keys out of sight take block byte 0, so that whatever their scale their operand is zero
    const auto product = [&](const PagedTile<FMT, D> &tv, f32x4 *o, auto masked) {
        uint32_t keep[4];
        if constexpr (!kFp8 && masked.value) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                keep[i] = ((see >> (2 * i)) & 1u ? 0xffffu : 0u) | ((see >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int u = 0; u < NCH; ++u) {
            u32x4 ph, pl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kFp8) {
                    ph[i] = hi[i];
                    if constexpr (LO) pl[i] = lo[i];
                } else {
                    uint32_t c = paged_block_pair<D>(tv.vs, i, u);
                    if constexpr (masked.value) c &= keep[i];
                    ph[i] = paged_scale_pair(hi[i], c);
                    if constexpr (LO) pl[i] = paged_scale_pair(lo[i], c);
                }
            }
            const bf16x8 v0 = paged_value<FMT, D>(tv, u, 0), v1 = paged_value<FMT, D>(tv, u, 1);
            const bf16x8 pb = __builtin_bit_cast(bf16x8, ph);
            o[2 * u] = mfma16x16x32(v0, pb, o[2 * u]);
            o[2 * u + 1] = mfma16x16x32(v1, pb, o[2 * u + 1]);
            if constexpr (LO) {
                const bf16x8 pc = __builtin_bit_cast(bf16x8, pl);
                o[2 * u] = mfma16x16x32(v0, pc, o[2 * u]);
                o[2 * u + 1] = mfma16x16x32(v1, pc, o[2 * u + 1]);
            }
        }
    };
    if (kFp8 ? !bad : full) {
        product(t, acc, std::false_type{});
    } else if (!bad) {
        product(t, acc, std::true_type{});
    } else {
        // column by column, each with the codes of the keys it does not see set to zero
#pragma unroll 1
        for (int c = 0; c < 16; ++c) {
            const uint32_t sc = (uint32_t)__shfl((int)see, 16 * g + c);
            PagedTile<FMT, D> tc = t;
            uint32_t w0 = 0, w1 = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w0 |= (sc >> e) & 1u ? 0xffu << (8 * e) : 0u;
                w1 |= (sc >> (4 + e)) & 1u ? 0xffu << (8 * e) : 0u;
            }
            if constexpr (PagedTile<FMT, D>::B8) {
#pragma unroll
                for (int u = 0; u < NCH; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        tc.v[u][2 * h] &= w0;
                        tc.v[u][2 * h + 1] &= w1;
                    }
            }
            f32x4 o[2 * NCH];
#pragma unroll
            for (int i = 0; i < 2 * NCH; ++i) o[i] = acc[i];
            product(tc, o, std::true_type{});
#pragma unroll
            for (int i = 0; i < 2 * NCH; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][r] = (lane & 15) == c ? o[i][r] : acc[i][r];
        }
    }
}

// 8 query elements d0 .. d0 + 7 of a row (16-bit, zeros past dim), raw
__device__ inline u32x4 paged_q8(const uint16_t *row, int d0, int dim, bool vec) {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (vec) {
        if (d0 < dim) w = *(const u32x4 *)(row + d0);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (d0 + e < dim) w[e / 2] |= (uint32_t)row[d0 + e] << (16 * (e & 1));
    }
    return w;
}

// Tiles in flight per wavefront: as many as leave two wavefronts to a SIMD (MXFP4, D = 128, 4 sequences of up to
// 128K keys: 100 us with two, 88 with three; one short sequence at D = 64: 14 with two, 11.7 with four).
constexpr int paged_sets(int fmt, int d) { return d == 64 ? 4 : d == 128 && fmt == CQKV_FMT_MXFP4 ? 3 : 2; }

template <int FMT, int D, bool F16, bool ONCE>
__global__ __launch_bounds__(256, (D < 256 ? 2 : 1)) void paged_attn_kernel(PagedAttnArgs a) {
    constexpr int NCH = D / 32, WAVES = 4, NS = paged_sets(FMT, D);
    __shared__ __attribute__((aligned(16))) float sm_o[WAVES][16][D + 4];
    __shared__ float sm_m[WAVES][16], sm_l[WAVES][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;

    // the piece: sequence, kv head (fastest, so that with 8 kv heads an XCD takes one head of every
    // sequence: the same mix of lengths everywhere), and its slot
    int b = -1, rest = 0, slot = -1;
    uint32_t u = 0;
    if (a.parts == 0) {
        b = (int)blockIdx.x / a.kv_heads;
        rest = (int)blockIdx.x % a.kv_heads;
    } else {
        uint64_t first = 0;
        b = piece_sequence(a, blockIdx.x, lane, u, first);
        if (b >= 0) {
            rest = (int)(blockIdx.x - (uint32_t)first);
            slot = (int)(first >> 32) + rest;
        }
        if (b < 0) return;
    }
    // (uniform, which the compiler does not see through the sums over lanes: the pages' resources must be
    // scalars, or every load becomes a loop over the lanes' values)
    b = __builtin_amdgcn_readfirstlane(b);
    rest = __builtin_amdgcn_readfirstlane(rest);
    slot = __builtin_amdgcn_readfirstlane(slot);
    const PagedSeq sq = paged_seq(a, b);
    int hk = rest, tb = sq.t0, te = sq.t1;
    if (a.parts == 0) {
        if (seq_tiles(a, sq) < 0) return;
    } else {
        const SeqWork w = seq_work(a, sq, u);
        const int piece = rest / a.kv_heads, len = (int)((uint32_t)w.n / (uint32_t)w.pieces), more = w.n - len * w.pieces;
        hk = rest - piece * a.kv_heads;
        tb = sq.t0 + piece * len + min(piece, more);
        te = tb + len + (piece < more ? 1 : 0);
        if (w.pieces < 2) slot = -1;
    }

    // column blocks of 16 in 1, 2 or 4 wavefronts, which take the same tiles
    const int ncols = min(sq.lq, a.max_q) * a.group;
    const int cshift = ncols <= 16 ? 0 : ncols <= 32 ? 1 : 2, step = WAVES >> cshift;
    const int c0 = 16 * (wave & ((1 << cshift) - 1)), ncb = min(16, ncols - c0);
    int t = tb + (wave >> cshift);
    if (ncb <= 0) t = te;  // (3 blocks: the fourth wavefront has none)

    const scalar_i32 *table = (const scalar_i32 *)a.pt.table + (int64_t)b * a.pt.stride;
    const int tshift = a.pt.shift - 5, tmask = (1 << tshift) - 1;
    // the page id of a tile; -1 past the end
    const auto page_id = [&](int i) { return i < te ? table[i >> tshift] : -1; };
    const auto load = [&](PagedTile<FMT, D> &r, int i, int id) {
        const PageRsrc p = page_rsrc(a, id, hk, (uint32_t)id < (uint32_t)a.pt.n_pages);
        paged_load<FMT, D, ONCE>(r, p, 32u * (uint32_t)(i & tmask), lane);
    };
    int page[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) page[i] = page_id(t + i * step);

    PagedCol col;
    bf16x8 qhi[NCH], qlo[NCH];
    u32x4 qraw[NCH];
    {
        const bool ok = n < ncb;
        const int c = ok ? c0 + n : 0, qi = pf_div_group(c, a.group, a.group_m);
        const int head = hk * a.group + (c - qi * a.group);
        pf_key_range(qi, sq.lq, sq.lk, a.wl, a.wr, col.lo, col.hi);
        if (!ok) col.lo = col.hi = 0;
        col.qpos = qi + sq.lk - sq.lq;
        col.slope2 = a.alibi && ok ? a.alibi[(int64_t)b * a.alibi_bs + head] * kLog2e : 0.0f;
        const uint16_t *row = (const uint16_t *)a.q + (int64_t)(sq.first + qi) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
        for (int j = 0; j < NCH; ++j) qraw[j] = paged_q8(row, paged_qdim<FMT, D>(j, g), ok ? a.dim : 0, a.q_vec);
    }
    // keys that every column of the wavefront sees
    int lo_max, hi_min, unused;
    pf_key_range(pf_div_group(min(c0, ncols - 1), a.group, a.group_m), sq.lq, sq.lk, a.wl, a.wr, unused, hi_min);
    pf_key_range(pf_div_group(c0 + max(ncb, 1) - 1, a.group, a.group_m), sq.lq, sq.lk, a.wl, a.wr, lo_max, unused);

    PagedTile<FMT, D> tile[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        load(tile[i], t + i * step, page[i]);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        if constexpr (F16) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = f16_bits_to_f32((qraw[j][e / 2] >> (16 * (e & 1))) & 0xffffu);
            split_bf16x8(x, qhi[j], qlo[j]);
        } else {
            qhi[j] = __builtin_bit_cast(bf16x8, qraw[j]);
        }
    }

    f32x4 acc[2 * NCH];
#pragma unroll
    for (int i = 0; i < 2 * NCH; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -__builtin_inff(), l_run = 0.0f;
    const auto compute = [&](PagedTile<FMT, D> &r, int i, int id) {
        if ((uint32_t)id >= (uint32_t)a.pt.n_pages) return;  // a hole has no keys
        const int key0 = 32 * i;
        const bool full = key0 >= lo_max && key0 + 32 <= hi_min;
        paged_compute<FMT, D, F16>(r, a, key0, sq.lk, full, qhi, qlo, col, lane, m_run, l_run, acc);
    };
    // register sets take turns; the scheduling barriers keep the loads of one set issued before the
    // next set's, so each wait covers the set about to be used. Page ids are read a round ahead.
    for (; t < te; t += NS * step) {
        int ahead[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) ahead[i] = page_id(t + (NS + i) * step);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i == 0 || t + i * step < te) compute(tile[i], t + i * step, page[i]);
            __builtin_amdgcn_sched_barrier(0);
            load(tile[i], t + (NS + i) * step, ahead[i]);
            __builtin_amdgcn_sched_barrier(0);
            page[i] = ahead[i];
        }
    }

    // ---- merge the wavefronts of each column block ----
    const float l_col = group16_sum(l_run);
    if (n < ncb) {
#pragma unroll
        for (int v = 0; v < NCH; ++v)
#pragma unroll
            for (int i = 0; i < 4; i += 2)
                *(f32x4 *)&sm_o[wave][n][32 * v + 8 * g + 2 * i] =
                    f32x4{acc[2 * v][i], acc[2 * v + 1][i], acc[2 * v][i + 1], acc[2 * v + 1][i + 1]};
    }
    if (g == 0) {
        sm_m[wave][n] = m_run;
        sm_l[wave][n] = l_col;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < ncols * (D / 2); idx += WAVES * 64) {
        const int cc = idx / (D / 2), d = 2 * (idx % (D / 2)), w0 = cc >> 4, c = cc & 15;
        if (d >= a.dim) continue;  // plane row padding
        float M = -__builtin_inff();
        for (int w = w0; w < WAVES; w += 1 << cshift) M = fmaxf(M, sm_m[w][c]);
        float wsum = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int w = w0; w < WAVES; w += 1 << cshift) {
            // (a wavefront without a visible key, sum 0, has nothing to add; a NaN sum is kept)
            const float l = sm_l[w][c], f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sm_m[w][c] - M);
            const f32x2 v = *(const f32x2 *)&sm_o[w][c][d];
            wsum += l * f;
            o0 += l == 0.0f ? 0.0f : v.x * f;
            o1 += l == 0.0f ? 0.0f : v.y * f;
        }
        o0 = wsum == 0.0f ? 0.0f : o0 / wsum;
        o1 = wsum == 0.0f ? 0.0f : o1 / wsum;
        if (slot >= 0) {
            const int64_t at = (int64_t)slot * a.slot_cols + cc;
            *(f32x2 *)(a.part_o + at * D + d) = f32x2{o0, o1};
            if (d == 0) a.part_lse[at] = pf_piece_lse(M, wsum);
        } else {
            const int qi = pf_div_group(cc, a.group, a.group_m), head = hk * a.group + (cc - qi * a.group);
            const int64_t at = (int64_t)(sq.first + qi) * a.o_st + (int64_t)head * a.o_sh + d;
            store_elem(a.out, at, F16 ? CQKV_F16 : CQKV_BF16, o0);
            if (d + 1 < a.dim) store_elem(a.out, at + 1, F16 ? CQKV_F16 : CQKV_BF16, o1);
        }
    }
}

template <int FMT, int D>
inline void launch_paged_attn_d(bool f16, bool once, dim3 grid, hipStream_t st, const PagedAttnArgs &a) {
    if (f16 && once) hipLaunchKernelGGL((paged_attn_kernel<FMT, D, true, true>), grid, dim3(256), 0, st, a);
    else if (f16) hipLaunchKernelGGL((paged_attn_kernel<FMT, D, true, false>), grid, dim3(256), 0, st, a);
    else if (once) hipLaunchKernelGGL((paged_attn_kernel<FMT, D, false, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_kernel<FMT, D, false, false>), grid, dim3(256), 0, st, a);
}
template <int FMT>
inline void launch_paged_attn(int dk, bool f16, bool once, dim3 grid, hipStream_t st, const PagedAttnArgs &a) {
    if (dk == 64) launch_paged_attn_d<FMT, 64>(f16, once, grid, st, a);
    else if (dk == 128) launch_paged_attn_d<FMT, 128>(f16, once, grid, st, a);
    else launch_paged_attn_d<FMT, 256>(f16, once, grid, st, a);
}

#define CQKV_PAGED_ATTN_LAUNCHER(F) \
    void paged_attn_launch_##F(int dk, bool f16, bool once, dim3 grid, hipStream_t st, const PagedAttnArgs &a);
CQKV_PAGED_ATTN_LAUNCHER(2)
CQKV_PAGED_ATTN_LAUNCHER(4)
CQKV_PAGED_ATTN_LAUNCHER(5)

}  // namespace cqkv
