// Attention over a page pool, many columns per kv head (chunks of prompts): a column is a (query, head
// of the group) pair, query-major, 32 to a wavefront, up to 256 to a workgroup. Included by
// paged_inst.hip, one object per format.
//
// The pages' codes become MFMA operands of the queries' dtype once per workgroup: every thread loads 16
// codes of K and 16 of V of a 64-key tile and writes them to LDS as operands: keys exactly (E4M3 codes as
// they are, their f32 scale multiplies the scores; MX codes times their power of two), values times their
// scales, rounded to the dtype as a dequantized cache holds them; K rows in the order that
// makes the S^T registers of a lane whole groups of 8 keys (key bits 2 and 3 exchanged), V^T rows of 8-key
// chunks straight from the pool's 8-token tiles. From there it
// is the dense prefill's core: S^T(t + 1) on the MFMA pipe while the VALU exponentiates S(t), then
// O^T += V^T(t) P^T(t) while it sums P(t) and takes the maxima of S(t + 1). Two LDS stages each: step t
// reads K(t + 1) and V(t) and writes K(t + 2) and V(t + 1), whose codes were requested a step before.
// Bound by the MFMA and VALU work of the softmax; the conversion costs about 64 VALU instructions of a
// wavefront per tile beside the softmax's 110 and 32 exponentials.
// 512 tokens against 16K keys, FP8, 32 / 8 heads, D = 128: 157 us under the profiler, 0.86 PFLOP/s (151 us for a
// call with its merge); 1023 tokens against 7K keys, MXFP8: 139 us.
#pragma once

#include "paged_attn.h"
#include "prefill_core.h"

namespace cqkv {

// Geometry: W wavefronts, tiles of BK keys, NP pieces of E codes of K and of V per thread (K: E head dims
// of a key; V: E / 8 head dims of 8 keys).
template <int D, int W>
struct ChunkGeom {
    using P = PfGeom<D>;
    static constexpr int NT = 64 * W, BK = P::BK, PER = BK * D / NT;
    static constexpr int E = PER < 16 ? 8 : 16, NP = PER / E;
    static constexpr int KP = D / E, VP = D / (E / 8);  // pieces of a key row, of 8 keys
    static_assert(PER % E == 0, "whole pieces");
};

// A thread's codes and scales of one tile, in flight.
template <int FMT, int E>
struct ChunkK {
    static constexpr int CW = FMT == CQKV_FMT_MXFP4 ? E / 8 : E / 4;
    uint32_t c[CW];
    uint32_t s;
};
template <int FMT, int D, int E>
struct ChunkV {
    static constexpr int CW = FMT == CQKV_FMT_MXFP4 ? E / 8 : E / 4;
    static constexpr int SW = FMT == CQKV_FMT_FP8 ? 8 : D / 16;
    uint32_t c[CW];
    uint32_t s[SW];
};

template <int N>
PF_INLINE void chunk_words(uint32_t (&o)[N], const rsrc_t &r, uint32_t off) {
    if constexpr (N == 4) {
        const u32x4 w = ld128(r, off);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = w[i];
    } else if constexpr (N == 2) {
        const u32x2 w = ld64(r, off);
        o[0] = w.x;
        o[1] = w.y;
    } else {
        o[0] = ld32(r, off);
    }
}
// Piece of a thread: id = first + lane, first uniform (64 wavefront + pass * threads). codes, scales:
// resources of the page that holds the piece's 32-key block; row0: row of the tile's first key in that
// page (negative where the block is the tile's second, in a page of 32). Codes of consecutive pieces are
// consecutive, of K and of V.
template <int FMT, int D, int W>
PF_INLINE void chunk_load_k(ChunkK<FMT, ChunkGeom<D, W>::E> &o, const rsrc_t &codes, const rsrc_t &scales, int first,
                            int lane, int row0) {
    using C = ChunkGeom<D, W>;
    constexpr int BYTES = C::E / (FMT == CQKV_FMT_MXFP4 ? 2 : 1);
    chunk_words(o.c, codes, (uint32_t)((row0 * C::KP + first) * BYTES) + (uint32_t)lane * BYTES);
    const uint32_t key = (uint32_t)(row0 + first / C::KP) + (uint32_t)lane / C::KP;
    if constexpr (FMT == CQKV_FMT_FP8) o.s = ld32(scales, key * 4);
    else o.s = __builtin_amdgcn_raw_buffer_load_b8(scales, key * (D / 32) + (uint32_t)lane % C::KP * C::E / 32, 0, 0);
}
template <int FMT, int D, int W>
PF_INLINE void chunk_load_v(ChunkV<FMT, D, ChunkGeom<D, W>::E> &o, const rsrc_t &codes, const rsrc_t &scales, int first,
                            int lane, int row0) {
    using C = ChunkGeom<D, W>;
    constexpr int BYTES = C::E / (FMT == CQKV_FMT_MXFP4 ? 2 : 1);
    chunk_words(o.c, codes, (uint32_t)((row0 / 8 * C::VP + first) * BYTES) + (uint32_t)lane * BYTES);
    constexpr int SW = ChunkV<FMT, D, C::E>::SW;
    const uint32_t kg = (uint32_t)(row0 / 8 + first / C::VP) + (C::VP < 64 ? (uint32_t)lane / C::VP : 0u);
#pragma unroll
    for (int i = 0; i < SW / 4; ++i) {
        const u32x4 w = ld128(scales, kg * (SW * 4) + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) o.s[4 * i + e] = w[e];
    }
}
// LDS offsets of a thread's pieces of pass 0 within a stage (those of pass p: a whole number of rows on).
// K: chunk 0 of the piece (its second one: bit 4 exchanged), key bits 2 and 3 exchanged. V^T: the first
// head dim's chunk (the second's: one row on, the same place in it).
template <int D, int W>
PF_INLINE uint32_t chunk_k_offset(int id) {
    using C = ChunkGeom<D, W>;
    const int key = id / C::KP, c = id % C::KP * (C::E / 8);
    const int row = (key & ~12) | ((key & 4) << 1) | ((key & 8) >> 1);
    return row * PfGeom<D>::ROW + ((c ^ swz<D>(row)) << 4);
}
template <int D, int W>
PF_INLINE uint32_t chunk_v_offset(int id) {
    using C = ChunkGeom<D, W>;
    const int kg = id / C::VP, d = id % C::VP * (C::E / 8);
    return d * PfGeom<D>::VTROW + ((kg ^ swz_vt<PfGeom<D>::VTROW>(d)) << 4);
}

template <bool F16>
PF_INLINE uint32_t chunk_pack(float a, float b) { return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b); }

// The codes of one key as operands, exact: 16-byte chunks of its LDS row.
template <int FMT, int D, int W, bool F16>
PF_INLINE void chunk_store_k(const ChunkK<FMT, ChunkGeom<D, W>::E> &k, uint8_t *stage, uint32_t at) {
    using C = ChunkGeom<D, W>;
#pragma unroll
    for (int i8 = 0; i8 < C::E / 8; ++i8) {
        u32x4 w;
        // FP8: the bare codes; block byte 0 of the MX formats has zero codes
        const float s = FMT == CQKV_FMT_FP8 ? 1.0f : __uint_as_float(k.s << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (FMT != CQKV_FMT_MXFP4) {
                const uint32_t x = k.c[2 * i8 + i / 2];
                if constexpr (F16)
                    w[i] = i & 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, s, true))
                                 : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, s, false));
                else
                    w[i] = i & 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, true))
                                 : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, false));
            } else {
                const uint32_t x = k.c[i8] >> (8 * i);
                if constexpr (F16) w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s, 0));
                else w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s, 0));
            }
        }
        *(u32x4 *)(stage + (at ^ (16 * i8))) = w;
    }
}

// Codes and scales of keys past the end (nv of the 8 lie before it) may be any bytes: zeros.
template <int FMT, int D, int E>
PF_INLINE void chunk_cut_v(ChunkV<FMT, D, E> &v, int nv) {
    using V = ChunkV<FMT, D, E>;
    nv = max(nv, 0);
    if constexpr (FMT == CQKV_FMT_MXFP4) {
        const uint32_t keep = nv >= 8 ? ~0u : (1u << (4 * nv)) - 1u;
#pragma unroll
        for (int i = 0; i < V::CW; ++i) v.c[i] &= keep;
    } else {
        const uint64_t keep = nv >= 8 ? ~0ull : (1ull << (8 * nv)) - 1ull;
#pragma unroll
        for (int i = 0; i < V::CW; ++i) v.c[i] &= (uint32_t)(keep >> (32 * (i & 1)));
    }
    constexpr int BPK = FMT == CQKV_FMT_FP8 ? 4 : D / 32;  // scale bytes of a key
#pragma unroll
    for (int w = 0; w < V::SW; ++w)
#pragma unroll
        for (int y = 0; y < 4; ++y)
            if ((4 * w + y) / BPK >= nv) v.s[w] &= ~(0xffu << (8 * y));
}
// E / 8 head dims of 8 keys as operands: one 16-byte chunk of each V^T row.
template <int FMT, int D, int W, bool F16>
PF_INLINE void chunk_store_v(const ChunkV<FMT, D, ChunkGeom<D, W>::E> &v, uint8_t *stage, uint32_t at, int lane,
                             int first) {
    using C = ChunkGeom<D, W>;
    constexpr int DP = C::E / 8;  // head dims of a piece
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (FMT == CQKV_FMT_FP8) {
            s[e] = __uint_as_float(v.s[e]);
        } else {
            const int u = (first % C::VP + lane % C::VP) * DP / 32;  // the head dims' block
            if constexpr (D == 64) {
                s[e] = __uint_as_float(((v.s[e / 2] >> (16 * (e & 1) + 8 * u)) & 0xffu) << 23);
            } else {
                constexpr int NW = D / 128;
                const uint32_t w = NW == 1 || u < 4 ? v.s[NW * e] : v.s[NW * e + NW - 1];
                s[e] = __uint_as_float(((w >> (8 * (u & 3))) & 0xffu) << 23);
            }
        }
    }
#pragma unroll
    for (int i8 = 0; i8 < DP; ++i8) {
        float x[8];
        if constexpr (FMT == CQKV_FMT_MXFP4) {
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v.c[i8], 1.0f, 0);
            const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v.c[i8], 1.0f, 1);
            const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v.c[i8], 1.0f, 2);
            const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v.c[i8], 1.0f, 3);
            x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
            x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v.c[2 * i8 + i], false);
                const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(v.c[2 * i8 + i], true);
                x[4 * i] = a.x; x[4 * i + 1] = a.y; x[4 * i + 2] = b.x; x[4 * i + 3] = b.y;
            }
        }
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = chunk_pack<F16>(x[2 * i] * s[2 * i], x[2 * i + 1] * s[2 * i + 1]);
        *(u32x4 *)(stage + at + i8 * PfGeom<D>::VTROW) = w;
    }
}
// The keys of the 8 (bits) with a value of this piece that is not finite.
template <int FMT, int D, int E>
PF_INLINE uint32_t chunk_bad_keys(const ChunkV<FMT, D, E> &v) {
    uint32_t m = 0;
    if constexpr (FMT != CQKV_FMT_MXFP4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            bool bad = false;
#pragma unroll
            for (int i8 = 0; i8 < E / 8; ++i8) bad |= ((v.c[2 * i8 + e / 4] >> (8 * (e & 3))) & 0x7fu) == 0x7fu;
            if constexpr (FMT == CQKV_FMT_FP8) bad |= (v.s[e] & 0x7f800000u) == 0x7f800000u;
            m |= bad ? 1u << e : 0u;
        }
    }
    return m;
}

// Key of S^T register j of block mb, lane half h, from the tile's first: 32 mb + 16 (j / 8) + 8 h + j % 8.
template <int D>
PF_INLINE void chunk_mask(f32x16 *s, const PfState<D> &st, int k0, int lane, float mval) {
    int u = k0 + 8 * (lane >> 5) - st.qlo;  // key - qlo of register 0
    asm volatile("" : "+v"(u));
    const uint32_t w = (uint32_t)(st.qhi - st.qlo);
#pragma unroll
    for (int mb = 0; mb < PfGeom<D>::MB; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if ((uint32_t)(u + 32 * mb + 16 * (j >> 3) + (j & 7)) >= w) s[mb][j] = mval;
}
template <int MB>
PF_INLINE void chunk_logit(f32x16 *s, const PfLogit &lg, int k0, int lane) {
    if (lg.cap2 > 0.0f) {
        const float two_cap = 2.0f * lg.cap2;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = __builtin_amdgcn_exp2f(s[mb][j] * lg.e2);
                s[mb][j] = lg.cap2 - two_cap * __builtin_amdgcn_rcpf(e + 1.0f);
            }
    }
    if (lg.alibi) {
        const int d0 = lg.pos - (k0 + 8 * (lane >> 5));
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int dist = d0 - (32 * mb + 16 * (j >> 3) + (j & 7));
                s[mb][j] -= lg.slope2 * (float)(dist < 0 ? -dist : dist);
            }
    }
}

// Factors of this lane's 32 (16) scores of a tile, x = s * factor: the softmax scale in exp2 units, times
// the key's FP8 scale (from LDS, `ksc` at the tile's first key; register j of block mb is key
// 32 mb + 16 (j / 8) + 8 h + j % 8). SHIFT: x - m_run, one FMA.
template <int FMT, bool SHIFT, int D>
PF_INLINE void chunk_scale(f32x16 *s, const PfState<D> &st, const float *ksc, int lane) {
    if constexpr (FMT == CQKV_FMT_FP8) {
        const float *p = ksc + 8 * (lane >> 5);
#pragma unroll
        for (int mb = 0; mb < PfGeom<D>::MB; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 f = *(const f32x4 *)(p + 32 * mb + 16 * (i >> 1) + 4 * (i & 1));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = s[mb][4 * i + e];
                    s[mb][4 * i + e] = SHIFT ? __builtin_fmaf(x, f[e], st.negm) : x * f[e];
                }
            }
    } else if constexpr (SHIFT) {
        pf_shift_scaled<PfGeom<D>::MB>(s, st.c2, st.negm);
    } else {
        pf_scale<PfGeom<D>::MB>(s, st.c2);
    }
}

// O^T += V^T P^T of a tile with values that are not finite at the keys `bad` (bits, uniform), some of
// which some column does not see: those keys stay out of the products and are added one by one to the
// columns that see them.
template <bool F16, int D>
PF_INLINE void chunk_pv_bad(PfState<D> &st, const u32x4 *pop, const uint8_t *v_lds, const PfAddr<D> &ad,
                            uint64_t bad, int k0, int lane) {
    using op_t = pf_op_t<F16>;
    using G = PfGeom<D>;
    // (opaque, or the addresses below are kept in registers across the whole key loop)
    asm volatile("" : "+v"(lane));
    const int h = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < G::KK; ++kk) {
        const uint32_t b = (uint32_t)(bad >> (16 * kk + 8 * h)) & 0xffu;
        uint32_t keep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            keep[i] = ((b >> (2 * i)) & 1u ? 0u : 0xffffu) | ((b >> (2 * i + 1)) & 1u ? 0u : 0xffff0000u);
#pragma unroll
        for (int md = 0; md < G::MD; ++md) {
            u32x4 v = *(const u32x4 *)(v_lds + ad.v[kk] + md * 32 * G::VTROW);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] &= keep[i];
            st.acc[md] = mfma32x32x16(__builtin_bit_cast(op_t, v), __builtin_bit_cast(op_t, pop[kk]), st.acc[md]);
        }
    }
    while (bad) {
        const int key = __builtin_ctzll(bad);
        bad &= bad - 1;
        // the key's weight in this lane's column: 16-key step key / 16, lane half (key / 8) % 2
        uint32_t w = 0;
#pragma unroll
        for (int kk = 0; kk < G::KK; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (kk == key / 16 && i == (key & 7) / 2) w = pop[kk][i];
        w = (uint32_t)__shfl((int)w, (lane & 31) + 32 * ((key >> 3) & 1));
        w = key & 1 ? w >> 16 : w & 0xffffu;
        const float p = F16 ? f16_bits_to_f32(w) : bf16_bits_to_f32(w);
        const bool see = k0 + key >= st.qlo && k0 + key < st.qhi;
#pragma unroll
        for (int md = 0; md < G::MD; ++md)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (j % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // few reads in flight: registers
                const int d = 32 * md + 8 * (j >> 2) + 4 * h + (j & 3);
                const uint32_t x = *(const uint16_t *)(v_lds + d * G::VTROW +
                                                       (((key >> 3) ^ swz_vt<G::VTROW>(d)) << 4) + 2 * (key & 7));
                const float v = F16 ? f16_bits_to_f32(x) : bf16_bits_to_f32(x);
                if (see) st.acc[md][j] += p * v;
            }
    }
}

// One tile t of a wavefront (not its last): S(t) in cur, K(t + 1) at k_next, V(t) at v_cur. put_k / put_v
// convert the codes of later tiles and request the next ones, among the products of the two blocks (X:
// their VALU instructions per product); mask_next masks the scaled S(t + 1), whatever the scales of the
// keys out of sight are.
template <int FMT, bool LOGIT, bool F16, int D, int X, typename MaskFn, typename PutK, typename PutV>
PF_INLINE void chunk_tile(f32x16 *cur, f32x16 *nxt, u32x4 *pop, PfState<D> &st, const uint8_t *k_next,
                          const float *ksc_next, const uint8_t *v_cur, const PfAddr<D> &ad, int k1, int lane,
                          const PfLogit &lg, bool masked, MaskFn &&mask_next, PutK &&put_k, PutV &&put_v) {
    using G = PfGeom<D>;
    pf_qk<F16, D>(nxt, st, k_next, ad, f32x16{});
    pf_exp<F16, G::MB>(pop, cur);
    put_k();
    pf_block_schedule<G::V1 + X / 2, 0, G::NM>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * G::MB; ++i) asm volatile("" ::"v"(pop[i]));
    if (LOGIT) {
        chunk_scale<FMT, false>(nxt, st, ksc_next, lane);
        chunk_logit<G::MB>(nxt, lg, k1, lane);
    }
    pf_pv<F16, D, 0>(st, pop, v_cur, ad);
    pf_psum<F16, D>(st, pop);
    put_v();
    if (LOGIT) pf_shift<G::MB>(nxt, st.negm);
    else chunk_scale<FMT, true>(nxt, st, ksc_next, lane);
    float mx = pf_rowmax<G::MB>(nxt);
    pf_block_schedule<G::V2 + X, 0, G::NM>();
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {  // few tiles: scores relative to m_run, so the mask and the maximum come after them
        mask_next(nxt);
        mx = pf_rowmax<G::MB>(nxt);
    }
    mx = pf_max_halves(mx);
    const bool need = mx > st.thr;
    if (__builtin_expect(__any(need), 0)) pf_rescale(nxt, st, mx, need);
}

// LDS read offsets of a step from two bases (K, V^T): the chunk bits of the others are an exclusive or
// away, one VALU instruction where a register each would be held across the loop (the 12 of D = 128
// pushed the kernel past 256 registers). Opaque, so that they are made again in every step.
template <int D>
PF_INLINE void chunk_addr(PfAddr<D> &ad, uint32_t &kbase, uint32_t &vbase) {
    asm volatile("" : "+v"(kbase), "+v"(vbase));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) ad.k[i] = kbase ^ (uint32_t)(i << 5);
#pragma unroll
    for (int i = 0; i < PfGeom<D>::KK; ++i) ad.v[i] = vbase ^ (uint32_t)(i << 5);
}

// LDS of this wavefront's writes visible to the workgroup, and the workgroup's to it (global loads in
// flight are not waited for).
PF_INLINE void chunk_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int FMT, int D, int W, bool F16, bool LOGIT>
__global__ __launch_bounds__(W * 64, 1) void paged_chunk_kernel(PagedAttnArgs a) {
    using G = PfGeom<D>;
    using C = ChunkGeom<D, W>;
    constexpr int BK = C::BK, NC = 32 * W;
    __shared__ __attribute__((aligned(1024))) uint8_t ks0[G::KTILE];
    __shared__ __attribute__((aligned(1024))) uint8_t ks1[G::KTILE];
    __shared__ __attribute__((aligned(1024))) uint8_t vs0[G::VTILE];
    __shared__ __attribute__((aligned(1024))) uint8_t vs1[G::VTILE];
    __shared__ __attribute__((aligned(16))) float sm_ks0[BK], sm_ks1[BK];  // FP8: the factors of K's stages
    __shared__ uint32_t sm_bad[2];  // slow pass: keys of the tile with values that are not finite
    __shared__ int sm_holes, sm_any;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qr = lane & 31, h = lane >> 5;
    // blocks of columns of the sequences that this kernel takes, the last ones (with the most keys) first;
    // planes fastest, so that the workgroups of one plane's blocks share an XCD and its L2
    const int hk = (int)blockIdx.x % a.kv_heads, rest = (int)blockIdx.x / a.kv_heads;
    const int split = rest % a.chunk_splits;
    int idx = a.chunk_blocks - 1 - rest / a.chunk_splits;
    int b = -1, cb = 0;
    for (int base = 0; base < a.pt.batch; base += 64) {
        int n = 0;
        if (base + lane < a.pt.batch) {
            const int first = min(max(a.pt.cu[base + lane], 0), a.pt.total);
            const int len = min(min(max(a.pt.cu[base + lane + 1], first), a.pt.total) - first, a.max_q);
            const int64_t cols = (int64_t)len * a.group;
            n = cols > a.chunk_from ? (int)((cols + NC - 1) / NC) : 0;
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
            b = base + w;
            cb = idx - __builtin_amdgcn_readlane(sum - n, w);
            break;
        }
        idx -= __builtin_amdgcn_readlane(sum, 63);
    }
    if (b < 0) return;
    const PagedSeq sq = paged_seq(a, b);
    const int lq = sq.lq, lk = sq.lk;
    const int64_t ncols = (int64_t)min(lq, a.max_q) * a.group, c0 = (int64_t)cb * NC;
    const int ns = chunk_splits(a, sq);
    if (split >= ns) return;
    const int q0 = (int)((uint32_t)c0 / (uint32_t)a.group), cr0 = (int)(c0 - (int64_t)q0 * a.group);
    const int ncol = (int)min((int64_t)NC, ncols - c0);
    const auto query_of = [&](int c) { return pf_div_group(c, a.group, a.group_m); };

    // the block's key tiles within the split's range of the sequence's
    int kt_begin;
    int ntiles = pf_block_tiles(q0, q0 + query_of(cr0 + ncol - 1), lq, lk, a.wl, a.wr, BK, kt_begin);
    {
        const int first = sq.t0 * 32 / BK + split * a.chunk_tps;
        const int last = split == ns - 1 ? 0x7fffffff : first + a.chunk_tps;
        const int end = min(kt_begin + ntiles, last);
        kt_begin = max(kt_begin, first);
        ntiles = max(end - kt_begin, 0);
    }
    const bool wave_live = 32 * wave < ncol;
    int lo, hi, lo_last, hi_first;
    pf_key_range(q0 + query_of(cr0 + min(32 * wave, ncol - 1)), lq, lk, a.wl, a.wr, lo, hi_first);
    pf_key_range(q0 + query_of(cr0 + min(32 * wave + 32, ncol) - 1), lq, lk, a.wl, a.wr, lo_last, hi);
    const int wtiles = wave_live ? min(max((hi + BK - 1) / BK - kt_begin, 0), ntiles) : 0;

    PfState<D> st;
    PfLogit lg = {};
    {
        const bool ok = 32 * wave + qr < ncol;
        const int c = cr0 + min(32 * wave + qr, ncol - 1), qc = query_of(c), qi = q0 + qc;
        const int head = hk * a.group + (c - qc * a.group);
        const uint16_t *row = (const uint16_t *)a.q + (int64_t)(sq.first + qi) * a.q_st + (int64_t)head * a.q_sh;
        const float qs = a.scale_log2;
        st.c2 = qs == 0.0f ? 1.17549435e-38f : qs;
        st.mraw = 0.0f;  // (unused: scores are masked after their scaling)
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) {
            // (as they are: the scores are scaled in f32)
            st.qop[ks] = paged_q8(row, 16 * ks + 8 * h, ok ? a.dim : 0, a.q_vec);
        }
        if (ok) pf_key_range(qi, lq, lk, a.wl, a.wr, st.qlo, st.qhi);
        else st.qlo = st.qhi = 0;
        if (LOGIT) {
            lg.cap2 = a.cap2;
            lg.e2 = a.cap2 > 0.0f ? 2.0f * kLog2e / a.cap2 : 0.0f;
            lg.alibi = a.alibi != nullptr;
            lg.slope2 = a.alibi ? a.alibi[(int64_t)b * a.alibi_bs + head] * kLog2e : 0.0f;
            lg.pos = qi + lk - lq;
        }
    }

    const auto start = [&] {
        st.m_run = st.thr = -__builtin_inff();
        st.l_run = st.negm = 0.0f;
        st.negv = f32x16{};
#pragma unroll
        for (int md = 0; md < G::MD; ++md) st.acc[md] = f32x16{};
    };
    start();

    const scalar_i32 *table = (const scalar_i32 *)a.pt.table + (int64_t)b * a.pt.stride;
    const int tshift = a.pt.shift - 5, tmask = (1 << tshift) - 1;
    const int kb_end = (min(lk, (kt_begin + ntiles) * BK) + 31) / 32;  // 32-key blocks up to the last tile's
    if (tid == 0) sm_holes = sm_any = 0;
    __syncthreads();
    {
        bool hole = false;
        for (int i = kt_begin * BK / 32 + tid; i < kb_end; i += C::NT)
            hole |= (uint32_t)a.pt.table[(int64_t)b * a.pt.stride + (i >> tshift)] >= (uint32_t)a.pt.n_pages;
        if (hole) sm_holes = 1;
    }
    __syncthreads();
    const bool holes = __builtin_amdgcn_readfirstlane(sm_holes) != 0;
    // page id of 32-key block i of the sequence (of its last one past the end)
    const auto page_id = [&](int i) { return table[min(i, kb_end - 1) >> tshift]; };
    const auto is_page = [&](int page) { return (uint32_t)page < (uint32_t)a.pt.n_pages; };

    ChunkK<FMT, C::E> kr[C::NP];
    ChunkV<FMT, D, C::E> vr[C::NP];
    // 32-key block of the tile that piece p of this wavefront lies in (uniform)
    const auto k_block = [&](int p) { return (64 * wave + p * C::NT) / C::KP / 32; };
    const auto v_block = [&](int p) { return (64 * wave + p * C::NT) / C::VP / 4; };
    // Pages of the tiles whose codes the next step requests. Their ids are read before a barrier, whose wait
    // covers them (a scalar load in the middle of a step would wait for every LDS read in flight), the
    // resources made after it. A hole, or a tile past the end, has an empty resource: loads give zeros.
    int kpage[C::NP], vpage[C::NP];
    rsrc_t krc[C::NP], krs[C::NP], vrc[C::NP], vrs[C::NP];
    const auto next_pages = [&](int tk, int tv) {
#pragma unroll
        for (int p = 0; p < C::NP; ++p) {
            kpage[p] = tk < ntiles ? page_id((kt_begin + tk) * (BK / 32) + k_block(p)) : -1;
            vpage[p] = tv < ntiles ? page_id((kt_begin + tv) * (BK / 32) + v_block(p)) : -1;
        }
    };
    const auto resources = [&] {
#pragma unroll
        for (int p = 0; p < C::NP; ++p) {
            const bool kok = is_page(kpage[p]), vok = is_page(vpage[p]);
            const int64_t kp = kok ? (int64_t)kpage[p] * a.kv_heads + hk : 0;
            const int64_t vp = vok ? (int64_t)vpage[p] * a.kv_heads + hk : 0;
            krc[p] = pf_rsrc(a.k.codes + kp * a.k.codes_plane, kok ? a.k.codes_plane : 0u);
            krs[p] = pf_rsrc(a.k.scales + kp * a.k.scales_plane, kok ? a.k.scales_plane : 0u);
            vrc[p] = pf_rsrc(a.v.codes + vp * a.v.codes_plane, vok ? a.v.codes_plane : 0u);
            vrs[p] = pf_rsrc(a.v.scales + vp * a.v.scales_plane, vok ? a.v.scales_plane : 0u);
        }
    };
    // the codes of tile t into registers
    const auto load_k = [&](int t) {
#pragma unroll
        for (int p = 0; p < C::NP; ++p)
            chunk_load_k<FMT, D, W>(kr[p], krc[p], krs[p], 64 * wave + p * C::NT, lane,
                                    32 * ((((kt_begin + t) * (BK / 32) + k_block(p)) & tmask) - k_block(p)));
    };
    const auto load_v = [&](int t) {
#pragma unroll
        for (int p = 0; p < C::NP; ++p)
            chunk_load_v<FMT, D, W>(vr[p], vrc[p], vrs[p], 64 * wave + p * C::NT, lane,
                                    32 * ((((kt_begin + t) * (BK / 32) + v_block(p)) & tmask) - v_block(p)));
    };
    uint32_t k_at = chunk_k_offset<D, W>(tid), v_at = chunk_v_offset<D, W>(tid);
    // pass p's pieces: NT / KP key rows on (a multiple of 32: the same swizzle), NT / VP chunks on
    static_assert(C::NP == 1 || (C::NT / C::KP % 16 == 0 && C::VP <= C::NT), "passes of whole rows");
    const auto store_k = [&](uint8_t *stage, float *ksc) {
#pragma unroll
        for (int p = 0; p < C::NP; ++p) {
            chunk_store_k<FMT, D, W, F16>(kr[p], stage + p * (C::NT / C::KP) * G::ROW, k_at);
            // (a scale's sign bit is zero but in the bytes of keys past the end, which are masked)
            if constexpr (FMT == CQKV_FMT_FP8)
                ksc[(tid + p * C::NT) / C::KP] = __builtin_fabsf(__uint_as_float(kr[p].s)) * st.c2;
        }
    };
    const auto store_v = [&](uint8_t *stage) {
#pragma unroll
        for (int p = 0; p < C::NP; ++p)
            chunk_store_v<FMT, D, W, F16>(vr[p], stage, v_at ^ (uint32_t)((p * (C::NT / C::VP)) << 4), lane,
                                          64 * wave + p * C::NT);
    };
    // keys that every column of the workgroup sees
    int wlo_max, whi_min, unused;
    pf_key_range(q0, lq, lk, a.wl, a.wr, unused, whi_min);
    pf_key_range(q0 + query_of(cr0 + ncol - 1), lq, lk, a.wl, a.wr, wlo_max, unused);
    // Codes of V(t), before they are converted: the end of the keys, and values that are not finite where
    // some column does not see some key (0 times them is NaN): the pass is then done again, slowly.
    const auto check_v = [&](int t, bool slow) {
        const int k0 = (kt_begin + t) * BK;
        if (k0 >= wlo_max && k0 + BK <= whi_min) return;
#pragma unroll
        for (int p = 0; p < C::NP; ++p) {
            const int kg = (tid + p * C::NT) / C::VP;
            // (opaque: few tiles come here, and the work must not be done ahead of the branch for all)
#pragma unroll
            for (uint32_t &c : vr[p].c) asm volatile("" : "+v"(c));
#pragma unroll
            for (uint32_t &c : vr[p].s) asm volatile("" : "+v"(c));
            chunk_cut_v<FMT, D, C::E>(vr[p], lk - (k0 + 8 * kg));
            if constexpr (FMT != CQKV_FMT_MXFP4) {
                const uint32_t bad = chunk_bad_keys<FMT, D, C::E>(vr[p]);
                if (bad && slow) atomicOr(&sm_bad[kg >> 2], bad << (8 * (kg & 3)));
                else if (bad) sm_any = 1;
            }
        }
    };

    if (ntiles > 0) {
        // K(0), K(1) and V(0) into LDS, the codes of K(2) and V(1) in flight
        next_pages(0, 0);
        resources();
        load_k(0);
        load_v(0);
        next_pages(1, 1);
        resources();
        store_k(ks0, sm_ks0);
        load_k(1);
        check_v(0, false);
        store_v(vs0);
        load_v(1);
        next_pages(2, 2);
        resources();
        store_k(ks1, sm_ks1);
        load_k(2);
        next_pages(3, 2);
    }
    __syncthreads();

    const auto tile_masked = [&](int t) {
        const int k0 = (kt_begin + t) * BK;
        return holes || !(k0 >= lo_last && k0 + BK <= hi_first);
    };
    const auto mask = [&](f32x16 *s, int t) {
        const int k0 = (kt_begin + t) * BK;
        const float mval = -__builtin_inff();
        chunk_mask(s, st, k0, lane, mval);
        if (holes) {
#pragma unroll
            for (int mb = 0; mb < G::MB; ++mb)
                if (!is_page(page_id(k0 / 32 + mb)))
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[mb][j] = mval;
        }
    };
    f32x16 sa[G::MB], sb[G::MB];
    u32x4 pop[2 * G::MB];
    PfAddr<D> ad;
    pf_addr_init<D>(ad, lane);
    uint32_t kbase = ad.k[0], vbase = ad.v[0] - G::VBIAS;
    chunk_addr<D>(ad, kbase, vbase);
    if (wtiles > 0) {
        pf_qk<F16, D>(sa, st, ks0, ad, f32x16{});
        chunk_scale<FMT, false>(sa, st, sm_ks0, lane);  // (negm is 0 here)
        if (LOGIT) chunk_logit<G::MB>(sa, lg, kt_begin * BK, lane);
        if (tile_masked(0)) mask(sa, 0);
        const float mx = pf_max_halves(pf_rowmax<G::MB>(sa));
        const bool need = mx > st.thr;
        if (__any(need)) pf_rescale(sa, st, mx, need);
    }
    __syncthreads();  // K(0) is read: its stage takes K(2)

    // Step t: K(t + 1) and V(t) are in LDS; K(t + 2) goes into K(t)'s stage and V(t + 1) into V(t - 1)'s,
    // both read by every wavefront before the barrier that ended step t - 1.
    constexpr int X = (2 * C::E * C::NP + G::NM - 1) / G::NM;  // conversion VALU instructions per product
    int t = 0;
    const auto put_k = [&](uint8_t *stage, float *ksc) {
        store_k(stage, ksc);
        load_k(t + 3);
    };
    const auto put_v = [&](uint8_t *stage) {
        store_v(stage);
        load_v(t + 2);
    };
    const auto step_end = [&] {
        next_pages(t + 4, t + 3);
        chunk_barrier();
        ++t;
    };
#define CHUNK_STEP(CUR, NXT, KN, SN, KW, SW, VC, VW)                                                    \
    {                                                                                                   \
        chunk_addr<D>(ad, kbase, vbase);                                                                \
        resources();                                                                                    \
        const bool masked = tile_masked(t + 1);                                                         \
        check_v(t + 1, false);                                                                          \
        __builtin_amdgcn_sched_barrier(0);                                                              \
        chunk_tile<FMT, LOGIT, F16, D, X>(                                                              \
            CUR, NXT, pop, st, KN, SN, VC, ad, (kt_begin + t + 1) * BK, lane, lg, masked,               \
            [&](f32x16 *s) { mask(s, t + 1); }, [&] { put_k(KW, SW); }, [&] { put_v(VW); });            \
        step_end();                                                                                     \
    }
    while (t + 1 < wtiles) {
        CHUNK_STEP(sa, sb, ks1, sm_ks1, ks0, sm_ks0, vs0, vs1)
        if (t + 1 >= wtiles) break;
        CHUNK_STEP(sb, sa, ks0, sm_ks0, ks1, sm_ks1, vs1, vs0)
    }
#undef CHUNK_STEP
    // the wavefront's last tile, and the tiles that only later columns of the workgroup see
    if (wtiles > 0) {
        chunk_addr<D>(ad, kbase, vbase);
        if (t & 1) pf_last_tile<F16, D, 0>(sb, pop, st, vs1, ad);
        else pf_last_tile<F16, D, 0>(sa, pop, st, vs0, ad);
    }
#pragma unroll
    for (int md = 0; md < G::MD; ++md) asm volatile("" : "+v"(st.acc[md]));
    while (t < ntiles) {
        resources();
        put_k(t & 1 ? ks1 : ks0, t & 1 ? sm_ks1 : sm_ks0);
        check_v(t + 1, false);
        put_v(t & 1 ? vs0 : vs1);
        step_end();
    }
    if constexpr (FMT != CQKV_FMT_MXFP4) {
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(sm_any) != 0, 0)) {
            start();
#pragma unroll 1
            for (t = 0; t < ntiles; ++t) {
                __syncthreads();  // the last tile is read
                if (tid < 2) sm_bad[tid] = 0;
                next_pages(t, t);
                resources();
                load_k(t);
                load_v(t);
                __syncthreads();
                store_k(ks0, sm_ks0);
                check_v(t, true);
                store_v(vs0);
                __syncthreads();
                if (t >= wtiles) continue;
                chunk_addr<D>(ad, kbase, vbase);
                pf_qk<F16, D>(sa, st, ks0, ad, f32x16{});
                chunk_scale<FMT, false>(sa, st, sm_ks0, lane);
                if (LOGIT) chunk_logit<G::MB>(sa, lg, (kt_begin + t) * BK, lane);
                if (tile_masked(t)) mask(sa, t);
                pf_shift<G::MB>(sa, st.negm);
                const float mx = pf_max_halves(pf_rowmax<G::MB>(sa));
                const bool need = mx > st.thr;
                if (__any(need)) pf_rescale(sa, st, mx, need);
                pf_exp<F16, G::MB>(pop, sa);
                const uint64_t bad = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)sm_bad[0]) |
                                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)sm_bad[1]) << 32;
                chunk_pv_bad<F16, D>(st, pop, vs0, ad, bad, (kt_begin + t) * BK, lane);
                pf_psum<F16, D>(st, pop);
            }
        }
    }

    // ---- normalise and write O: lane (qr, h), head dims 32 md + 8 (j / 4) + 4 h + j % 4 ----
    const float l = pf_sum_halves(st.l_run);
    if (32 * wave + qr >= ncol) return;
    const int c = cr0 + 32 * wave + qr, qc = query_of(c);
    const int64_t token = sq.first + q0 + qc;
    const int head = hk * a.group + (c - qc * a.group);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (ns > 1) {  // this split's normalised rows and their log2-sum-exp
        const int64_t rows = (int64_t)a.pt.total * a.q_heads, row = split * rows + token * a.q_heads + head;
        if (h == 0) a.chunk_lse[row] = pf_piece_lse(st.m_run, l);
        if (l == 0.0f) return;  // no weight: the merge does not read the row
        float *po = a.chunk_o + row * D + 4 * h;
#pragma unroll
        for (int md = 0; md < G::MD; ++md)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(f32x4 *)(po + 32 * md + 8 * j) = f32x4{st.acc[md][4 * j] * inv, st.acc[md][4 * j + 1] * inv,
                                                         st.acc[md][4 * j + 2] * inv, st.acc[md][4 * j + 3] * inv};
        return;
    }
    uint16_t *orow = (uint16_t *)a.out + token * a.o_st + (int64_t)head * a.o_sh;
#pragma unroll
    for (int md = 0; md < G::MD; ++md)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * md + 8 * j + 4 * h;
            const u32x2 w = {chunk_pack<F16>(st.acc[md][4 * j] * inv, st.acc[md][4 * j + 1] * inv),
                             chunk_pack<F16>(st.acc[md][4 * j + 2] * inv, st.acc[md][4 * j + 3] * inv)};
            if (a.o_vec) {
                if (d < a.dim) *(u32x2 *)(orow + d) = w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < a.dim) orow[d + e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
            }
        }
}

// Wavefronts of 32 columns in a workgroup: 8 fill a CU, so a tile is converted once there (32 / 8 heads, a
// chunk of 512 against 16K keys, FP8, D = 128: 159 us; 4 wavefronts, two workgroups a CU: 251); at D = 256
// the registers allow 4.
constexpr int chunk_waves(int d) { return d < 256 ? 8 : 4; }

template <int FMT, int D>
inline void launch_paged_chunk_d(bool f16, bool logit, dim3 grid, hipStream_t st, const PagedAttnArgs &a) {
    constexpr int W = chunk_waves(D);
    const dim3 block(64 * W);
    if (f16 && logit) hipLaunchKernelGGL((paged_chunk_kernel<FMT, D, W, true, true>), grid, block, 0, st, a);
    else if (f16) hipLaunchKernelGGL((paged_chunk_kernel<FMT, D, W, true, false>), grid, block, 0, st, a);
    else if (logit) hipLaunchKernelGGL((paged_chunk_kernel<FMT, D, W, false, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_chunk_kernel<FMT, D, W, false, false>), grid, block, 0, st, a);
}
template <int FMT>
inline void launch_paged_chunk(int dk, bool f16, bool logit, dim3 grid, hipStream_t st, const PagedAttnArgs &a) {
    if (dk == 64) launch_paged_chunk_d<FMT, 64>(f16, logit, grid, st, a);
    else if (dk == 128) launch_paged_chunk_d<FMT, 128>(f16, logit, grid, st, a);
    else launch_paged_chunk_d<FMT, 256>(f16, logit, grid, st, a);
}

#define CQKV_PAGED_CHUNK_LAUNCHER(F) \
    void paged_chunk_launch_##F(int dk, bool f16, bool logit, dim3 grid, hipStream_t st, const PagedAttnArgs &a);
CQKV_PAGED_CHUNK_LAUNCHER(2)
CQKV_PAGED_CHUNK_LAUNCHER(4)
CQKV_PAGED_CHUNK_LAUNCHER(5)

}  // namespace cqkv
