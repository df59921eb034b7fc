// The per-wavefront core of the MFMA prefill: S^T = K Q^T from an LDS key tile, the online softmax in
// registers, O^T += V^T P^T from an LDS V^T tile, and the schedule that interleaves them. Shared by the
// dense prefill (prefill_attn.hip) and the chunk attention over a page pool (paged_chunk.h).
#pragma once

#include <type_traits>

#include "cqkv_device.h"

namespace cqkv {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ inline f32x16 mfma32x32x16(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mfma32x32x16(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// MFMA operands of the input dtype: q, K, V^T and P all in bf16, or all in f16
template <bool F16>
using pf_op_t = typename std::conditional<F16, f16x8, bf16x8>::type;

__device__ inline u32x4 ldg128(const uint16_t *p) { return *(const u32x4 *)p; }

// LDS K tile layout: 64 rows (keys) x 2 D bytes, no padding; the 16-byte chunk c of row r sits at
// chunk position c ^ swz(r). At D = 128 (16 chunks a row) swz takes 16 distinct values over any 16
// consecutive rows (the 16 rows of one ds_read_b128 pass); at D = 64 (8 chunks a row, two rows per
// 256 bytes of banks) (r % 2, c ^ swz(r)) takes 16 distinct values over them: either way the
// reads are conflict-free.
template <int D>
__device__ inline int swz(int r) {
    if constexpr (D >= 128) return ((r & 7) << 1) | ((r >> 3) & 1);  // rows of 16 or 32 chunks
    else return (r >> 1) & 7;
}
// V^T tile layout in LDS: D rows (head dims) x VTROW bytes (keys of the tile); the 16-byte chunk j
// (8 keys) of row d sits at position j ^ swz_vt(d). With 128-byte rows, over any 16 consecutive
// rows (d % 2, position) takes 16 distinct values; with 64-byte rows, (d % 4, position) does: a
// ds_read_b128 of one chunk across 16 rows is conflict-free either way.
template <int VTROW>
__device__ inline int swz_vt(int d) {
    if constexpr (VTROW == 128) return (d >> 1) & 7;
    else return (d >> 2) & 3;
}
// Per head dim:
//  * the workgroup: W wavefronts of 32 columns, NC columns in all (8 at D <= 128, two per SIMD; 4
//    at D = 256, one per SIMD with VGPRs and AGPRs, as the 32 x 256 accumulator, the queries and
//    the scores take more than 256 registers);
//  * key tiles of BK keys (64; 32 at D = 256, so that four ring stages of K and V^T fit in LDS):
//    MB 32-key blocks of S, KK 16-key steps of O^T += V^T P^T;
//  * 16-dim k-steps of S = K Q^T, 32-dim blocks of O^T, bytes of a K row and tile, of a V^T row
//    (BK keys) and tile, and each wavefront's 1 KB copies of a tile: K rows (BK / W) w .., V^T rows
//    (D / W) w .. in pieces of 1024 / VTROW rows.
//  * The V^T stages follow the four K stages in LDS: VBIAS shifts V^T read offsets so that
//    (stage - VBIAS) + block offset fits the 16-bit DS offset.
//  * VALU instructions per MFMA of the two blocks of a tile step (scores: exponentials and
//    conversions; then row sums, shift and row maximum).
template <int D>
struct PfGeom {
    static constexpr int W = D == 256 ? 4 : 8, NC = 32 * W;
    static constexpr int BK = D == 256 ? 32 : 64, MB = BK / 32, KK = BK / 16, VTROW = 2 * BK;
    static constexpr int KS = D / 16, MD = D / 32;
    static constexpr int ROW = 2 * D, KTILE = BK * ROW, VTILE = D * VTROW;
    static constexpr int RPC = 1024 / ROW;  // K rows per copy
    static constexpr int KCP = KTILE / 1024 / W, VCP = VTILE / 1024 / W;
    static constexpr int CP = KCP + VCP;    // copies per wavefront and tile
    static constexpr uint32_t VBIAS = 4 * KTILE;
    static constexpr int NM = MB * KS;      // MFMAs per block (S(t + 1); O^T += V^T P^T)
    static constexpr int V1 = (24 * MB + NM - 1) / NM, V2 = (32 * MB + NM - 1) / NM;
    static constexpr int V2C = (16 * MB + NM - 1) / NM;  // block 2 when the MFMA adds -m_run
    // D = 256: the queries enter the MFMA as given and the scores are scaled in f32 (the shift
    // becomes one FMA); with sums over 256 dims the rounding of pre-scaled queries to the dtype
    // moved outputs by up to 3 bf16 ulps
    static constexpr bool QRAW = D == 256;
    static_assert(NM == MD * KK, "both blocks of a step have NM products");
};

typedef __attribute__((address_space(3))) void lds_void;

#define PF_INLINE __device__ __attribute__((always_inline)) inline

// A buffer resource from wavefront-uniform values, built in scalar registers (the compiler can
// otherwise move the address to vector registers and wrap each copy in a per-lane loop).
PF_INLINE rsrc_t pf_rsrc(const void *base, uint32_t bytes) {
    const uint64_t p = (uint64_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
    return make_rsrc((const void *)(((uint64_t)hi << 32) | lo), __builtin_amdgcn_readfirstlane(bytes));
}
// s_waitcnt vmcnt(n) (gfx9 encoding; expcnt and lgkmcnt left at their maxima)
#define PF_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt((((n) & 15) | (((n) >> 4) << 14)) | 0x0f70)

template <int D>
struct PfState {
    u32x4 qop[D / 16];  // Q^T operands (16-dim steps ks) of this wavefront's 32 columns, raw bits
    f32x16 acc[D / 32]; // O^T: 32-dim block md
    float negm;      // -m_run (0 before the first key), added to the raw scores
    f32x16 negv;     // negm in every register: the initial value of the score products when
                     // the scores need no f32 scaling or terms before the shift
    float m_run, l_run;
    float c2;        // scores' factor when the queries enter unscaled (QRAW): scale * log2(e)
    float mraw;      // the mask value of unscaled scores: -inf times the sign of c2
    float thr;       // the row maximum moves when a tile's maximum exceeds thr: -inf before the
                     // row's first key, then 8 (p stays below 2^8)
    int qlo, qhi;    // visible keys of this lane's query
};

constexpr int kDsRead = 0x100, kMfma = 0x008, kValu = 0x402;  // sched_group_barrier classes (VALU + TRANS)

// Orders a block of NM MFMAs with its NM LDS operand reads, VALU VALU instructions per MFMA
// and the VMEM (tile copy) instructions: four reads first, then MFMA, read, copy, VALU x VALU,
// so each MFMA's operand was requested four MFMAs earlier and the VALU work fills the MFMA
// pipe's busy cycles.
template <int VALU, int VMEM = 0, int NM = 16>
PF_INLINE void pf_block_schedule() {
#pragma unroll
    for (int i = 0; i < 4; ++i) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        if (i < NM - 4) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
        if (i < VMEM) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
        if (VALU > 0) __builtin_amdgcn_sched_group_barrier(kValu, VALU, 0);
    }
}

// Per-lane LDS read offsets from the first stage of each ring, kept in registers and made opaque
// at every step, so each read is one register plus a constant that fits the 16-bit DS offset
// field (stage, key block, head-dim block); left alone, the compiler keeps a register per
// (stage, offset) pair.
template <int D>
struct PfAddr {
    uint32_t k[D / 16];           // K row qr, chunk 2 ks + h (swizzled), of key block 0
    uint32_t v[PfGeom<D>::KK];    // VBIAS + V^T row qr, chunk 2 kk + h (swizzled), of head-dim block 0
};
// The V^T stages follow the four K stages; biasing the V^T offsets by their size (64 KB at
// D = 128) leaves (stage address - bias) + head-dim block offset, below 64 KB, as the constant
// part.
template <int D>
PF_INLINE void pf_addr_init(PfAddr<D> &ad, int lane) {
    const int qr = lane & 31, h = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
        ad.k[ks] = qr * PfGeom<D>::ROW + (((2 * ks + h) ^ swz<D>(qr)) << 4);
#pragma unroll
    for (int kk = 0; kk < PfGeom<D>::KK; ++kk)
        ad.v[kk] = PfGeom<D>::VBIAS + qr * PfGeom<D>::VTROW +
                   (((2 * kk + h) ^ swz_vt<PfGeom<D>::VTROW>(qr)) << 4);
}
template <int D>
PF_INLINE void pf_addr_opaque(PfAddr<D> &ad) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(ad.k[i]));
#pragma unroll
    for (int i = 0; i < PfGeom<D>::KK; ++i) asm volatile("" : "+v"(ad.v[i]));
}

// S^T (BK keys x 32 queries) = K Q^T for the tile at k_lds: MB 32-key blocks.
template <bool F16, int D>
PF_INLINE void pf_qk(f32x16 *s, const PfState<D> &st, const uint8_t *k_lds, const PfAddr<D> &ad,
                     const f32x16 &c0) {
    using op_t = pf_op_t<F16>;
    constexpr int KS = D / 16, MB = PfGeom<D>::MB;
    op_t kop[MB * KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
            kop[KS * mb + ks] = __builtin_bit_cast(
                op_t, *(const u32x4 *)(k_lds + ad.k[ks] + 32 * mb * PfGeom<D>::ROW));
    // with two key blocks their chains alternate, so consecutive products are independent
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
        s[mb] = mfma32x32x16(kop[KS * mb], __builtin_bit_cast(op_t, st.qop[0]), c0);
#pragma unroll
    for (int ks = 1; ks < KS; ++ks)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
            s[mb] = mfma32x32x16(kop[KS * mb + ks], __builtin_bit_cast(op_t, st.qop[ks]), s[mb]);
}

// Soft-capping and ALiBi of the raw scores of a tile whose first key is k0 (exp2 units, in the
// reference's order: cap * tanh(s / cap), then - slope * |pos - key|; fa_logit,
// candle-core/kernels/flash_attn_impl.h:42-47). pos is the lane's query position in key
// coordinates.
struct PfLogit {
    float cap2;   // softcap * log2(e) (0: off)
    float e2;     // 2 log2(e) / cap2: exp2(s * e2) = e^(2 s / cap2)
    float slope2; // ALiBi slope * log2(e) of the lane's head
    int alibi;    // slopes given
    int pos;
};
// cap * tanh(x / cap) = cap - 2 cap / (e^(2x / cap) + 1): one exp2 and one reciprocal, exact
// limits at both ends (e -> inf: cap; e -> 0: -cap), absolute error ~1e-7 cap
template <int MB>
PF_INLINE void pf_logit(f32x16 *s, const PfLogit &lg, int k0, int lane) {
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
        const int d0 = lg.pos - (k0 + 4 * (lane >> 5));  // pos - key of register 0
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int dist = d0 - (32 * mb + 8 * (j >> 2) + (j & 3));
                s[mb][j] -= lg.slope2 * (float)(dist < 0 ? -dist : dist);
            }
    }
}

// masks scores of keys outside the lane's visible range (tiles that cross a range end only)
template <int D>
PF_INLINE void pf_mask(f32x16 *s, const PfState<D> &st, int k0, int lane,
                       float mval = -__builtin_inff()) {
    const int h = lane >> 5;
    // key - qlo of register 0, made opaque so the per-register offsets stay immediates
    int u = k0 + 4 * h - st.qlo;
    asm volatile("" : "+v"(u));
    const uint32_t w = (uint32_t)(st.qhi - st.qlo);
#pragma unroll
    for (int mb = 0; mb < PfGeom<D>::MB; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if ((uint32_t)(u + 32 * mb + 8 * (j >> 2) + (j & 3)) >= w) s[mb][j] = mval;
}

PF_INLINE float pf_max_halves(float x) {  // max of lanes l and l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
PF_INLINE float pf_sum_halves(float x) {  // sum of lanes l and l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// scores relative to the running maximum
template <int MB>
PF_INLINE void pf_scale(f32x16 *s, float c) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[mb][j] *= c;
}
// unscaled scores to the exponent: s * c - m_run, one FMA each
template <int MB>
PF_INLINE void pf_shift_scaled(f32x16 *s, float c, float negm) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[mb][j] = __builtin_fmaf(s[mb][j], c, negm);
}
template <int MB>
PF_INLINE void pf_shift(f32x16 *s, float negm) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[mb][j] += negm;
}

// this lane's maximum over the tile (two chains: the two key blocks, or the even and odd
// registers of one)
template <int MB>
PF_INLINE float pf_rowmax(const f32x16 *s) {
    if constexpr (MB == 2) {
        float m0 = s[0][0], m1 = s[1][0];
#pragma unroll
        for (int j = 1; j < 16; ++j) {
            m0 = fmaxf(m0, s[0][j]);
            m1 = fmaxf(m1, s[1][j]);
        }
        return fmaxf(m0, m1);
    } else {
        float m0 = s[0][0], m1 = s[0][1];
#pragma unroll
        for (int j = 2; j < 16; j += 2) {
            m0 = fmaxf(m0, s[0][j]);
            m1 = fmaxf(m1, s[0][j + 1]);
        }
        return fmaxf(m0, m1);
    }
}

// The row maximum moves (rare): s is shifted to the new maximum, O and the row sum rescaled.
// Q carries scale * log2(e) and pf_shift adds -m_run, so s is the exponent of p = exp2(s)
// relative to m_run.
template <int D>
PF_INLINE void pf_rescale(f32x16 *s, PfState<D> &st, float mx, bool need) {
    const bool fresh = st.m_run == -__builtin_inff();
    const float shift = need ? mx : 0.0f;
    const float m_new = need ? (fresh ? 0.0f : st.m_run) + mx : st.m_run;
    const float alpha = need ? __builtin_amdgcn_exp2f(st.m_run - m_new) : 1.0f;
#pragma unroll
    for (int mb = 0; mb < PfGeom<D>::MB; ++mb)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[mb][j] -= shift;
#pragma unroll
    for (int md = 0; md < D / 32; ++md) st.acc[md] *= alpha;
    st.l_run *= alpha;
    st.m_run = m_new;
    st.thr = m_new == -__builtin_inff() ? -__builtin_inff() : 8.0f;
    st.negm -= shift;  // -m_new: 0 - mx for a row's first keys, -m_run - mx after
#pragma unroll
    for (int j = 0; j < 16; ++j) st.negv[j] = st.negm;
}

// p = exp2(s), packed to the P^T operands of the dtype (raw bits)
template <bool F16, int MB>
PF_INLINE void pf_exp(u32x4 *pop, const f32x16 *s) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = __builtin_amdgcn_exp2f(s[mb][8 * half + 2 * e]);
                const float p1 = __builtin_amdgcn_exp2f(s[mb][8 * half + 2 * e + 1]);
                if constexpr (F16) {
                    w[e] = pack_f16x2(p0, p1);
                } else {
                    const bf16x2 pp = {(__bf16)p0, (__bf16)p1};
                    w[e] = __builtin_bit_cast(uint32_t, pp);
                }
            }
            pop[2 * mb + half] = u32x4{w[0], w[1], w[2], w[3]};
        }
}

// the row sum adds the bf16 values the product uses, two per dot2 instruction, in two chains
// (each word goes through a scalar: clang's __builtin_bit_cast of a vector element reads
// element 0)
template <bool F16>
PF_INLINE float pf_dot2_ones(uint32_t w, float acc) {
    if constexpr (F16) {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        const f16x2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w), ones, acc, false);
    } else {
        const bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), ones, acc, false);
    }
}
template <bool F16, int D>
PF_INLINE void pf_psum(PfState<D> &st, const u32x4 *pop) {
    float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * PfGeom<D>::MB; ++i) {
        const u32x4 w = pop[i];
        const uint32_t w0 = w.x, w1 = w.y, w2 = w.z, w3 = w.w;
        a0 = pf_dot2_ones<F16>(w0, a0);
        a1 = pf_dot2_ones<F16>(w1, a1);
        a0 = pf_dot2_ones<F16>(w2, a0);
        a1 = pf_dot2_ones<F16>(w3, a1);
    }
    st.l_run += a0 + a1;
}

// O^T += V^T P^T over the V^T tile at v_lds. 16-key step kk = keys 16 kk + [0, 16): the P^T
// operand holds S^T registers 8 (kk % 2) .. +7 of key block kk / 2, i.e. lane half h holds keys
// 16 kk + 8 (e / 4) + 4 h + e % 4 in k-slot 8 h + e; the pre-pass stores V^T keys in that order
// (bits 2 and 3 of the key swapped), so the A operand of lane (d, h) is chunk 2 kk + h of row d.
// (BIAS: what ad.v carries beyond the offset in the stage)
template <bool F16, int D, uint32_t BIAS = PfGeom<D>::VBIAS>
PF_INLINE void pf_pv(PfState<D> &st, const u32x4 *pop, const uint8_t *v_lds, const PfAddr<D> &ad) {
    using op_t = pf_op_t<F16>;
    constexpr int MD = D / 32, KK = PfGeom<D>::KK;
    op_t vt[KK * MD];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int md = 0; md < MD; ++md)
            vt[MD * kk + md] = __builtin_bit_cast(
                op_t, *(const u32x4 *)(v_lds + (ad.v[kk] - BIAS) + md * 32 * PfGeom<D>::VTROW));
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int md = 0; md < MD; ++md)
            st.acc[md] = mfma32x32x16(vt[MD * kk + md], __builtin_bit_cast(op_t, pop[kk]), st.acc[md]);
}

// One key tile t of a wavefront (not the last), with S(t) in `cur`:
//  * block 1: S(t + 1) = K(t + 1) Q^T into `nxt` on the MFMA pipe while the VALU turns S(t)
//    into P(t) = exp2(S(t));
//  * on tiles that cross a range end, S(t + 1) is masked;
//  * block 2: O += V(t)^T P(t) on the MFMA pipe while the VALU adds up the row sum of P(t),
//    shifts S(t + 1) by -m_run and takes its row maximum; the copies of a later tile
//    (issue_copies) are issued among its first MFMAs;
//  * then, rarely, the row maximum moves (pf_rescale).
// At D = 64 each block has half the MFMAs of D = 128 for the same softmax work: twice the VALU
// instructions go between consecutive MFMAs.
template <bool LOGIT, bool F16, int D, typename IssueCopies>
PF_INLINE void pf_tile(f32x16 *cur, f32x16 *nxt, u32x4 *pop, PfState<D> &st,
                       const uint8_t *k_next, const uint8_t *v_cur, const PfAddr<D> &ad,
                       bool masked, int k1, int lane, const PfLogit &lg, IssueCopies &&issue_copies) {
    using G = PfGeom<D>;
    constexpr int NM = G::NM;  // MFMAs per block
    // scores that need no f32 scaling or terms start from -m_run in the MFMA: no shift
    constexpr bool CM = !G::QRAW && !LOGIT;
    if constexpr (CM) pf_qk<F16, D>(nxt, st, k_next, ad, st.negv);
    else pf_qk<F16, D>(nxt, st, k_next, ad, f32x16{});
    pf_exp<F16, G::MB>(pop, cur);
    pf_block_schedule<G::V1, 0, NM>();
    __builtin_amdgcn_sched_barrier(0);
    // P(t) is used only after the branch below: pin its computation to block 1
#pragma unroll
    for (int i = 0; i < 2 * G::MB; ++i) asm volatile("" ::"v"(pop[i]));
    if (LOGIT) {
        if constexpr (G::QRAW) pf_scale<G::MB>(nxt, st.c2);
        pf_logit<G::MB>(nxt, lg, k1, lane);
    }
    // (unscaled scores of the QRAW form take the mask value that their scaling turns into -inf)
    if (masked) pf_mask(nxt, st, k1, lane, G::QRAW && !LOGIT ? st.mraw : -__builtin_inff());
    issue_copies();
    pf_pv<F16, D>(st, pop, v_cur, ad);
    pf_psum<F16, D>(st, pop);
    if (G::QRAW && !LOGIT) pf_shift_scaled<G::MB>(nxt, st.c2, st.negm);
    else if (!CM) pf_shift<G::MB>(nxt, st.negm);
    float mx = pf_rowmax<G::MB>(nxt);
    pf_block_schedule<CM ? G::V2C : G::V2, G::CP, NM>();
    __builtin_amdgcn_sched_barrier(0);
    mx = pf_max_halves(mx);
    const bool need = mx > st.thr;
    if (__builtin_expect(__any(need), 0)) pf_rescale(nxt, st, mx, need);
}

// The last key tile: P(t) and O += V(t)^T P(t).
template <bool F16, int D, uint32_t BIAS = PfGeom<D>::VBIAS>
PF_INLINE void pf_last_tile(const f32x16 *cur, u32x4 *pop, PfState<D> &st,
                            const uint8_t *v_cur, const PfAddr<D> &ad) {
    pf_exp<F16, PfGeom<D>::MB>(pop, cur);
    pf_pv<F16, D, BIAS>(st, pop, v_cur, ad);
    pf_psum<F16, D>(st, pop);
    pf_block_schedule<(D == 256 ? PfGeom<D>::V1 : 128 / D), 0, PfGeom<D>::NM>();
}

}  // namespace cqkv
