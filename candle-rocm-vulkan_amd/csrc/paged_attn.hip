// Host side of the attention over a page pool (cqkv_paged_attention) and the merge of its key splits.
#include "paged_chunk.h"

#include <algorithm>

namespace cqkv {

// Merge of the pieces: o = sum_s w_s o_s / sum_s w_s, w_s = 2^(lse_s - max lse). A row outside every
// sequence, past max_q of its sequence, or written whole by its only workgroup is left alone.
//
// Bound by latency: the row's sequence and its slots have to be found, then its pieces. D / 4 lanes take a row, so a wavefront has 256 / D heads of a token at once. Few rows (DEEP): a
// workgroup for them, its 8 wavefronts taking the pieces 8 at a time. Many rows: a wavefront takes `per`
// such groups of a token, so the sequence is found once for them, two in flight. 256 rows of up to 20 pieces:
// 4.9 us (a wavefront per row 21); 33472 rows of 2: 13 us (33).
template <int D, bool DEEP>
__global__ __launch_bounds__(DEEP ? 512 : 256) void paged_combine_kernel(PagedAttnArgs a, int out_f16, int per) {
    constexpr int LPR = D / 4, RW = 64 / LPR, NG = DEEP ? 1 : 2, NP = DEEP ? 8 : 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int idx = DEEP ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
    const int groups = (a.q_heads + RW - 1) / RW, runs = (groups + per - 1) / per;
    const int token = idx / runs, g0 = (idx - token * runs) * per, g1 = min(g0 + per, groups);
    if (token >= a.pt.total) return;
    // the sequence, and the slots in front of its; sequences in steps of 64, whose loads are independent
    const int batch = a.pt.batch;
    int b = -1;
    uint64_t tiles = 0;
#pragma unroll 4
    for (int i = lane; i < batch; i += 64) {
        const PagedSeq ls = paged_seq_lane(a, i);
        if (token >= ls.first && token < ls.first + ls.lq) b = i;
        tiles += (uint32_t)max(seq_tiles(a, ls), 0);
    }
    const uint64_t at_lane = __ballot(b >= 0);
    if (!at_lane) return;
    b = __builtin_amdgcn_readlane(b, __builtin_ctzll(at_lane));
    uint32_t u = 0x40000000u;
    uint64_t slots = 0;
    if (a.parts) {
        u = piece_tiles(a, tiles, lane);
#pragma unroll 4
        for (int i = lane; i < b; i += 64) slots += seq_pieces(a, seq_work(a, paged_seq_lane(a, i), u)) >> 32;
        slots = readlane64(wave_scan2(slots, lane), 63);
    }
    const PagedSeq sq = paged_seq(a, b);
    const int qi = token - sq.first;
    if (qi >= min(sq.lq, a.max_q)) return;
    const bool chunk = chunk_takes(a, sq);
    const int np = chunk ? chunk_splits(a, sq) : seq_work(a, sq, u).pieces;
    if (np < 2) return;
    const float *pl = chunk ? a.chunk_lse : a.part_lse, *po = chunk ? a.chunk_o : a.part_o;
    const int64_t step = chunk ? (int64_t)a.pt.total * a.q_heads : (int64_t)a.kv_heads * a.slot_cols;
    const int d0 = 4 * (lane % LPR);
    for (int gg = g0; gg < g1; gg += NG) {
        float M[NG], wsum[NG];
        f32x4 acc[NG];
        int head[NG];
        int64_t at[NG];  // piece s: row at + s * step of the partials
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            M[i] = -__builtin_inff();
            wsum[i] = 0.0f;
            acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            head[i] = min(min(gg + i, g1 - 1) * RW + lane / LPR, a.q_heads - 1);
            const int hk = pf_div_group(head[i], a.group, a.group_m);
            at[i] = chunk ? (int64_t)token * a.q_heads + head[i]
                          : (int64_t)(slots + (uint32_t)hk) * a.slot_cols + qi * a.group + (head[i] - hk * a.group);
        }
        for (int s0 = DEEP ? NP * wave : 0; s0 < np; s0 += DEEP ? 8 * NP : NP) {
            float e[NG][NP];
            f32x4 v[NG][NP];
#pragma unroll
            for (int i = 0; i < NG; ++i)
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int64_t row = at[i] + min(s0 + j, np - 1) * step;
                    e[i][j] = pl[row];
                    v[i][j] = *(const f32x4 *)(po + row * D + d0);
                }
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                float mx = M[i];
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    if (s0 + j >= np) e[i][j] = -__builtin_inff();
                    mx = fmaxf(mx, e[i][j]);
                }
                const float f = M[i] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(M[i] - mx);
                acc[i] *= f;
                wsum[i] *= f;
                M[i] = mx;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    // (a piece without a visible key, or too small to count, adds nothing; NaN is kept)
                    const float w = e[i][j] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(e[i][j] - mx);
                    wsum[i] += w;
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][c] += w == 0.0f ? 0.0f : w * v[i][j][c];
                }
            }
        }
        if constexpr (DEEP) {
            __shared__ f32x4 sm_acc[8][64];
            __shared__ float sm_m[8][64], sm_w[8][64];
            sm_acc[wave][lane] = acc[0];
            sm_m[wave][lane] = M[0];
            sm_w[wave][lane] = wsum[0];
            __syncthreads();
            if (wave) return;
            for (int w = 1; w < 8; ++w) M[0] = fmaxf(M[0], sm_m[w][lane]);
            acc[0] = f32x4{0.f, 0.f, 0.f, 0.f};
            wsum[0] = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const float l = sm_w[w][lane], f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sm_m[w][lane] - M[0]);
                const f32x4 v = sm_acc[w][lane];
                wsum[0] += l * f;
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[0][c] += f == 0.0f ? 0.0f : v[c] * f;
            }
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (gg + i >= g1 || (gg + i) * RW + lane / LPR >= a.q_heads) continue;
            const int64_t out = (int64_t)token * a.o_st + (int64_t)head[i] * a.o_sh + d0;
            f32x4 o;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = wsum[i] == 0.0f ? 0.0f : acc[i][c] / wsum[i];
            if (a.o_vec) {
                if (d0 < a.dim) {
                    u32x2 w;
                    if (out_f16) w = u32x2{pack_f16x2(o.x, o.y), pack_f16x2(o.z, o.w)};
                    else w = u32x2{pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w)};
                    *(u32x2 *)((uint16_t *)a.out + out) = w;
                }
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (d0 + c < a.dim) store_elem(a.out, out + c, out_f16 ? CQKV_F16 : CQKV_BF16, o[c]);
            }
        }
    }
}

static int paged_cus() {
    constexpr int kMaxDev = 64;
    static int cache[kMaxDev];
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDev) {
        (void)hipGetLastError();
        return 256;
    }
    if (!cache[dev]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) {
            (void)hipGetLastError();
            n = 256;
        }
        cache[dev] = n;
    }
    return cache[dev];
}

// The launches of a call. Sequences of at most `from` columns per kv head take the decode kernel, longer
// ones the chunk kernel.
struct PagedPlan {
    int parts, slot_cols;
    bool once;  // a tile is read by one wavefront in most sequences of the decode kernel
    int from, chunk_blocks, chunk_splits, chunk_tps, chunk_bk;
    size_t part_lse, chunk_o, chunk_lse, total;  // workspace offsets and size
};
static PagedPlan paged_plan(int32_t d, int32_t batch, int32_t total, int32_t q_heads, int32_t kv_heads, int32_t max_q,
                            int32_t max_kv, int32_t wl, int32_t wr) {
    PagedPlan p = {};
    const int dk = kernel_dim(d), group = q_heads / kv_heads;
    const int64_t cols = (int64_t)max_q * group, cus = paged_cus();
    // keys that a sequence's queries may see: the window's and the chunk's
    int64_t keys = max_kv;
    if (wl >= 0 && wr >= 0) keys = std::min<int64_t>(keys, (int64_t)wl + max_q + wr);
    // three blocks of 16 columns, four at D = 256 (16 sequences, FP8, bf16: D = 128, 4K keys, 32 columns 55 us
    // against the chunk kernel's 78, 48 columns 81 and 82, 64 columns 88 and 72; D = 256, up to 8K keys, 64
    // columns 99 and 107)
    p.from = dk == 256 ? 64 : 48;
    const bool many = cols > p.from;
    // (next to a long sequence: the tokens that the others have on average)
    const int64_t others = batch > 1 ? (std::max(total - max_q, 1) + batch - 2) / (batch - 1) : 1;
    p.once = (many ? others * group : cols) <= 16;
    if (many && batch == 1) p.from = 0;  // the one sequence: no launch for short ones
    const int64_t rows = (int64_t)total * q_heads;
    size_t at = 0;
    const auto take = [&](int64_t floats) {
        const size_t o = at;
        at += ((size_t)floats * 4 + 255) & ~(size_t)255;
        return o;
    };
    p.slot_cols = (int)((std::min<int64_t>(cols, p.from) + 15) / 16 * 16);
    if (keys > 32 * kPieceTiles && p.from) {
        // One round of the chip's workgroups where the planes leave most of them to cut with (4 sequences of up to
        // 128K keys, MXFP4, 64 / 8 heads, 32 planes of 512 workgroups: 87 us; two rounds 114), else three, whose
        // last is short (64 sequences of up to 8K keys, FP8, 32 / 8 heads, 512 planes: 137 us; longer pieces 151).
        // Half long and half short sequences: 192 planes 53 and 56 us, 256 planes 84 and 68.
        const int64_t slots = cus * (dk < 256 ? 2 : 1), planes = (int64_t)batch * kv_heads;
        p.parts = (int)(8 * planes <= 3 * slots ? slots - planes : 3 * slots);
        // slots: at most 2 parts, and one more than the parts for every plane
        const int64_t cut = std::min<int64_t>(2 * p.parts, p.parts + planes);
        take(cut * p.slot_cols * dk);
        p.part_lse = take(cut * p.slot_cols);
    }
    p.chunk_bk = dk == 256 ? 32 : 64;
    if (many) {
        // column blocks: those that sequences of more than `from` columns may fill (the launch), and those
        // that they fill if max_q is the longest one's length (the splits)
        const int64_t all = (int64_t)total * group;
        const int nc = 32 * chunk_waves(dk);
        p.chunk_blocks = (int)std::min<int64_t>(all / nc + std::min<int64_t>(batch, all / (p.from + 1)), 1 << 24);
        const int64_t rest = std::max<int64_t>(all - cols, 0);
        const int64_t blocks = ((cols + nc - 1) / nc + (rest + nc - 1) / nc * (rest > (int64_t)p.from * (batch - 1))) * kv_heads;
        // as many splits as end soonest: rounds of the chip over the length of a split, and what its partials
        // cost to write and merge, in tiles (64 keys of 256 columns take about 0.5 us, 4 MB at 8 TB/s)
        const int64_t ct = (keys + p.chunk_bk - 1) / p.chunk_bk + 1, slots = cus;
        int best = 1;
        double cost = 1e30;
        for (int cs = 1; cs <= 16 && (cs == 1 || ct / cs >= 8); ++cs) {
            const double merge = cs > 1 ? (double)blocks * cs * nc * dk * 8 / 4e6 : 0.0;
            const double c = (double)((blocks * cs + slots - 1) / slots) * ((double)ct / cs + 4.0) + merge;
            if (c < cost * 0.97) {
                best = cs;
                cost = c;
            }
        }
        p.chunk_tps = (int)((ct + best - 1) / best);
        p.chunk_splits = (int)((ct + p.chunk_tps - 1) / p.chunk_tps);
        if (p.chunk_splits > 1) {
            p.chunk_o = take(p.chunk_splits * rows * dk);
            p.chunk_lse = take(p.chunk_splits * rows);
        }
    }
    p.total = at;
    return p;
}

}  // namespace cqkv

using namespace cqkv;

extern "C" size_t cqkv_paged_attention_workspace_bytes(const cqkv_side *k_side, int32_t batch,
                                                       int32_t total, int32_t q_heads,
                                                       int32_t max_q_len, int32_t max_kv_len,
                                                       int32_t window_left, int32_t window_right) {
    clear_error();
    if (check_side(k_side, "cqkv_paged_attention_workspace_bytes") != CQKV_OK || batch <= 0 ||
        total <= 0 || q_heads <= 0 || q_heads % k_side->kv_heads || max_q_len <= 0 || max_kv_len <= 0)
        return 0;
    return paged_plan(k_side->head_dim, batch, total, q_heads, k_side->kv_heads, max_q_len, max_kv_len,
                      window_left, window_right)
        .total;
}

extern "C" int cqkv_paged_attention(const void *q, const int64_t q_strides[2], int32_t dtype,
                                    const cqkv_side *k_side, const cqkv_side *v_side,
                                    const cqkv_pages *pages, const int32_t *kv_lens, int32_t total,
                                    int32_t q_heads, int32_t max_q_len, int32_t max_kv_len,
                                    float softmax_scale, int32_t window_left, int32_t window_right,
                                    float softcap, const float *alibi_slopes,
                                    int32_t alibi_batch_stride, void *out,
                                    const int64_t out_strides[2], void *workspace,
                                    size_t workspace_bytes, cqkv_stream_t stream) {
    clear_error();
    static const char *who = "cqkv_paged_attention";
    PagedAttnArgs a = {};
    if (!k_side || !v_side) return fail(CQKV_ERR_ARG, "%s: null side", who);
    if (int rc = check_pool(who, k_side, v_side, pages, total, &a.pt)) return rc;
    if (dtype != CQKV_BF16 && dtype != CQKV_F16)
        return fail(CQKV_ERR_ARG, "%s: dtype %d (bf16 or f16 queries)", who, dtype);
    const int hkv = k_side->kv_heads, d = k_side->head_dim;
    if (q_heads <= 0 || q_heads % hkv != 0)
        return fail(CQKV_ERR_ARG, "%s: q_heads %d kv_heads %d", who, q_heads, hkv);
    if (max_q_len < 0 || max_kv_len < 0)
        return fail(CQKV_ERR_ARG, "%s: max_q_len %d max_kv_len %d", who, max_q_len, max_kv_len);
    if (max_kv_len > 1 << 30) return fail(CQKV_ERR_ARG, "%s: max_kv_len %d above 2^30", who, max_kv_len);
    if (!(softcap >= 0.0f) || softcap == __builtin_inff())
        return fail(CQKV_ERR_ARG, "%s: softcap %g (finite, >= 0; 0 disables it)", who, (double)softcap);
    if (alibi_slopes && alibi_batch_stride != 0 && alibi_batch_stride != q_heads)
        return fail(CQKV_ERR_ARG, "%s: alibi batch stride %d (0 or q_heads %d)", who, alibi_batch_stride, q_heads);
    if ((int64_t)max_q_len * (q_heads / hkv) > 1 << 24)
        return fail(CQKV_ERR_ARG, "%s: max_q_len * q_heads / kv_heads = %lld above 2^24", who,
                    (long long)max_q_len * (q_heads / hkv));
    if (total == 0 || pages->batch == 0 || max_q_len == 0) return CQKV_OK;
    if (!q || !out || !q_strides || !out_strides || !kv_lens)
        return fail(CQKV_ERR_ARG, "%s: null pointer argument", who);
    a.k = pool_side(k_side);
    a.v = pool_side(v_side);
    a.q = q;
    a.out = out;
    a.q_st = q_strides[0];
    a.q_sh = q_strides[1];
    a.o_st = out_strides[0];
    a.o_sh = out_strides[1];
    a.kv_lens = kv_lens;
    a.max_q = max_q_len;
    a.max_kv = max_kv_len;
    a.kv_heads = hkv;
    a.q_heads = q_heads;
    a.group = q_heads / hkv;
    a.group_m = pf_group_m(a.group);
    a.dim = d;
    a.o_vec = d % 4 == 0 && (uintptr_t)out % 8 == 0 && a.o_st % 4 == 0 && a.o_sh % 4 == 0;
    a.q_vec = d % 8 == 0 && (uintptr_t)q % 16 == 0 && a.q_st % 8 == 0 && a.q_sh % 8 == 0;
    // (windows past every position, so that sums with positions stay in 32 bits)
    a.wl = std::min(window_left, 1 << 30);
    a.wr = std::min(window_right, (1 << 30) - 1);
    a.scale_log2 = softmax_scale * kLog2e;
    a.cap2 = softcap * kLog2e;
    a.alibi = alibi_slopes;
    a.alibi_bs = alibi_batch_stride;
    const PagedPlan p = paged_plan(d, pages->batch, total, q_heads, hkv, max_q_len, max_kv_len, window_left,
                                   window_right);
    a.parts = p.parts;
    a.slot_cols = p.slot_cols;
    a.chunk_from = p.from;
    a.chunk_blocks = p.chunk_blocks;
    a.chunk_splits = p.chunk_splits;
    a.chunk_tps = p.chunk_tps;
    a.chunk_bk = p.chunk_bk;
    const int64_t wgs = p.from ? p.parts + (int64_t)pages->batch * hkv : 0;
    const int64_t kgs = (int64_t)p.chunk_splits * p.chunk_blocks * hkv;
    // the merge: head groups of a token, few with a workgroup each, many in runs that make 4096 wavefronts
    const int64_t groups = (q_heads * kernel_dim(d) + 255) / 256;
    const bool deep = total * groups <= 512;
    const int per = deep ? 1 : (int)std::clamp<int64_t>(total * groups / 4096, 1, 8);
    const int64_t runs = total * ((groups + per - 1) / per), cgs = deep ? runs : (runs + 3) / 4;
    if (wgs > 0x7fffffffll / 512 || cgs > 0x7fffffffll / 256 || runs > 0x7fffffffll - 4 || kgs > 0x7fffffffll / 512)
        return fail(CQKV_ERR_ARG, "%s: %lld workgroups exceed one launch", who, (long long)std::max({wgs, cgs, kgs}));
    hipStream_t st = (hipStream_t)stream;
    void *ws = workspace;
    bool owned = false;
    if (p.total) {
        if (ws && workspace_bytes < p.total)
            return fail(CQKV_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, p.total);
        if ((uintptr_t)ws % 16) return fail(CQKV_ERR_ARG, "%s: workspace not 16-byte aligned", who);
        if (!ws) {
            CQKV_HIP_CHECK(hipMallocAsync(&ws, p.total, st));
            owned = true;
        }
        a.part_o = (float *)ws;
        a.part_lse = (float *)((char *)ws + p.part_lse);
        a.chunk_o = (float *)((char *)ws + p.chunk_o);
        a.chunk_lse = (float *)((char *)ws + p.chunk_lse);
    }
    const int dk = kernel_dim(d);
    const bool f16 = dtype == CQKV_F16;
    const bool logit = a.cap2 > 0.0f || a.alibi;
    hipError_t e = hipSuccess;
    if (kgs) {  // the long sequences first: they take longest
        const dim3 grid((unsigned)kgs);
        if (k_side->format == CQKV_FMT_FP8) paged_chunk_launch_5(dk, f16, logit, grid, st, a);
        else if (k_side->format == CQKV_FMT_MXFP8) paged_chunk_launch_4(dk, f16, logit, grid, st, a);
        else paged_chunk_launch_2(dk, f16, logit, grid, st, a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && wgs) {
        const dim3 grid((unsigned)wgs);
        if (k_side->format == CQKV_FMT_FP8) paged_attn_launch_5(dk, f16, p.once, grid, st, a);
        else if (k_side->format == CQKV_FMT_MXFP8) paged_attn_launch_4(dk, f16, p.once, grid, st, a);
        else paged_attn_launch_2(dk, f16, p.once, grid, st, a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && p.total) {
#define CQKV_COMBINE(D)                                                                                           \
    if (deep) hipLaunchKernelGGL((paged_combine_kernel<D, true>), dim3(cgs), dim3(512), 0, st, a, (int)f16, per); \
    else hipLaunchKernelGGL((paged_combine_kernel<D, false>), dim3(cgs), dim3(256), 0, st, a, (int)f16, per)
        if (dk == 64) {
            CQKV_COMBINE(64);
        } else if (dk == 128) {
            CQKV_COMBINE(128);
        } else {
            CQKV_COMBINE(256);
        }
#undef CQKV_COMBINE
        e = hipGetLastError();
    }
    if (owned) {
        const hipError_t fe = hipFreeAsync(ws, st);
        if (e == hipSuccess) e = fe;
    }
    if (e != hipSuccess) return fail(CQKV_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
    return CQKV_OK;
}
