// Host side of the attention over a page pool (cqkv_paged_attention) and the merge of its key splits.
#include "paged_chunk.h"

#include <algorithm>

namespace cqkv {

// Merge of the splits: o = sum_s w_s o_s / sum_s w_s, w_s = 2^(lse_s - max lse). One wavefront per row
// (packed token, query head); a row outside every sequence, past max_q of its sequence, or of a
// sequence in one split (written by its only workgroup) is left alone. The row's sequence is the number
// of prefix sums at or below it, counted 64 at a time.
template <int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttnArgs a, int out_f16) {
    constexpr int NP = D == 256 ? 2 : 1;  // element pairs per lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * 4 + wave, rows = (int64_t)a.pt.total * a.q_heads;
    if (row >= rows) return;
    const int token = (int)(row / a.q_heads), head = (int)(row % a.q_heads);
    int b = -1;
    for (int base = 0; base <= a.pt.batch; base += 64) {
        const bool at = base + lane <= a.pt.batch && min(max(a.pt.cu[base + lane], 0), a.pt.total) <= token;
        const uint64_t m = __ballot(at);
        b += __builtin_popcountll(m);
        if (m != ~0ull) break;
    }
    if (b < 0 || b >= a.pt.batch) return;
    const PagedSeq sq = paged_seq(a, b);
    const int qi = token - sq.first, ns = chunk_takes(a, sq) ? chunk_splits(a, sq) : paged_splits(a, sq);
    if (qi < 0 || qi >= min(sq.lq, a.max_q) || ns < 2) return;
    const bool active = lane < D / 2 / NP;
    const float *lse = a.part_lse + row;
    float M = -__builtin_inff();
    for (int s = lane; s < ns; s += 64) M = fmaxf(M, lse[s * rows]);
    M = wave_max(M);
    float wsum = 0.0f, acc[2 * NP] = {};
    const float *po = a.part_o + row * D + 2 * (active ? lane : 0);
    const int64_t step = rows * D;
    for (int s0 = 0; s0 < ns; s0 += 64) {
        const int nn = min(ns - s0, 64);
        const float e = lane < nn ? lse[(s0 + lane) * rows] : -__builtin_inff();
        const float w = e == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(e - M);
        for (int s1 = 0; s1 < nn; s1 += 8) {
            f32x2 v[8][NP];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    v[i][p] = *(const f32x2 *)(po + (s0 + min(s1 + i, nn - 1)) * step + 128 * p);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (s1 + i >= nn) break;
                const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s1 + i));
                if (ws == 0.0f) continue;
                wsum += ws;
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    acc[2 * p] += ws * v[i][p].x;
                    acc[2 * p + 1] += ws * v[i][p].y;
                }
            }
        }
    }
    if (!active) return;
    const int64_t at = (int64_t)token * a.o_st + (int64_t)head * a.o_sh;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = 128 * p + 2 * lane + e;
            const float o = wsum == 0.0f ? 0.0f : acc[2 * p + e] / wsum;
            if (j < a.dim) store_elem(a.out, at + j, out_f16 ? CQKV_F16 : CQKV_BF16, o);
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

// The launches of a call. Sequences of at most `from` columns per kv head take the decode kernel (nb
// column blocks of 16 per workgroup), longer ones the chunk kernel.
struct PagedPlan {
    int nb, col_blocks, splits, tps;
    int from, waves, chunk_blocks, chunk_splits, chunk_tps, chunk_bk;
    size_t lse, total;  // workspace offsets
};
static PagedPlan paged_plan(int32_t format, int32_t d, int32_t batch, int32_t total, int32_t q_heads,
                            int32_t kv_heads, int32_t max_q, int32_t max_kv, int32_t wl, int32_t wr) {
    PagedPlan p = {};
    const int dk = kernel_dim(d), group = q_heads / kv_heads;
    const int64_t cols = (int64_t)max_q * group;
    p.from = dk == 256 ? 16 : 64;
    // the decode kernel's columns (the long sequences of the call are not its)
    const int64_t few = std::min<int64_t>(cols, p.from / group * group);
    p.nb = few <= 16 ? 1 : few <= 32 ? 2 : 4;
    p.col_blocks = (int)((few + 16 * p.nb - 1) / (16 * p.nb));
    // keys that a sequence's queries may see: the window's and the chunk's
    int64_t keys = max_kv;
    if (wl >= 0) keys = std::min<int64_t>(keys, (int64_t)wl + max_q + std::max(wr, 0));
    const int64_t tiles = (keys + 31) / 32 + 1;
    const int wv = p.nb == 1 && format != CQKV_FMT_MXFP4 && dk < 256 ? 8 : 4;
    // as many workgroups as fill the chip (one of 8 wavefronts per CU, or two of 4), pieces of at
    // least two tiles per wavefront, and of at most 128 tiles, so that sequences of different
    // lengths even out
    const int64_t cus = paged_cus();
    const int64_t wgs = cus * (8 / wv), planes = (int64_t)batch * kv_heads * p.col_blocks;
    int64_t s = std::max<int64_t>((wgs + planes - 1) / std::max<int64_t>(planes, 1), batch > 1 ? (tiles + 127) / 128 : 1);
    s = std::min(s, std::max<int64_t>(1, tiles / (2 * wv)));
    s = std::max<int64_t>(1, std::min<int64_t>(s, 256));
    p.tps = (int)((tiles + s - 1) / s);
    p.splits = (int)((tiles + p.tps - 1) / p.tps);
    p.chunk_bk = dk == 256 ? 32 : 64;
    if (cols > p.from) {
        // sequences that may have more than `from` columns, and the column blocks they may fill
        const int64_t all = (int64_t)total * group;
        p.waves = dk == 256 || cols <= 128 ? 4 : 8;
        const int64_t nseq = std::min<int64_t>(batch, all / (p.from + 1));
        p.chunk_blocks = (int)std::min<int64_t>(all / (32 * p.waves) + nseq, 1 << 24);
        const int64_t ct = (keys + p.chunk_bk - 1) / p.chunk_bk + 1;
        const int64_t blocks = std::max<int64_t>((int64_t)p.chunk_blocks * kv_heads, 1);
        int64_t cs = (cus * (8 / p.waves) + blocks - 1) / blocks;
        cs = std::max<int64_t>(1, std::min<int64_t>({cs, ct / 8, 32}));
        p.chunk_tps = (int)((ct + cs - 1) / cs);
        p.chunk_splits = (int)((ct + p.chunk_tps - 1) / p.chunk_tps);
    }
    const size_t rows = (size_t)total * q_heads, most = (size_t)std::max(p.splits, p.chunk_splits);
    if (most > 1) {
        p.lse = (most * rows * dk * 4 + 255) & ~(size_t)255;
        p.total = p.lse + ((most * rows * 4 + 255) & ~(size_t)255);
    }
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
    return paged_plan(k_side->format, k_side->head_dim, batch, total, q_heads, k_side->kv_heads, max_q_len,
                      max_kv_len, window_left, window_right)
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
    a.wl = window_left;
    a.wr = window_right;
    a.scale_log2 = softmax_scale * kLog2e;
    a.cap2 = softcap * kLog2e;
    a.alibi = alibi_slopes;
    a.alibi_bs = alibi_batch_stride;
    const PagedPlan p = paged_plan(k_side->format, d, pages->batch, total, q_heads, hkv, max_q_len, max_kv_len, window_left,
                                   window_right);
    a.splits = p.splits;
    a.tps = p.tps;
    a.col_blocks = p.col_blocks;
    a.chunk_from = p.from;
    a.chunk_blocks = p.chunk_blocks;
    a.chunk_splits = p.chunk_splits;
    a.chunk_tps = p.chunk_tps;
    a.chunk_bk = p.chunk_bk;
    // a call whose only sequence is the chunk kernel's has nothing for the decode kernel (a shorter one
    // than max_q_len says still would: then its columns are counted on the device, so both run)
    const bool few = p.chunk_blocks == 0 || pages->batch > 1 || total < max_q_len || (int64_t)total * a.group <= p.from;
    const int64_t wgs = few ? (int64_t)p.splits * p.col_blocks * pages->batch * hkv : 0;
    const int64_t kgs = (int64_t)p.chunk_splits * p.chunk_blocks * hkv;
    const int64_t cgs = ((int64_t)total * q_heads + 3) / 4;
    if (wgs > 0x7fffffffll / 512 || cgs > 0x7fffffffll / 256 || kgs > 0x7fffffffll / 512)
        return fail(CQKV_ERR_ARG, "%s: %lld workgroups exceed one launch", who, (long long)std::max({wgs, cgs, kgs}));
    hipStream_t st = (hipStream_t)stream;
    void *ws = workspace;
    bool owned = false;
    if (p.total) {
        if (ws && workspace_bytes < p.total)
            return fail(CQKV_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, p.total);
        if (!ws) {
            CQKV_HIP_CHECK(hipMallocAsync(&ws, p.total, st));
            owned = true;
        }
        a.part_o = (float *)ws;
        a.part_lse = (float *)((char *)ws + p.lse);
    }
    const int dk = kernel_dim(d);
    const bool f16 = dtype == CQKV_F16;
    const bool logit = a.cap2 > 0.0f || a.alibi;
    hipError_t e = hipSuccess;
    if (kgs) {  // the long sequences first: they take longest
        const dim3 grid((unsigned)kgs);
        if (k_side->format == CQKV_FMT_FP8) paged_chunk_launch_5(dk, p.waves, f16, logit, grid, st, a);
        else if (k_side->format == CQKV_FMT_MXFP8) paged_chunk_launch_4(dk, p.waves, f16, logit, grid, st, a);
        else paged_chunk_launch_2(dk, p.waves, f16, logit, grid, st, a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && wgs) {
        const dim3 grid((unsigned)wgs);
        if (k_side->format == CQKV_FMT_FP8) paged_attn_launch_5(dk, p.nb, f16, grid, st, a);
        else if (k_side->format == CQKV_FMT_MXFP8) paged_attn_launch_4(dk, p.nb, f16, grid, st, a);
        else paged_attn_launch_2(dk, p.nb, f16, grid, st, a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && p.total) {
        const dim3 cg((unsigned)cgs);
        if (dk == 64) hipLaunchKernelGGL(paged_combine_kernel<64>, cg, dim3(256), 0, st, a, (int)f16);
        else if (dk == 128) hipLaunchKernelGGL(paged_combine_kernel<128>, cg, dim3(256), 0, st, a, (int)f16);
        else hipLaunchKernelGGL(paged_combine_kernel<256>, cg, dim3(256), 0, st, a, (int)f16);
        e = hipGetLastError();
    }
    if (owned) {
        const hipError_t fe = hipFreeAsync(ws, st);
        if (e == hipSuccess) e = fe;
    }
    if (e != hipSuccess) return fail(CQKV_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
    return CQKV_OK;
}
