// One format's instantiations of the page pool kernels (compiled once per format with
// -DCQKV_PAGED_FMT=<format id>, so the formats build in parallel).
#include "paged_chunk.h"
#include "paged_rows.h"

#ifndef CQKV_PAGED_FMT
#error "compile with -DCQKV_PAGED_FMT=<format id>"
#endif

#define CQKV_CAT2(a, b) a##b
#define CQKV_CAT(a, b) CQKV_CAT2(a, b)

namespace cqkv {

void CQKV_CAT(paged_append_launch_, CQKV_PAGED_FMT)(int dk, int rope, dim3 grid, hipStream_t st,
                                                   const PagedRowsArgs &a) {
    launch_append_dim<CQKV_PAGED_FMT>(dk, rope, grid, st, a);
}

void CQKV_CAT(paged_dequant_launch_, CQKV_PAGED_FMT)(int dk, dim3 grid, hipStream_t st,
                                                    const PagedRowsArgs &a) {
    launch_dequant<CQKV_PAGED_FMT>(dk, grid, st, a);
}

void CQKV_CAT(paged_attn_launch_, CQKV_PAGED_FMT)(int dk, bool f16, bool once, dim3 grid, hipStream_t st,
                                                 const PagedAttnArgs &a) {
    launch_paged_attn<CQKV_PAGED_FMT>(dk, f16, once, grid, st, a);
}

void CQKV_CAT(paged_chunk_launch_, CQKV_PAGED_FMT)(int dk, bool f16, bool logit, dim3 grid,
                                                  hipStream_t st, const PagedAttnArgs &a) {
    launch_paged_chunk<CQKV_PAGED_FMT>(dk, f16, logit, grid, st, a);
}

}  // namespace cqkv
