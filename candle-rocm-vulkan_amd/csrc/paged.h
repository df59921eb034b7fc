// The page pool shared by the paged entry points (paged_rows.hip, paged_attn.hip): a pair of cache
// sides whose planes are (page, kv head), a page table per sequence, and packed token rows.
#pragma once

#include "cqkv_device.h"
#include "cqkv_host.h"

namespace cqkv {

typedef __attribute__((address_space(4))) const int32_t scalar_i32;  // wavefront-uniform loads

// Page table of the call. A page holds 2^shift tokens, so a position's page and row are a shift and
// a mask. Page ids outside [0, n_pages) are holes.
struct PageTable {
    const int32_t *table;
    int64_t stride;
    const int32_t *cu;  // batch + 1 first rows of the sequences
    int32_t max_pages, n_pages, batch, shift, total;
};

// Plane bytes and format of one side of the pool.
struct PoolSide {
    uint8_t *codes, *scales;
    uint32_t codes_plane, scales_plane;
};

inline PoolSide pool_side(const cqkv_side *s) {
    PoolSide p;
    p.codes = (uint8_t *)s->codes;
    p.scales = (uint8_t *)s->scales;
    p.codes_plane = (uint32_t)cqkv_codes_plane_bytes(s->format, s->head_dim, s->capacity);
    p.scales_plane = (uint32_t)cqkv_scales_plane_bytes(s->format, s->head_dim, s->capacity);
    return p;
}

// Checks a pool's sides (v null: one side alone) and its page table, and fills `p`.
int check_pool(const char *who, const cqkv_side *k, const cqkv_side *v, const cqkv_pages *pages,
               int32_t total, PageTable *p);

}  // namespace cqkv
