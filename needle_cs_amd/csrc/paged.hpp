// paged.hpp -- what the paged cache's kernels share: the cache as kernels see
// it, the checks of a caller's nhip_paged_cache, and one layer's pools.
#pragma once

#include "common.hpp"

namespace nhip {

// Checks a caller's cache (sizes, pointers, alignment); NHIP_OK or NHIP_ERR_ARG.
int32_t paged_check(const nhip_paged_cache* c);

constexpr int32_t kPagedMaxRows = 1 << 20;  // of a call

// One layer of a cache, for the kernels that read or write positions.
struct PagedLayer {
    int8_t* keys;         // [pages][kv_heads][page_size][qk]
    float* kscale;        // [pages][kv_heads][page_size]
    int8_t* values;       // [pages][kv_heads][page_size/16][v][16]
    float* vscale;
    const int32_t* tables;
    int32_t pages, page_shift, kv_heads, qk, v, sequences, width;
};

inline PagedLayer paged_layer(const nhip_paged_cache* c, int32_t layer)
{
    const size_t cells = (size_t)layer * c->pages * c->kv_heads * c->page_size;
    return {c->keys + cells * c->qk_dim,
            c->key_scales + cells,
            c->values + cells * c->v_dim,
            c->value_scales + cells,
            c->tables,
            c->pages,
            __builtin_ctz((unsigned)c->page_size),
            c->kv_heads,
            c->qk_dim,
            c->v_dim,
            c->sequences,
            c->width};
}

}  // namespace nhip
