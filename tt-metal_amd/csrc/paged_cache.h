// What the kernels of the paged key/value cache share: the shapes that a call names, and where elements lie.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ttmi.h"

namespace ttmi {

// bf16 activations [tokens, width], dense rows or TILE layout (the rows up to a multiple of 32 exist there, and are not read)
struct PagedRows { const void *data; int layout; uint32_t tokens, width; };
// the keys or the values: [pages, kv_heads, page_size, head_dim] in TILE layout, dtype BFLOAT16 or BFLOAT8_B
struct PagedCache { int dtype; uint32_t pages, kv_heads, page_size, head_dim; };
// what the requests of a step look like on the device
struct PagedStep { const int32_t *page_table; uint32_t requests, max_pages; const int32_t *cached, *row_starts; };

// most requests of one step: the prefix sums over them lie in LDS
constexpr uint32_t PAGED_MAX_REQUESTS = 4096;

// Byte at which 8 neighbouring elements of row t start (column a multiple of 8).  `width` is the row's length in elements, in TILE
// layout a multiple of 32.
__host__ __device__ __forceinline__ uint64_t row_bytes_at(uint32_t t, uint32_t width, uint32_t column, int tiled) {
    if (!tiled) return ((uint64_t)t * width + column) * 2;
    const uint64_t tile = (uint64_t)(t >> 5) * (width >> 5) + (column >> 5);
    return tile * 2048 + ((t >> 4 & 1) * 2 + (column >> 4 & 1)) * 512 + (t & 15) * 32 + (column & 15) * 2;
}

int paged_tables(const int32_t *cached, const int32_t *added, uint32_t requests, uint32_t page_size, const int32_t *page_table, uint32_t max_pages,
                 const int32_t *free_pages, uint32_t free_count, uint32_t tokens, int32_t *table_out, int32_t *slots, int32_t *starts, int32_t *counts, hipStream_t st);
int paged_write(const PagedRows &rows, uint32_t key_column, uint32_t value_column, const int32_t *slots, void *key_cache, void *value_cache, const PagedCache &cache, hipStream_t st);

struct PagedAttentionArgs {
    PagedRows rows; uint32_t query_column;
    const void *key_cache, *value_cache; PagedCache cache;
    PagedStep step;
    uint32_t heads; float scale; uint32_t window;      // window 0: none
    void *out;                                         // [tokens, heads * head_dim], layout as the rows
    void *workspace; size_t workspace_bytes;
};
size_t paged_attention_workspace_bytes(uint32_t tokens, uint32_t requests, uint32_t heads, const PagedCache &cache);
int paged_attention(const PagedAttentionArgs &args, hipStream_t st);

}  // namespace ttmi
