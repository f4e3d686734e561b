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

// Sums (maxima of numbers that are not negative) over the lanes up to and including this one, by DPP: no LDS and no barriers, the same in every wavefront.
template <int CTRL, int ROWS, typename T> __device__ __forceinline__ T lane_from(T x) {           // 0 where there is none
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <typename T, typename Join> __device__ __forceinline__ T running(T v, Join join) {
    v = join(v, lane_from<0x111, 0xf>(v));                      // 1, 2, 4, 8 lanes down within 16
    v = join(v, lane_from<0x112, 0xf>(v));
    v = join(v, lane_from<0x114, 0xf>(v));
    v = join(v, lane_from<0x118, 0xf>(v));
    v = join(v, lane_from<0x142, 0xa>(v));                      // lane 15 of each 16 to the next
    return join(v, lane_from<0x143, 0xc>(v));                   // lane 31 to the upper half
}
template <typename T> __device__ __forceinline__ T running_sum(T v) { return running(v, [](T a, T b) { return a + b; }); }
__device__ __forceinline__ uint32_t running_max(uint32_t v) { return running(v, [](uint32_t a, uint32_t b) { return max(a, b); }); }
template <typename T> __device__ __forceinline__ T last_lane(T v) { return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }

int paged_tables(const int32_t *cached, const int32_t *added, uint32_t requests, uint32_t page_size, const int32_t *page_table, uint32_t max_pages,
                 const int32_t *free_pages, uint32_t free_count, uint32_t tokens, int32_t *table_out, int32_t *slots, int32_t *starts, int32_t *counts, hipStream_t st);
int paged_write(const PagedRows &rows, uint32_t key_column, uint32_t value_column, const int32_t *slots, void *key_cache, void *value_cache, const PagedCache &cache, hipStream_t st);

struct PagedAttentionArgs {
    PagedRows rows; uint32_t query_column;
    const void *key_cache, *value_cache; PagedCache cache;
    PagedStep step;
    uint32_t heads; float scale; uint32_t window, sinks;       // window 0: none
    void *out;                                         // [tokens, heads * head_dim], layout as the rows
    void *workspace; size_t workspace_bytes;
};
// Queries and keys of a step by their positions; without caches (key_cache null) queries alone.
struct PagedRotationArgs {
    PagedRows rows; uint32_t query_column, heads, head_dim;
    uint32_t key_column, value_column; const int32_t *slots;
    void *key_cache, *value_cache; PagedCache cache;
    PagedStep step;                                    // without its page table
    const float *frequencies; uint32_t rotary_dim; int interleaved;
    const float *query_norm, *key_norm; float epsilon, magnitude;
    void *out;                                         // [tokens, heads * head_dim], layout as the rows
};
int paged_rotate(const PagedRotationArgs &args, hipStream_t st);

int paged_fork(const int32_t *page_table, const int32_t *lengths, uint32_t requests, uint32_t max_pages, uint32_t page_size, const int32_t *parents, uint32_t children,
               const int32_t *free_pages, uint32_t free_count, int32_t *table_out, int32_t *lengths_out, int32_t *sources, int32_t *targets, int32_t *counts, hipStream_t st);
int paged_copy(void *const *caches, uint32_t count, const PagedCache &cache, const int32_t *sources, const int32_t *targets, uint32_t pairs, hipStream_t st);
size_t paged_release_workspace_bytes(uint32_t requests, uint32_t max_pages, uint32_t pages);
int paged_release(const int32_t *page_table, const int32_t *lengths, uint32_t requests, uint32_t max_pages, uint32_t page_size, uint32_t window, uint32_t sinks, uint32_t pages,
                  int32_t *table_out, int32_t *free_pages, int32_t *counts, void *workspace, hipStream_t st);

size_t paged_attention_workspace_bytes(uint32_t tokens, uint32_t requests, uint32_t heads, const PagedCache &cache);
int paged_attention(const PagedAttentionArgs &args, hipStream_t st);

}  // namespace ttmi
