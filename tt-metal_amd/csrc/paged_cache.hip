// A key/value cache in pages: the tables that say where every token lies, and the writes into it.
//
// A cache is one tensor [pages, kv_heads, page_size, head_dim] in TILE layout, bf16 or BFLOAT8_B; page_size and head_dim are
// multiples of 32, so 32 consecutive tokens of a head are head_dim / 32 whole tiles that follow each other in memory.  Token
// p of a request lies in slot table[p / page_size] * page_size + p % page_size.  A page number outside [0, pages), -1 among
// them, means that there is no page.  In BFLOAT8_B the 16 elements that share an exponent are neighbours of one token, so a
// token is written without a look at the ones around it.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bfp_dequant.h"
#include "paged_cache.h"
#include "ttmi_internal.h"

namespace ttmi {

// ---------------------------------------------------------------------------------------------------------------------------------
// Tables.  With c cached and n new tokens of request r, pages of S tokens and table rows of M entries
//   held = min(M, ceil(c / S))    want = min(M, ceil((c + n) / S))    base = sum over the requests before of want - held
//   table'[r, j] = table[r, j] for j < held, free[base + j - held] for held <= j < want as far as the list goes, else -1
//   start[r] = sum over the requests before of n,   slot[start + i] = place of token c + i
// Every workgroup makes both prefix sums for itself (requests / 256 values per lane, one pass over LDS): what a second launch, or
// a wait for another workgroup, costs is more than reading a few KB of lengths again.  Then the table's entries and the tokens
// are dealt out, one to a lane; a token finds its request by bisection in LDS.  Bound by the launch and by three loads that wait for each
// other (lengths, then the old table or the list): 3.9 us for 32 requests of 64 entries, 6.0 for 257 of 300 with 32,000 tokens.
// ---------------------------------------------------------------------------------------------------------------------------------
struct TablesDev {
    const int32_t *cached, *added, *table, *free_pages;
    int32_t *table_out, *slots, *starts, *counts;
    uint32_t requests, page_size, max_pages, free_count, tokens;
};

__device__ __forceinline__ uint32_t pages_of(uint64_t tokens, uint32_t page_size, uint32_t max_pages) {
    const uint64_t pages = (tokens + page_size - 1) / page_size;
    return pages < max_pages ? (uint32_t)pages : max_pages;
}

__global__ __launch_bounds__(256) void paged_tables_kernel(const TablesDev p) {
    extern __shared__ uint32_t prefix[];                      // starts[requests + 1], base[requests + 1]
    uint32_t *const starts = prefix, *const base = prefix + p.requests + 1;
    __shared__ uint64_t wave_sum[4][2];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t each = (p.requests + 255) / 256, first = threadIdx.x * each;
    auto length = [](int32_t v) { return (uint32_t)max(v, 0); };

    uint64_t rows = 0, taken = 0;                             // of this lane's requests
    for (uint32_t r = first; r < min(first + each, p.requests); ++r) {
        const uint32_t c = length(p.cached[r]), n = length(p.added[r]);
        rows += n;
        taken += pages_of((uint64_t)c + n, p.page_size, p.max_pages) - pages_of(c, p.page_size, p.max_pages);
    }
    uint64_t rows_to = rows, taken_to = taken;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t a = __shfl_up(rows_to, d), b = __shfl_up(taken_to, d);
        if (lane >= (uint32_t)d) { rows_to += a; taken_to += b; }
    }
    if (lane == 63) { wave_sum[wave][0] = rows_to; wave_sum[wave][1] = taken_to; }
    __syncthreads();
    rows_to -= rows; taken_to -= taken;
    for (uint32_t w = 0; w < wave; ++w) { rows_to += wave_sum[w][0]; taken_to += wave_sum[w][1]; }
    for (uint32_t r = first; r < min(first + each, p.requests); ++r) {
        const uint32_t c = length(p.cached[r]), n = length(p.added[r]);
        starts[r] = (uint32_t)min(rows_to, (uint64_t)p.tokens);       // rows past the last one do not exist
        base[r] = (uint32_t)min(taken_to, (uint64_t)0xffffffffu);
        rows_to += n;
        taken_to += pages_of((uint64_t)c + n, p.page_size, p.max_pages) - pages_of(c, p.page_size, p.max_pages);
    }
    uint64_t all_rows = 0, all_taken = 0;
    for (int w = 0; w < 4; ++w) { all_rows += wave_sum[w][0]; all_taken += wave_sum[w][1]; }
    if (threadIdx.x == 0) starts[p.requests] = (uint32_t)min(all_rows, (uint64_t)p.tokens);
    __syncthreads();

    // entry j of request r, as the new table has it; only entries that r holds already are read from the old one, so the two may be one
    auto page_at = [&](uint32_t r, uint32_t j) {
        const uint32_t c = length(p.cached[r]), held = pages_of(c, p.page_size, p.max_pages);
        if (j < held) return p.table[(uint64_t)r * p.max_pages + j];
        if (j >= pages_of((uint64_t)c + length(p.added[r]), p.page_size, p.max_pages)) return -1;
        const uint64_t at = (uint64_t)base[r] + (j - held);
        return at < p.free_count ? p.free_pages[at] : -1;
    };
    const uint64_t entries = (uint64_t)p.requests * p.max_pages, step = (uint64_t)gridDim.x * 256;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += step)
        p.table_out[i] = page_at((uint32_t)(i / p.max_pages), (uint32_t)(i % p.max_pages));
    for (uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x; t < p.tokens; t += step) {
        int32_t slot = -1;
        if (t < starts[p.requests]) {
            uint32_t low = 0, high = p.requests;              // starts[low] <= t < starts[high]
            while (high - low > 1) {
                const uint32_t mid = (low + high) / 2;
                if (starts[mid] <= t) low = mid; else high = mid;
            }
            const uint64_t position = (uint64_t)length(p.cached[low]) + (t - starts[low]);
            const uint64_t j = position / p.page_size;
            const int32_t page = j < p.max_pages ? page_at(low, (uint32_t)j) : -1;
            const int64_t at = (int64_t)page * p.page_size + (int64_t)(position % p.page_size);
            if (page >= 0 && at <= 0x7fffffff) slot = (int32_t)at;
        }
        p.slots[t] = slot;
    }
    if (blockIdx.x == 0) {
        for (uint32_t r = threadIdx.x; r <= p.requests; r += 256) p.starts[r] = (int32_t)starts[r];
        if (threadIdx.x == 0) {
            const uint64_t got = min(all_taken, (uint64_t)p.free_count);
            p.counts[0] = (int32_t)got;
            p.counts[1] = (int32_t)min(all_taken - got, (uint64_t)0x7fffffff);
        }
    }
}

int paged_tables(const int32_t *cached, const int32_t *added, uint32_t requests, uint32_t page_size, const int32_t *page_table, uint32_t max_pages,
                 const int32_t *free_pages, uint32_t free_count, uint32_t tokens, int32_t *table_out, int32_t *slots, int32_t *starts, int32_t *counts, hipStream_t st) {
    const TablesDev p{cached, added, page_table, free_pages, table_out, slots, starts, counts, requests, page_size, max_pages, free_count, tokens};
    const uint64_t work = std::max<uint64_t>((uint64_t)requests * max_pages, tokens);
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(std::max<uint64_t>((work + 255) / 256, 1), 1024);
    hipLaunchKernelGGL(paged_tables_kernel, dim3(blocks), dim3(256), 2 * ((size_t)requests + 1) * 4, st, p);
    return check_launch("paged_tables_kernel");
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Writes.  A lane moves a face row: 16 neighbouring elements of one token, 32 bytes of the activations, and 32 bytes of a bf16 cache
// or 16 codes and their exponent of a BFLOAT8_B one (the host packers' arithmetic).  Bound by latency: two loads that wait for each other (slot, row), then
// the stores; a copy moves twice as much in the time of the larger case below.  In TILE layout neighbouring
// lanes take neighbouring tokens, in row-major rows neighbouring columns: 16 lanes read 512 contiguous bytes, and where tokens lie
// next to each other in a page, as those of a prompt do, they write 512 (or 256) contiguous bytes too.  4100 tokens, 8 key heads of 128
// elements, into BFLOAT8_B: 26 MB in 9.8 us = 2.6 TB/s with the launch; 32 tokens into bf16: 3.2 us, the launch.
// ---------------------------------------------------------------------------------------------------------------------------------
struct WriteDev {
    const uint8_t *rows;
    const int32_t *slots;
    uint8_t *cache[2];
    uint64_t groups;                       // face rows of keys and values over all tokens
    uint32_t tokens, width, column16[2];   // first key and value column / 16
    uint32_t per_head, across;             // face rows of a head, and of all heads, per token
    uint32_t pages, kv_heads, page_size;
    int tiled;
};

template <bool PACK> __global__ __launch_bounds__(256) void paged_write_kernel(const WriteDev p) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < p.groups; i += (uint64_t)gridDim.x * 256) {
        uint32_t t, g;                                        // token, face row among those of its keys and values
        if (p.tiled) {
            const uint64_t band = i / (64 * p.across);
            const uint32_t rest = (uint32_t)(i - band * (64 * p.across));
            t = (uint32_t)band * 32 + (rest & 31);
            g = rest >> 5;
        } else {
            t = (uint32_t)(i / (2 * p.across));
            g = (uint32_t)(i - (uint64_t)t * (2 * p.across));
        }
        if (t >= p.tokens) continue;
        const int32_t slot = p.slots[t];
        if (slot < 0) continue;
        const uint32_t page = (uint32_t)slot / p.page_size, at = (uint32_t)slot - page * p.page_size;
        if (page >= p.pages) continue;
        const uint32_t which = g >= p.across ? 1 : 0, c = g - which * p.across;
        const u32x4 *from = reinterpret_cast<const u32x4 *>(p.rows + row_bytes_at(t, p.width, (p.column16[which] + c) * 16, p.tiled));
        const u32x4 lo = from[0], hi = from[1];

        const uint32_t head = c / p.per_head, f = c - head * p.per_head;      // face column of the head
        const uint64_t tile = (((uint64_t)page * p.kv_heads + head) * (p.page_size / 32) + at / 32) * (p.per_head / 2) + f / 2;
        const uint32_t face = (at >> 4 & 1) * 2 + (f & 1), row = at & 15;
        if (!PACK) {
            u32x4 *to = reinterpret_cast<u32x4 *>(p.cache[which] + tile * 2048 + face * 512 + row * 32);
            to[0] = lo;
            to[1] = hi;
            continue;
        }
        uint32_t bits[16], shared = 0, words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t w = e < 4 ? lo[e & 3] : hi[e & 3];
            bits[2 * e] = w << 16;
            bits[2 * e + 1] = w & 0xffff0000u;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) shared = max(shared, (bits[e] >> 23) & 0xffu);
#pragma unroll
        for (int e = 0; e < 16; ++e) words[e >> 2] |= to_code<7>(bits[e], shared) << (8 * (e & 3));
        uint8_t *to = p.cache[which] + tile * 1088;
        *reinterpret_cast<u32x4 *>(to + 64 + face * 256 + row * 16) = u32x4{words[0], words[1], words[2], words[3]};
        to[face * 16 + row] = (uint8_t)shared;
    }
}

int paged_write(const PagedRows &rows, uint32_t key_column, uint32_t value_column, const int32_t *slots, void *key_cache, void *value_cache, const PagedCache &cache, hipStream_t st) {
    if (!rows.tokens) return TTMI_OK;
    WriteDev p{};
    p.rows = (const uint8_t *)rows.data; p.slots = slots;
    p.cache[0] = (uint8_t *)key_cache; p.cache[1] = (uint8_t *)value_cache;
    p.tokens = rows.tokens; p.width = rows.width; p.tiled = rows.layout == TTMI_TILE;
    p.column16[0] = key_column / 16; p.column16[1] = value_column / 16;
    p.per_head = cache.head_dim / 16; p.across = cache.kv_heads * p.per_head;
    p.pages = cache.pages; p.kv_heads = cache.kv_heads; p.page_size = cache.page_size;
    const uint64_t tokens = p.tiled ? ((uint64_t)p.tokens + 31) / 32 * 32 : p.tokens;
    p.groups = tokens * 2 * p.across;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((p.groups + 255) / 256, 256 * 16);
    if (cache.dtype == TTMI_BFLOAT8_B) hipLaunchKernelGGL((paged_write_kernel<true>), dim3(blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_write_kernel<false>), dim3(blocks), dim3(256), 0, st, p);
    return check_launch("paged_write_kernel");
}

}  // namespace ttmi
