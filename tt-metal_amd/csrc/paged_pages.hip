// Pages of a key/value cache that several requests have in common, that change hands, and that nobody needs any longer.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bfp_dequant.h"
#include "paged_cache.h"
#include "ttmi_internal.h"

namespace ttmi {

__device__ __forceinline__ uint32_t tokens_of(int32_t length) { return (uint32_t)max(length, 0); }

// ---------------------------------------------------------------------------------------------------------------------------------
// Forks.  Row i of the new table goes on from row parent_i of the old one.  With n tokens of the parent and pages of S,
//   entry j = the parent's for j S < n, else -1
// but for the page begun, j = n / S where S does not divide n: the first of a parent's continuations keeps it, each other one takes the next
// page from the list, in the order of the continuations, into which the one begun is to be copied.
// As the tables of a step are made: every workgroup finds the first continuations (LDS, atomic minimum) and makes the prefix sum for itself,
// then the entries are dealt out.  Bound by the launch and three loads that wait for each other (parents, lengths, the page begun): 3.4 us for
// four continuations, 4.5 for 96.
// ---------------------------------------------------------------------------------------------------------------------------------
struct ForkDev {
    const int32_t *table, *lengths, *parents, *free_pages;
    int32_t *table_out, *lengths_out, *sources, *targets, *counts;
    uint32_t requests, max_pages, page_size, children, free_count;
};

__global__ __launch_bounds__(256) void paged_fork_kernel(const ForkDev p) {
    extern __shared__ uint32_t lds[];                          // first[requests], taken[children]: pages taken up to and by a continuation, bit 31: one by itself
    uint32_t *const first = lds, *const taken = lds + p.requests;
    __shared__ uint32_t wave_sum[4];
    constexpr uint32_t COPIES = 0x80000000u;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto parent_of = [&](uint32_t i) { return (uint32_t)p.parents[i]; };
    for (uint32_t r = threadIdx.x; r < p.requests; r += 256) first[r] = 0xffffffffu;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.children; i += 256)
        if (const uint32_t r = parent_of(i); r < p.requests) atomicMin(first + r, i);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.children; i += 256) {
        const uint32_t r = parent_of(i);
        bool copies = false;
        if (r < p.requests && first[r] != i) {
            const uint32_t n = tokens_of(p.lengths[r]), j = n / p.page_size;
            copies = n % p.page_size && j < p.max_pages && p.table[(uint64_t)r * p.max_pages + j] >= 0;
        }
        taken[i] = copies ? COPIES : 0;
    }
    __syncthreads();
    const uint32_t each = (p.children + 255) / 256, i0 = min(threadIdx.x * each, p.children), i1 = min(i0 + each, p.children);
    uint32_t sum = 0;
    for (uint32_t i = i0; i < i1; ++i) sum += taken[i] >> 31;
    uint32_t to = running_sum(sum);
    if (lane == 63) wave_sum[wave] = to;
    __syncthreads();
    to -= sum;
    for (uint32_t w = 0; w < wave; ++w) to += wave_sum[w];
    for (uint32_t i = i0; i < i1; ++i) {
        const uint32_t flag = taken[i];
        taken[i] = flag | to;
        to += flag >> 31;
    }
    const uint32_t all = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    __syncthreads();

    auto fresh = [&](uint32_t i) {                             // the page that continuation i copies into
        const uint32_t at = taken[i] & ~COPIES;
        return at < p.free_count ? p.free_pages[at] : -1;
    };
    const uint64_t entries = (uint64_t)p.children * p.max_pages, step = (uint64_t)gridDim.x * 256, id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    for (uint64_t e = id; e < entries; e += step) {
        const uint32_t i = (uint32_t)(e / p.max_pages), j = (uint32_t)(e - (uint64_t)i * p.max_pages), r = parent_of(i);
        int32_t page = -1;
        if (r < p.requests) {
            const uint32_t n = tokens_of(p.lengths[r]);
            if ((taken[i] & COPIES) && j == n / p.page_size) page = fresh(i);
            else if ((uint64_t)j * p.page_size < n) page = p.table[(uint64_t)r * p.max_pages + j];
        }
        p.table_out[e] = page;
    }
    for (uint64_t e = id; e < p.children; e += step) {
        const uint32_t i = (uint32_t)e, r = parent_of(i), n = r < p.requests ? tokens_of(p.lengths[r]) : 0;
        p.lengths_out[i] = (int32_t)n;
        const int32_t target = taken[i] & COPIES ? fresh(i) : -1;
        p.targets[i] = target >= 0 ? target : -1;
        p.sources[i] = target >= 0 ? p.table[(uint64_t)r * p.max_pages + n / p.page_size] : -1;
    }
    if (id == 0) {
        const uint32_t got = min(all, p.free_count);
        p.counts[0] = (int32_t)got;
        p.counts[1] = (int32_t)(all - got);
    }
}

int paged_fork(const int32_t *page_table, const int32_t *lengths, uint32_t requests, uint32_t max_pages, uint32_t page_size, const int32_t *parents, uint32_t children,
               const int32_t *free_pages, uint32_t free_count, int32_t *table_out, int32_t *lengths_out, int32_t *sources, int32_t *targets, int32_t *counts, hipStream_t st) {
    const ForkDev p{page_table, lengths, parents, free_pages, table_out, lengths_out, sources, targets, counts, requests, max_pages, page_size, children, free_count};
    const uint64_t work = std::max<uint64_t>((uint64_t)children * max_pages, children);
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(std::max<uint64_t>((work + 255) / 256, 1), 512);
    hipLaunchKernelGGL(paged_fork_kernel, dim3(blocks), dim3(256), ((size_t)requests + children) * 4, st, p);
    return check_launch("paged_fork_kernel");
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Copies of whole pages, the same ones in every cache of a model.  A page is contiguous: a workgroup moves 16 KB of one, four loads of a lane on their way
// together.  12 pages of 128 KB in each of 16 caches, among 96 pairs of which the others copy nothing: 50 MB in 11.2 us with the launch = 4.5 TB/s.
// ---------------------------------------------------------------------------------------------------------------------------------
constexpr uint32_t CACHES = 128;           // of one launch: their addresses are kernel arguments
struct CopyDev {
    uint8_t *caches[CACHES];
    const int32_t *sources, *targets;
    uint64_t page_bytes, items;
    uint32_t count, pages, pairs, pieces;  // pieces of a page
};
constexpr uint32_t COPY_LOADS = 4, COPY_PIECE = 256 * 16 * COPY_LOADS;

__global__ __launch_bounds__(256) void paged_copy_kernel(const CopyDev p) {
    for (uint64_t item = blockIdx.x; item < p.items; item += gridDim.x) {
        const uint32_t piece = (uint32_t)(item % p.pieces);
        const uint64_t rest = item / p.pieces;
        const uint32_t which = (uint32_t)(rest % p.count), pair = (uint32_t)(rest / p.count);
        const uint32_t source = (uint32_t)p.sources[pair], target = (uint32_t)p.targets[pair];
        if (source >= p.pages || target >= p.pages || source == target) continue;
        uint8_t *const cache = p.caches[which];
        const uint64_t at = (uint64_t)piece * COPY_PIECE + threadIdx.x * 16;
        const uint8_t *const from = cache + source * p.page_bytes + at;
        uint8_t *const to = cache + target * p.page_bytes + at;
        u32x4 v[COPY_LOADS];
#pragma unroll
        for (uint32_t i = 0; i < COPY_LOADS; ++i)
            if (at + i * 4096 < p.page_bytes) v[i] = *reinterpret_cast<const u32x4 *>(from + i * 4096);
#pragma unroll
        for (uint32_t i = 0; i < COPY_LOADS; ++i)
            if (at + i * 4096 < p.page_bytes) *reinterpret_cast<u32x4 *>(to + i * 4096) = v[i];
    }
}

int paged_copy(void *const *caches, uint32_t count, const PagedCache &c, const int32_t *sources, const int32_t *targets, uint32_t pairs, hipStream_t st) {
    CopyDev p{};
    p.sources = sources; p.targets = targets; p.pages = c.pages; p.pairs = pairs;
    p.page_bytes = (uint64_t)c.kv_heads * (c.page_size / 32) * (c.head_dim / 32) * (c.dtype == TTMI_BFLOAT8_B ? 1088 : 2048);
    p.pieces = (uint32_t)((p.page_bytes + COPY_PIECE - 1) / COPY_PIECE);
    for (uint32_t first = 0; first < count; first += CACHES) {
        p.count = std::min(CACHES, count - first);
        for (uint32_t i = 0; i < p.count; ++i) p.caches[i] = (uint8_t *)caches[first + i];
        p.items = (uint64_t)p.pieces * p.count * pairs;
        if (!p.items) return TTMI_OK;
        hipLaunchKernelGGL(paged_copy_kernel, dim3((uint32_t)std::min<uint64_t>(p.items, 1u << 20)), dim3(256), 0, st, p);
        if (int rc = check_launch("paged_copy_kernel")) return rc;
    }
    return TTMI_OK;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Release.  With n tokens of a request, pages of S and a window of W (0: none) behind K sinks, entry j is kept where
//   j S < n   and   (W = 0, or j S + S > n + 1 - W: the next token sees a token of it, or j S < K)
// and is -1 elsewhere.  The pages that no entry kept names, in ascending order, are the new list of free pages: the place of a free page in
// it is the number of free ones before it.
// A byte for every page says whether it is in use.  Small tables and pools: one launch, in which every workgroup marks them in its own LDS from the whole
// table and writes its share of the results.  Large ones: in memory, cleared, set by plain stores (all of them store the same, so nothing has to be
// atomic: 1000 requests with common pages would wait for each other, 22 us instead of 5), and counted by every workgroup up to its share.
// 32 rows of 64 entries, 4096 pages: 4.4 us, the launch, two passes and their barriers; 1000 rows of 512, 300,000 pages: 2.2 + 5.1 + 8.0 us, the last of them for reading
// the bytes once per workgroup (256 lanes with one load at a time 24 us, 1024 with four 8).
// ---------------------------------------------------------------------------------------------------------------------------------
struct ReleaseDev {
    const int32_t *table, *lengths;
    int32_t *table_out, *free_pages, *counts;
    uint8_t *used;                         // one byte for every page, whole 256 of them
    uint32_t requests, max_pages, page_size, window, sinks, pages, share;
};
// Which entries of a request's row are kept: j < held and (j >= from or j < sinks).  j S + S > n + 1 - W is j >= floor((n + 1 - W) / S).
struct Kept {
    uint32_t held, from, sinks;
    __device__ __forceinline__ Kept(uint32_t held, uint32_t from, uint32_t sinks) : held(held), from(from), sinks(sinks) {}
    __device__ __forceinline__ Kept(const ReleaseDev &p, int32_t length) {
        const uint32_t n = tokens_of(length);
        auto pages = [&](uint32_t tokens) { return tokens / p.page_size + (tokens % p.page_size != 0); };
        held = pages(n);
        from = p.window && n + 1 > p.window ? (n + 1 - p.window) / p.page_size : 0;
        sinks = pages(p.sinks);
    }
    __device__ __forceinline__ int32_t operator()(const ReleaseDev &p, uint32_t j, int32_t page) const { return j < held && (j >= from || j < sinks) && (uint32_t)page < p.pages ? page : -1; }
};
// sum of v over the workgroup
template <uint32_t WAVES> __device__ __forceinline__ uint32_t sum_over_all(uint32_t v, uint32_t *lds) {
    v = last_lane(running_sum(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) v += lds[w];
    return v;
}
// The free pages of [first, first + share), share a multiple of 1024, go to their places in the list, in a workgroup of LIST_WAVES wavefronts: what is in use before them is counted, and
// in the parts of the wavefronts before this one.
constexpr uint32_t LIST_WAVES = 16;
__device__ __forceinline__ void list_free(const ReleaseDev &p, const uint8_t *used, uint32_t first, uint32_t share, uint32_t *sums) {
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t mine = first + wave * (share / LIST_WAVES), quads = (p.pages + 255) / 256 * 16;
    auto count = [&](uint32_t from, uint32_t to, uint32_t id, uint32_t step) __attribute__((always_inline)) {
        uint32_t n = 0;
        for (uint32_t i = from + id; i < to; i += 4 * step) {
            u32x4 v[4];                                        // on their way together
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) v[k] = reinterpret_cast<const u32x4 *>(used)[min(i + k * step, quads - 1)];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (i + k * step < to) n += __popc(v[k][0]) + __popc(v[k][1]) + __popc(v[k][2]) + __popc(v[k][3]);
        }
        return n;
    };
    const uint32_t ahead = count(first / 16, min(mine / 16, quads), lane, 64);
    const uint32_t before = sum_over_all<LIST_WAVES>(count(0, first / 16, threadIdx.x, LIST_WAVES * 64), sums);
    const uint32_t all = before + sum_over_all<LIST_WAVES>(count(first / 16, quads, threadIdx.x, LIST_WAVES * 64), sums), free = p.pages - all;
    uint32_t place = mine - before - last_lane(running_sum(ahead));
    for (uint32_t page0 = mine; page0 < min(mine + share / LIST_WAVES, p.pages); page0 += 64) {
        const bool is_free = page0 + lane < p.pages && !used[page0 + lane];
        const uint64_t them = __ballot(is_free);
        if (is_free) p.free_pages[place + __popcll(them & ((1ull << lane) - 1))] = (int32_t)(page0 + lane);
        place += __popcll(them);
    }
    for (uint64_t i = (uint64_t)free + blockIdx.x * blockDim.x + threadIdx.x; i < p.pages; i += (uint64_t)gridDim.x * blockDim.x) p.free_pages[i] = -1;
    if (blockIdx.x == 0 && threadIdx.x == 0) { p.counts[0] = (int32_t)free; p.counts[1] = (int32_t)all; }
}

__global__ __launch_bounds__(LIST_WAVES * 64) void paged_release_small_kernel(const ReleaseDev p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t in_use[];               // a byte for every page, whole 256 of them
    __shared__ uint32_t sums[LIST_WAVES];
    const uint32_t quads = (p.pages + 255) / 256 * 16;
    for (uint32_t i = threadIdx.x; i < quads; i += LIST_WAVES * 64) reinterpret_cast<u32x4 *>(in_use)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
    // A wavefront has every 16th group of four rows, 64 rows apart: its lanes find what is kept of 16 groups, one row each, then the entries of four rows are on their way together
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr uint32_t ROWS = 4, STRIDE = LIST_WAVES * ROWS;
    for (uint32_t base = wave * ROWS; base < p.requests; base += 16 * STRIDE) {
        const Kept row(p, p.lengths[min(base + lane / ROWS * STRIDE + lane % ROWS, p.requests - 1)]);
        for (uint32_t g = 0; g < 16 && base + g * STRIDE < p.requests; ++g) {
            const uint32_t r0 = base + g * STRIDE;
            const bool mine = r0 / ROWS % gridDim.x == blockIdx.x;
            for (uint32_t j = lane; j < p.max_pages; j += 64) {
                int32_t page[ROWS];
#pragma unroll
                for (uint32_t k = 0; k < ROWS; ++k) page[k] = p.table[min(r0 + k, p.requests - 1) * p.max_pages + j];
#pragma unroll
                for (uint32_t k = 0; k < ROWS; ++k) {
                    if (r0 + k >= p.requests) break;
                    const Kept of{(uint32_t)__builtin_amdgcn_readlane(row.held, g * ROWS + k), (uint32_t)__builtin_amdgcn_readlane(row.from, g * ROWS + k), (uint32_t)__builtin_amdgcn_readlane(row.sinks, g * ROWS + k)};
                    const int32_t kept = of(p, j, page[k]);
                    if (kept >= 0) in_use[kept] = 1;
                    if (mine) p.table_out[(r0 + k) * p.max_pages + j] = kept;
                }
            }
        }
    }
    __syncthreads();
    list_free(p, in_use, blockIdx.x * p.share, p.share, sums);
}

__global__ __launch_bounds__(256) void paged_release_clear_kernel(u32x4 *used, uint32_t quads) {
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < quads; i += gridDim.x * 256) used[i] = u32x4{0, 0, 0, 0};
}
__global__ __launch_bounds__(256) void paged_release_mark_kernel(const ReleaseDev p) {
    const uint32_t across = (p.max_pages + 255) / 256;         // workgroups of a row
    for (uint64_t i = blockIdx.x; i < (uint64_t)p.requests * across; i += gridDim.x) {
        const uint32_t r = (uint32_t)(i / across), j = (uint32_t)(i - (uint64_t)r * across) * 256 + threadIdx.x;
        if (j >= p.max_pages) continue;
        const uint64_t e = (uint64_t)r * p.max_pages + j;
        const int32_t page = Kept(p, p.lengths[r])(p, j, p.table[e]);
        p.table_out[e] = page;
        if (page >= 0) p.used[page] = 1;
    }
}
__global__ __launch_bounds__(LIST_WAVES * 64) void paged_release_list_kernel(const ReleaseDev p) {
    __shared__ uint32_t sums[LIST_WAVES];
    list_free(p, p.used, blockIdx.x * p.share, p.share, sums);
}

// Where one launch, whose every workgroup reads the whole table, is the shorter way (three launches).  Entries and pages: 32 x 64 entries, 4096 pages 4.6 us (7.6);
// 128 x 64, 65,536 pages 6.8 (9.1); 256 x 64, 65,536 pages 8.8 (9.1), 256 x 128 11.1 (9.1).  Turns of a wavefront, each four rows of 64 entries one after the other, whatever
// the entries: 4096 pages, 4 x 512 (8 turns) 8.0 (7.7), 32 x 512 (8) 8.7 (7.7), 4 x 1024 (16) 12.1 (7.7), 1024 x 16 (16) 21.9 (7.8), 1 x 4096 (64) 16.2 (7.8), 1 x 16384 (256) 54
// (7.6).  All replayed from a graph; called one by one, three launches cost the host 13.6 us, so that 8.7 are the shorter way there.
constexpr uint32_t SMALL_TABLE = 1u << 14, SMALL_POOL = 1u << 16, SMALL_TURNS = 8;
static bool small_release(uint32_t requests, uint32_t max_pages, uint32_t pages) {
    const uint64_t turns = ((uint64_t)requests + 63) / 64 * std::max<uint64_t>(((uint64_t)max_pages + 63) / 64, 1);
    return (uint64_t)requests * max_pages <= SMALL_TABLE && pages <= SMALL_POOL && turns <= SMALL_TURNS;
}
size_t paged_release_workspace_bytes(uint32_t requests, uint32_t max_pages, uint32_t pages) { return small_release(requests, max_pages, pages) ? 0 : ((size_t)pages + 255) / 256 * 256; }

int paged_release(const int32_t *page_table, const int32_t *lengths, uint32_t requests, uint32_t max_pages, uint32_t page_size, uint32_t window, uint32_t sinks, uint32_t pages,
                  int32_t *table_out, int32_t *free_pages, int32_t *counts, void *workspace, hipStream_t st) {
    ReleaseDev p{page_table, lengths, table_out, free_pages, counts, (uint8_t *)workspace, requests, max_pages, page_size, window, sinks, pages, 0};
    const uint32_t most = (uint32_t)std::min<uint64_t>(((uint64_t)pages + 2047) / 2048, 256);     // workgroups that list
    p.share = (uint32_t)((((uint64_t)pages + most - 1) / most + 1023) / 1024 * 1024);
    const dim3 blocks((uint32_t)(((uint64_t)pages + p.share - 1) / p.share));
    if (small_release(requests, max_pages, pages)) {
        hipLaunchKernelGGL(paged_release_small_kernel, blocks, dim3(LIST_WAVES * 64), ((size_t)pages + 255) / 256 * 256, st, p);
        return check_launch("paged_release_small_kernel");
    }
    const uint32_t quads = (uint32_t)(((uint64_t)pages + 255) / 256 * 16);
    hipLaunchKernelGGL(paged_release_clear_kernel, dim3(std::min((quads + 255) / 256, 1024u)), dim3(256), 0, st, (u32x4 *)workspace, quads);
    if (int rc = check_launch("paged_release_clear_kernel")) return rc;
    if ((uint64_t)requests * max_pages) {
        hipLaunchKernelGGL(paged_release_mark_kernel, dim3((uint32_t)std::min<uint64_t>((uint64_t)requests * ((max_pages + 255) / 256), 1u << 16)), dim3(256), 0, st, p);
        if (int rc = check_launch("paged_release_mark_kernel")) return rc;
    }
    hipLaunchKernelGGL(paged_release_list_kernel, blocks, dim3(LIST_WAVES * 64), 0, st, p);
    return check_launch("paged_release_list_kernel");
}

}  // namespace ttmi
