// Attention of new tokens over a paged key/value cache (paged_cache.hip says how one is laid out).
//
// Request r has cached_r tokens from before and n_r = row_starts[r + 1] - row_starts[r] new ones, all of them in the cache.  Row
// row_starts[r] + i of the activations is token p = cached_r + i.  For each of its heads, with the key head that its group shares,
//   out = sum_j softmax_j(scale q . k_j) v_j    over the tokens p - window < j <= p that have a page
// and zeros where nothing is left.
//
// Common to both kernels
//   rows       the heads that share a key head are rows of one product: row rho of (request, key head) is token rho / group, head
//              rho % group of the group, so a decode step of 4 heads per key head is 4 rows, a chunk of 512 tokens 2048
//   units      (request, key head, tile of ROWS rows).  A unit's tokens are cut into pieces of a common length, which is chosen from the
//              lengths on the device so that the whole step comes to about `target` pieces: requests of any lengths, one long one among
//              them, fill the chip evenly.  Every wavefront makes the same prefix sums over the requests (1 us for 64 of them) and
//              takes pieces blockIdx, blockIdx + gridDim, ...  A unit of one piece is stored at once; the others leave (maximum, sum, fp32
//              accumulators) in memory, and whoever comes last joins them, in the order of the pieces: results do not depend on
//              who that is.  The join costs 3 us for one row tile, 8 for five, 15 for 256 rows of 128 elements in four parts
//   softmax    one pass: running maximum m and sum l per row in fp32, weights exp2(s - m).  m only moves when a score passes it
//              by more than 2^8 in weight, so that the accumulators are hardly ever rescaled (two prompts of 5000 tokens, 32 heads on 8
//              key heads, window 4096: 527 us, 566 where m always moves)
//   products   keys times queries and values times weights, both transposed: a lane's accumulators belong to one row, so m, l and the
//              rescaling are the lane's own, and the weights leave the first product in the very lanes that the second one
//              wants them in (the tokens of a k step are permuted alike on both sides).  Weights are rounded to bf16 for
//              the second product, as the values are, and l is the sum of the rounded ones: what a row is divided by is what it
//              was multiplied with, so a row of one token is that token's value (v_dot2_f32_bf16 adds two at a time).  Rows of
//              few tokens have no others for the roundings to cancel against: in the block where a row ends what the rounding
//              took off is a second product.  Elsewhere it is left out: results are 2.0e-3 to 2.2e-3 off 64 bits (2-norm over 2-norm, scores
//              with a spread of 2), with it everywhere 1.7e-3, the rounding of the result alone.  It would cost 32 users x 2000 tokens in bf16 63.0 us
//              instead of 61.8, drafts of 5 tokens 69.0 (66.6), 8 users x 16000 in BFLOAT8_B 124 (98), 512 tokens behind 7680 114 (86), prompts 691 (527)
//   masks      a score that does not count becomes -inf, its weight 0.  bf16 values that no row of the unit sees (behind the last token,
//              before the window) are zeroed on their way into LDS: 0 x NaN is NaN.  Where rows of a unit see different tokens, or one
//              ends (what a rounding took off may have either sign), values that are not finite are taken out as well, and two
//              products with ones in their places say which rows see them.  Block floats are always finite here: see block_scale
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "bfp_dequant.h"
#include "paged_cache.h"
#include "ttmi_internal.h"

namespace ttmi {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

struct AttentionDev {
    const uint8_t *rows, *keys, *values;
    const int32_t *table, *cached, *starts;
    uint8_t *out;
    uint32_t tokens, out_rows, width, query_column, requests, max_pages;
    uint32_t pages, kv_heads, page_blocks, heads, group, window;
    uint32_t least_rows, most_rows;        // requests of that many rows per key head are this launch's
    uint32_t target, slots;                // about how many pieces the step is cut into; partial results that fit
    uint32_t *counters;                    // pieces of a unit that are done, by the unit's first slot; all zero between launches
    uint8_t *partial;
    float scale;                           // |scale| log2(e)
    uint32_t flip;                         // sign bits of the queries, for a negative scale
    int tiled, zero_rows;                  // zero_rows: this launch clears the rows of no request
};

constexpr uint32_t COUNTERS = 4096;        // at most 2 `target` slots, each could be a unit's first
constexpr float LAZY = 8.f;                // how far (log2) a score may pass the running maximum

// Operands go from LDS through a ring of this many, so that a product finds its own in registers.  Four took 537 us where two take 527 (two prompts of
// 5000 tokens with a window of 4096): they are eight registers more, which are spilled.
constexpr int AHEAD = 2;
// Reads of LDS and products stay in the order in which they are written; everything else may pass.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x476); }

// ---- the work of a step ---------------------------------------------------------------------------------------------------------
struct Request { uint32_t start, added, cached; };
__device__ __forceinline__ uint32_t start_at(const AttentionDev &p, uint32_t r) { return min((uint32_t)max(p.starts[r], 0), p.tokens); }
// Request r from what memory says of it.  `taken`: rows up to here belong to the requests before.  Row starts ascend, and then it changes nothing; where they
// do not, it keeps two requests from the same rows.
__device__ __forceinline__ Request request_of(uint32_t start, uint32_t end, int32_t cached, uint32_t taken) {
    const uint32_t from = max(start, taken), to = max(end, from);
    return {from, to - from, (uint32_t)max(cached, 0)};
}
__device__ __forceinline__ Request request_at(const AttentionDev &p, uint32_t r, uint32_t taken) { return request_of(start_at(p, r), start_at(p, r + 1), p.cached[r], taken); }
// Positions in masks, which compare signed differences.  No page holds a token from 2^31 - 1 on: positions there, behind what the page table
// can name, see what one at 2^31 - 1 sees of it.
__device__ __forceinline__ uint32_t in_table(uint32_t position) { return min(position, 0x7fffffffu); }
// first token that a row at `position` sees
__device__ __forceinline__ uint32_t first_seen(const AttentionDev &p, uint32_t position) {
    return p.window && position >= p.window ? position - p.window + 1 : 0u;
}

// Token and head of rows: rho = token * group + head.  A piece's rows are counted from its first token on, where the quotient is small: a product
// with the reciprocal is off by one at most.
struct Rows {
    uint32_t token0, base, group;
    float inverse;
    __device__ __forceinline__ Rows(uint32_t token0, uint32_t group) : token0(token0), base(token0 * group), group(group), inverse(__builtin_amdgcn_rcpf((float)group)) {}
    __device__ __forceinline__ void at(uint32_t rho, uint32_t &token, uint32_t &head) const {
        const uint32_t n = rho - base;
        uint32_t q = (uint32_t)((float)n * inverse);
        int32_t rest = (int32_t)(n - q * group);
        if (rest < 0) { --q; rest += group; }
        if (rest >= (int32_t)group) { ++q; rest -= group; }
        token = token0 + q;
        head = (uint32_t)rest;
    }
};

template <int ROWS> struct Extent {
    uint32_t units, blocks;                // units of the request; 32-token blocks that one of them has at most
    __device__ __forceinline__ Extent(const AttentionDev &p, const Request &q) {
        const uint64_t rows = (uint64_t)q.added * p.group;
        if (rows < p.least_rows || rows > p.most_rows) { units = blocks = 0; return; }
        units = (uint32_t)((rows + ROWS - 1) / ROWS) * p.kv_heads;
        const uint32_t end = min((q.cached + q.added - 1) / 32 + 1, p.max_pages * p.page_blocks), begin = min(first_seen(p, q.cached) / 32, end);
        blocks = end - begin;
        if (p.window) blocks = (uint32_t)min((uint64_t)blocks, ((uint64_t)p.window + ROWS / p.group + 2) / 32 + 2);
        blocks = max(blocks, 1u);
    }
};

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

// The pieces of the step.  Every wavefront makes the plan for itself: a lane has `each` requests, one where there are at most 64.
struct Plan {
    uint32_t each, piece, pieces;          // blocks of a piece, pieces of the step
    uint32_t first_piece, first_slot;      // of this lane's requests
    uint32_t begin, end;                   // first row of the first request, end of the last one's rows
    Request q;                             // this lane's first request
};
template <int ROWS, int STEP> __device__ __forceinline__ Plan make_plan(const AttentionDev &p) {
    const uint32_t lane = threadIdx.x & 63;
    Plan plan;
    plan.each = (p.requests + 63) / 64;
    const uint32_t r0 = min(lane * plan.each, p.requests), r1 = min(r0 + plan.each, p.requests);
    uint32_t start = 0, end = 0;           // of the first one; these loads are on their way together
    int32_t cached = 0;
    if (r0 < r1) { start = start_at(p, r0); end = start_at(p, r0 + 1); cached = p.cached[r0]; }
    uint32_t top = max(start, end);        // up to the end of this lane's requests
    for (uint32_t r = r0 + 2; r <= r1; ++r) top = max(top, start_at(p, r));
    top = running_max(top);
    plan.end = last_lane(top);
    const uint32_t taken = lane_from<0x138, 0xf>(top);         // by the lanes before
    plan.q = r0 < r1 ? request_of(start, end, cached, taken) : Request{0, 0, 0};
    plan.begin = __builtin_amdgcn_readfirstlane(plan.q.start);
    float work = 0.f, units = 0.f;
    Request q = plan.q;
    for (uint32_t r = r0; r < r1; ++r) {
        if (r > r0) q = request_at(p, r, q.start + q.added);
        const Extent<ROWS> e(p, q);
        work += (float)e.units * (float)e.blocks;
        units += (float)e.units;
    }
    work = last_lane(running_sum(work));
    units = last_lane(running_sum(units));
    // the last piece of a unit is on average half a piece: that many more come to about one for each resident workgroup
    const float aim = fmaxf((float)p.target - 0.5f * units, 0.25f * (float)p.target);
    plan.piece = ((uint32_t)fminf(fmaxf(ceilf(work / aim), 1.f), 1e9f) + STEP - 1) / STEP * STEP;
    uint32_t pieces = 0, slots = 0;        // of this lane's requests: pieces, and those of units with more than one
    q = plan.q;
    for (uint32_t r = r0; r < r1; ++r) {
        if (r > r0) q = request_at(p, r, q.start + q.added);
        const Extent<ROWS> e(p, q);
        const uint32_t parts = (e.blocks + plan.piece - 1) / plan.piece;
        pieces += e.units * parts;
        if (parts > 1) slots += e.units * parts;
    }
    const uint32_t pieces_to = running_sum(pieces), slots_to = running_sum(slots);
    plan.first_piece = pieces_to - pieces;
    plan.first_slot = slots_to - slots;
    plan.pieces = last_lane(pieces_to);
    return plan;
}

// One piece: rows [row0, row0 + rows) of a request and key head, blocks [begin, end) of those that the unit sees.
struct Piece {
    Request q;
    uint32_t r, kv, row0, rows, begin, end, parts, part, slot;
    uint32_t token0, token1;               // first and last token of the unit, counted from the request's first new one
};
// False where the unit has fewer pieces than others of its request, and this is none of them.
template <int ROWS> __device__ __forceinline__ bool piece_at(const AttentionDev &p, const Plan &plan, uint32_t index, Piece &x) {
    const uint32_t owner = __popcll(__ballot(plan.first_piece <= index)) - 1;
    uint32_t at = __builtin_amdgcn_readlane(plan.first_piece, owner), most, units;
    x.slot = __builtin_amdgcn_readlane(plan.first_slot, owner);
    x.r = owner * plan.each;
    x.q = {(uint32_t)__builtin_amdgcn_readlane(plan.q.start, owner), (uint32_t)__builtin_amdgcn_readlane(plan.q.added, owner), (uint32_t)__builtin_amdgcn_readlane(plan.q.cached, owner)};
    for (uint32_t i = 0;; ++i) {
        const Extent<ROWS> e(p, x.q);
        units = e.units;
        most = (e.blocks + plan.piece - 1) / plan.piece;
        if (index < at + units * most || i + 1 >= plan.each || x.r + 1 >= p.requests) break;
        at += units * most;
        if (most > 1) x.slot += units * most;
        x.q = request_at(p, ++x.r, x.q.start + x.q.added);
    }
    if (index - at >= units * most) return false;              // only if the lengths changed meanwhile
    uint32_t local = index - at;
    x.kv = local % p.kv_heads; local /= p.kv_heads;
    x.part = local % most;
    const uint32_t tile = units / p.kv_heads - 1 - local / most;                       // the last tile of a chunk sees most: first
    const uint32_t all_rows = x.q.added * p.group;
    x.row0 = tile * ROWS;
    x.rows = min((uint32_t)ROWS, all_rows - x.row0);
    x.token0 = x.row0 / p.group;
    x.token1 = (x.row0 + x.rows - 1) / p.group;
    const uint32_t end = min((x.q.cached + x.token1) / 32 + 1, p.max_pages * p.page_blocks), begin = min(first_seen(p, x.q.cached + x.token0) / 32, end);
    x.parts = max((end - begin + plan.piece - 1) / plan.piece, 1u);
    x.begin = min(begin + x.part * plan.piece, end);
    x.end = min(x.begin + plan.piece, end);
    x.slot += (tile * p.kv_heads + x.kv) * most;
    return x.part < x.parts;
}

// Where the blocks first, first + STRIDE, ... of a piece lie, 64 at a time: lane i has the byte at which the keys, and the values, of entry i
// start, 0 (page 0) for what has no page or lies past the end.
template <int STRIDE, int BLOCK_BYTES> struct Blocks {
    uint32_t low, high;
    uint64_t pages;                        // bit i: entry i has a page
    __device__ __forceinline__ void load(const AttentionDev &p, const Piece &x, uint32_t first) {
        const uint32_t b = first + (threadIdx.x & 63) * STRIDE, column = b / p.page_blocks;
        const int32_t page = b < x.end ? p.table[(uint64_t)x.r * p.max_pages + column] : -1;
        const bool there = (uint32_t)page < p.pages;
        const uint64_t at = there ? (((uint64_t)page * p.kv_heads + x.kv) * p.page_blocks + (b - column * p.page_blocks)) * BLOCK_BYTES : 0;
        low = (uint32_t)at;
        high = (uint32_t)(at >> 32);
        pages = __ballot(there);
    }
    __device__ __forceinline__ uint64_t at(uint32_t i) const { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(high, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(low, i); }
    __device__ __forceinline__ bool has(uint32_t i) const { return pages >> i & 1; }
};

// ---- softmax ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float floor_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ float max_over_halves(float v) {
    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1]));
}
__device__ __forceinline__ float sum_over_halves(float v) {
    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(o[0]) + __uint_as_float(o[1]);
}
__device__ __forceinline__ float max_over_quarters(float v) {
    const auto o = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max_over_halves(fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1])));
}
__device__ __forceinline__ float sum_over_quarters(float v) {
    const auto o = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return sum_over_halves(__uint_as_float(o[0]) + __uint_as_float(o[1]));
}

// sum + both bf16 of a word
__device__ __forceinline__ float add_pair(uint32_t pair, float sum) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), sum, false);
}

// ---- partial results -------------------------------------------------------------------------------------------------------------------
// Stored past the L2 of the XCD (sc1): a release of all that the L2 holds would cost more than the kernel.  Loaded as any other memory, behind
// an acquire: nobody has read these lines before in the launch, and loads past the L2 were slower.
__device__ __forceinline__ void put_quad(uint8_t *to, const f32x4 &v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(to), "v"(v) : "memory");
}
__device__ __forceinline__ f32x4 get_quad(const uint8_t *from) { return *reinterpret_cast<const f32x4 *>(from); }
// Called by the whole workgroup once its partial result is on its way; true for the one that finds all the others' there.
__device__ __forceinline__ bool last_of(const AttentionDev &p, const Piece &x, uint32_t *flag) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // this wavefront's stores have arrived
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t *counter = p.counters + x.slot;
        const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == x.parts - 1;
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    if (!*flag) return false;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    return true;
}

// LDS that lanes of one wavefront hand each other: the hardware keeps a wavefront's accesses in order, this keeps the compiler to it.
__device__ __forceinline__ void lanes_in_order() {
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// bf16 values that are not finite.  KEEP_FINITE: zeros in their places; ONES_UP, ONES_DOWN: ones where adding the value would add +inf or
// NaN, or -inf or NaN, zeros elsewhere (a NaN is both: inf - inf).
enum Pick { KEEP_FINITE, ONES_UP, ONES_DOWN };
__device__ __forceinline__ uint32_t pick(uint32_t v, Pick how) {            // two values
    const uint32_t size = v & 0x7fff7fffu, gone = (size + 0x00800080u) & 0x80008000u, nan = size + 0x007f007fu;     // bit 15 of each half
    if (how == KEEP_FINITE) return v & ~((gone >> 15) * 0xffffu);
    return ((gone & (nan | (how == ONES_DOWN ? v : ~v))) >> 15) * 0x3f80u;
}
__device__ __forceinline__ u32x4 pick(u32x4 v, Pick how) { return u32x4{pick(v[0], how), pick(v[1], how), pick(v[2], how), pick(v[3], how)}; }

// What a mantissa of 1 stands for in a face row of block floats: 2^(E - 133), as a float.  The exponent byte of a row that infinities or
// NaN were written into, 255, is read as 254, so that every value is finite; below 7 (numbers under 2^-119) it is read as 7.
__device__ __forceinline__ float block_scale(uint32_t e) { return __uint_as_float((min(max(e, 7u), 254u) - 6u) << 23); }
// eight block floats of a face row as bf16, exactly
__device__ __forceinline__ u32x4 expand8(uint32_t w0, uint32_t w1, float scale) {
    const uint32_t m0 = w0 & 0x7f7f7f7fu, m1 = w1 & 0x7f7f7f7fu;
    return u32x4{activations_pair<0>(w0, m0, scale), activations_pair<2>(w0, m0, scale), activations_pair<0>(w1, m1, scale), activations_pair<2>(w1, m1, scale)};
}

// Zeros for the rows of no request: those before the first one's and behind the last one's, with the rows that fill up the last tiles.
__device__ __forceinline__ void clear_rows(const AttentionDev &p, uint32_t head_dim, uint32_t before, uint32_t behind) {
    const uint32_t width = p.heads * head_dim, pieces = width / 8;
    const uint64_t all = (uint64_t)(before + p.out_rows - behind) * pieces;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t row = (uint32_t)(i / pieces);
        *reinterpret_cast<u32x4 *>(p.out + row_bytes_at(row < before ? row : row - before + behind, width, (uint32_t)(i % pieces) * 8, p.tiled)) = u32x4{0, 0, 0, 0};
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Few rows (decode, drafts): bound by reading the cache.  Four wavefronts share a unit of MT x 16 rows and take its 32-token blocks in
// turn, each with softmax state of its own; they are joined at the end.  v_mfma_f32_16x16x32_bf16.
//   32 users x 4000 tokens, 8 key heads of 128 elements, 4 query heads to each: bf16 94 us = 5.6 TB/s (a large copy moves 4.9); BFLOAT8_B
//   72 us = 3.9 TB/s, its vector ALU two thirds busy with the expansion (4 instructions for a value).  17 query heads to a key head, two row
//   tiles: 98 and 83 us.  One user, 1500 tokens: 11 us, of which launch 2.5, plan and piece 2, first loads 2, joins 4
//   keys     go from memory into the registers of the MFMA operand (16 bytes per lane, whole tiles); block floats are expanded there
//   values   go through 32 tokens of LDS that belong to the wavefront (no barriers) for their transposition: ds_read_b64_tr_b16 for
//            bf16; block floats as words of four columns, of which each of four products takes one byte
// The next block is asked for as soon as a block's keys are multiplied and its values are in LDS.  Nothing should spill in that loop: a reload
// from scratch memory waits for all loads before it, the next block's among them (two row tiles of 128 elements in BFLOAT8_B with 66 spilled
// registers: 185 us instead of 83).  Hence the scheduling barriers between products of different operands.  One and two row tiles have no spilled
// registers; five row tiles of 64 elements do not fit: 46 are spilled for BFLOAT8_B, 14 for bf16, and some are reloaded in every block.
// ---------------------------------------------------------------------------------------------------------------------------------
template <int D, bool PACKED> struct StreamShape {
    static constexpr int SLABS = D / 32, TILE_BYTES = PACKED ? 1088 : 2048;
    static constexpr int COLS = PACKED ? (D + 63) / 64 * 4 : D / 16;               // accumulators of four values
    // packed tile in LDS: [even tile 0 | odd tile 32] + face column * 528 + face row * 256 + row * 16, exponents at 1088: the words that
    // 32 lanes read at once (2 tiles, 2 face columns, 2 groups of rows, 4 words) lie in 32 banks
    static constexpr int STAGE = PACKED ? SLABS * 1152 : D * 64;
    static constexpr int CHUNKS = SLABS * TILE_BYTES / 16, LOADS = (CHUNKS + 63) / 64;
};
template <int D, bool PACKED> struct StreamBlock {
    using S = StreamShape<D, PACKED>;
    u32x4 k[2][PACKED ? 1 : S::SLABS];
    u32x2v codes[2][PACKED ? S::SLABS : 1];
    uint32_t exps[2][PACKED ? S::SLABS : 1];
    u32x4 v[S::LOADS];
    __device__ __forceinline__ void load_values(const uint8_t *base, int lane) {
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) v[i] = *reinterpret_cast<const u32x4 *>(base + min(i * 64 + lane, S::CHUNKS - 1) * 16);
    }
    __device__ __forceinline__ void load(const uint8_t *keys, const uint8_t *values, uint64_t at, int lane) {
        const uint8_t *base = keys + at;
        const int x = lane & 15, g = lane >> 4;
#pragma unroll
        for (int th = 0; th < 2; ++th)
#pragma unroll
            for (int s = 0; s < S::SLABS; ++s) {
                if constexpr (PACKED) {
                    codes[th][s] = *reinterpret_cast<const u32x2v *>(base + s * 1088 + 64 + (th * 2 + (g >> 1)) * 256 + x * 16 + (g & 1) * 8);
                    exps[th][s] = base[s * 1088 + (th * 2 + (g >> 1)) * 16 + x];
                } else {
                    k[th][s] = *reinterpret_cast<const u32x4 *>(base + s * 2048 + th * 1024 + (g >> 1) * 512 + x * 32 + (g & 1) * 16);
                }
            }
        load_values(values + at, lane);
    }
};

template <int D, int MT, bool PACKED>
__global__ __launch_bounds__(256, (MT <= 2 && D <= 128) || D == 64 ? 2 : 1) void paged_attention_stream_kernel(const AttentionDev p) {
    using S = StreamShape<D, PACKED>;
    constexpr int ROWS = MT * 16, NACC = MT * S::COLS;          // NACC quads of accumulators
    constexpr int JOIN = 2 * (NACC * 16 + MT * 8) * 64;         // bytes: two wavefronts' state
    constexpr int LDS = 4 * S::STAGE > JOIN ? 4 * S::STAGE : JOIN;
    constexpr bool Q_IN_LDS = MT > 2 || (MT == 2 && D > 64);    // the registers are needed for the next block
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    __shared__ u32x4 queries[Q_IN_LDS ? MT * S::SLABS * 64 : 1];
    __shared__ uint32_t flag;
    const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Plan plan = make_plan<ROWS, 4>(p);

    typedef __attribute__((address_space(3))) uint8_t lds_byte;
    lds_byte *const stage = (lds_byte *)lds + wave * S::STAGE;
    uint32_t to[S::LOADS];                                      // where this lane's pieces of a block's values go
#pragma unroll
    for (int n = 0; n < S::LOADS; ++n) {
        const uint32_t c = n * 64 + lane, tile = c / 68, cc = c % 68, f = (cc - 4) >> 4, r = (cc - 4) & 15;
        to[n] = !PACKED ? c * 16 : tile * 1152 + (cc < 4 ? 1088 + cc * 16 : (tile & 1) * 32 + (f & 1) * 528 + (f >> 1) * 256 + r * 16);
    }
    const uint32_t out_width = p.heads * D;

    for (uint32_t index = blockIdx.x; index < plan.pieces; index += gridDim.x) {
        Piece pc;
        if (!piece_at<ROWS>(p, plan, index, pc)) continue;
        // this wavefront's blocks: pc.begin + wave, + 4, ...; the first one is asked for before the queries
        const uint32_t mine = pc.end > pc.begin + wave ? (pc.end - pc.begin - wave + 3) / 4 : 0;
        Blocks<4, S::SLABS * S::TILE_BYTES> blocks;
        StreamBlock<D, PACKED> b;
        uint64_t at = 0;
        bool there = false;
        auto request = [&](uint32_t i) __attribute__((always_inline)) {
            if (i >= mine) return;
            if ((i & 63) == 0) blocks.load(p, pc, pc.begin + wave + i * 4);
            at = blocks.at(i & 63);
            there = blocks.has(i & 63);
            b.load(p.keys, p.values, at, lane);
        };
        request(0);
        bf16x8 q[Q_IN_LDS ? 1 : MT][S::SLABS];
        uint32_t row_token[MT];
        const Rows rows(pc.token0, p.group);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            uint32_t head;
            rows.at(pc.row0 + min((uint32_t)(mt * 16 + x), pc.rows - 1), row_token[mt], head);               // rows past the last repeat it
            head += pc.kv * p.group;
#pragma unroll
            for (int s = 0; s < S::SLABS; ++s) {
                if (Q_IN_LDS && (mt * S::SLABS + s) % 4 != wave) continue;
                const u32x4 w = *reinterpret_cast<const u32x4 *>(p.rows + row_bytes_at(pc.q.start + row_token[mt], p.width, p.query_column + head * D + s * 32 + g * 8, p.tiled)) ^ u32x4{p.flip, p.flip, p.flip, p.flip};
                if constexpr (Q_IN_LDS) queries[(mt * S::SLABS + s) * 64 + lane] = w;
                else q[mt][s] = __builtin_bit_cast(bf16x8, w);
            }
        }
        auto query = [&](int mt, int s) __attribute__((always_inline)) {
            if constexpr (Q_IN_LDS) return __builtin_bit_cast(bf16x8, queries[(mt * S::SLABS + s) * 64 + lane]);
            else return q[mt][s];
        };
        f32x4 acc[MT][S::COLS];
        float m[MT], l[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt] = -INFINITY; l[mt] = 0.f;
#pragma unroll
            for (int c = 0; c < S::COLS; ++c) acc[mt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const uint32_t pos_min = pc.q.cached + pc.token0, pos_max = pc.q.cached + pc.token1;
        const uint32_t first_min = first_seen(p, pos_min), first_max = first_seen(p, pos_max);

        // values of a block into LDS
        auto put_values = [&](const u32x4 (&v)[S::LOADS]) __attribute__((always_inline)) {
            lanes_in_order();
#pragma unroll
            for (int n = 0; n < S::LOADS; ++n)
                if (n + 1 < S::LOADS || S::CHUNKS % 64 == 0 || n * 64 + lane < S::CHUNKS) *(__attribute__((address_space(3))) u32x4 *)(stage + to[n]) = v[n];
            lanes_in_order();
        };
        // bf16 values: zeros for the tokens outside [low, high]
        auto clear_values = [&](u32x4 (&v)[S::LOADS], uint32_t token0, uint32_t low, uint32_t high) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < S::LOADS; ++n) {
                const uint32_t t = token0 + (n & 1) * 16 + (lane >> 1 & 15);               // 64 pieces are a face row of a tile
                if (t < low || t > high) v[n] = u32x4{0, 0, 0, 0};
            }
        };
        auto value_operand = [&](int c) __attribute__((always_inline)) {
            union { s16x4 half[2]; bf16x8 v; } u;
#pragma unroll
            for (int th = 0; th < 2; ++th)
                u.half[th] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(stage + (c >> 1) * 2048 + th * 1024 + (c & 1) * 512 + lane * 8));
            return u.v;
        };
        // acc += values . weights
        auto add_values = [&](const bf16x8 (&w)[MT]) __attribute__((always_inline)) {
            auto product = [&](const bf16x8 v, int c) __attribute__((always_inline)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w[mt], acc[mt][c], 0, 0, 0);
            };
            if constexpr (PACKED) {
#pragma unroll
                for (int grp = 0; grp < S::COLS / 4; ++grp) {
                    const int tile = min(grp * 2 + (x >> 3), S::SLABS - 1);                  // columns past the head: any, not stored
                    lds_byte *const at = stage + tile * 1152, *const face = at + (tile & 1) * 32 + (x >> 2 & 1) * 528 + g * 64 + (x & 3) * 4;
                    uint32_t words[8], mags[8];
                    float scale[8];
#pragma unroll
                    for (int th = 0; th < 2; ++th) {
                        const uint32_t e = *(__attribute__((address_space(3))) uint32_t *)(at + 1088 + (th * 2 + (x >> 2 & 1)) * 16 + g * 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            words[th * 4 + i] = *(__attribute__((address_space(3))) uint32_t *)(face + th * 256 + i * 16);
                            mags[th * 4 + i] = words[th * 4 + i] & 0x7f7f7f7fu;
                            scale[th * 4 + i] = block_scale(e >> (8 * i) & 0xffu);
                        }
                    }
                    product(weights_operand8<0>(words, mags, scale), grp * 4 + 0);
                    product(weights_operand8<1>(words, mags, scale), grp * 4 + 1);
                    product(weights_operand8<2>(words, mags, scale), grp * 4 + 2);
                    product(weights_operand8<3>(words, mags, scale), grp * 4 + 3);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                bf16x8 ring[AHEAD];
#pragma unroll
                for (int c = 0; c < AHEAD; ++c) ring[c] = value_operand(c);
#pragma unroll
                for (int c = 0; c < S::COLS; ++c) {
                    product(ring[c % AHEAD], c);
                    if (c + AHEAD < S::COLS) ring[c % AHEAD] = value_operand(c + AHEAD);
                    keep_order();
                }
            }
        };
        // `next` is called once the block's registers are free
        auto work_on = [&](StreamBlock<D, PACKED> &b, uint32_t block, uint64_t at, auto &&next) __attribute__((always_inline)) {
            const uint32_t token0 = block * 32;
            const bool all_seen = token0 >= first_max && token0 + 31 <= pos_min;
            bool odd = false;                                   // values that are not finite, where rows see different tokens or one ends
            if constexpr (!PACKED) {
                if (__builtin_expect(!(token0 >= first_min && token0 + 31 <= pos_max), 0)) clear_values(b.v, token0, first_min, pos_max);
                if (__builtin_expect(token0 + 31 >= pos_min || (!all_seen && pc.token0 != pc.token1), 0)) {
                    uint32_t any = 0;
#pragma unroll
                    for (int n = 0; n < S::LOADS; ++n) {
                        const u32x4 taken = b.v[n] ^ pick(b.v[n], KEEP_FINITE);
                        b.v[n] ^= taken;
                        any |= taken[0] | taken[1] | taken[2] | taken[3];
                    }
                    odd = __ballot(any != 0) != 0;
                }
            }
            put_values(b.v);
            f32x4 s[2][MT];
#pragma unroll
            for (int th = 0; th < 2; ++th) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[th][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int sl = 0; sl < S::SLABS; ++sl) {
                    bf16x8 k;
                    if constexpr (PACKED) k = __builtin_bit_cast(bf16x8, expand8(b.codes[th][sl][0], b.codes[th][sl][1], block_scale(b.exps[th][sl])));
                    else k = __builtin_bit_cast(bf16x8, b.k[th][sl]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) s[th][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, query(mt, sl), s[th][mt], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!odd) next();
            // weights of a row tile rounded to bf16, or what the rounding took off; their sum goes to l
            auto weights = [&](int mt, bool rest) __attribute__((always_inline)) {
                const float base = floor_of(m[mt]);
                union { uint32_t words[4]; bf16x8 v; } u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(s[i >> 1][mt][(i & 1) * 2 + j], p.scale, -base));
                    uint32_t rounded = f32x2_to_bf16x2_rne(e[0], e[1]);
                    if (rest) rounded = f32x2_to_bf16x2_rne(e[0] - __uint_as_float(rounded << 16), e[1] - __uint_as_float(rounded & 0xffff0000u));
                    u.words[i] = rounded;
                    l[mt] = add_pair(rounded, l[mt]);
                }
                return u.v;
            };
            bf16x8 w[MT];
            float top[MT];
            bool move = false;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                if (!all_seen) {
                    const uint32_t pos = in_table(pc.q.cached + row_token[mt]), first = in_table(first_seen(p, pc.q.cached + row_token[mt]));
                    const int from = (int)(first - token0) - g * 4, to = (int)(pos - token0) - g * 4;
#pragma unroll
                    for (int th = 0; th < 2; ++th)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (th * 16 + i < from || th * 16 + i > to) s[th][mt][i] = -INFINITY;
                }
                top[mt] = fmaxf(fmaxf(s[0][mt][0], s[0][mt][1]), fmaxf(s[0][mt][2], s[0][mt][3]));
                top[mt] = fmaxf(top[mt], fmaxf(fmaxf(s[1][mt][0], s[1][mt][1]), fmaxf(s[1][mt][2], s[1][mt][3])));
                top[mt] = max_over_quarters(top[mt]) * p.scale;
                move |= top[mt] > m[mt] + LAZY || (m[mt] == -INFINITY && top[mt] > m[mt]);
            }
            if (__ballot(move)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const float next = fmaxf(m[mt], top[mt]), shrink = __builtin_amdgcn_exp2f(m[mt] - floor_of(next));
                    m[mt] = next;
                    l[mt] *= shrink;
#pragma unroll
                    for (int c = 0; c < S::COLS; ++c) acc[mt][c] *= shrink;
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) w[mt] = weights(mt, false);
            add_values(w);
            if (__builtin_expect(token0 + 31 >= pos_min, 0)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) w[mt] = weights(mt, true);
                add_values(w);
            }
            if (__builtin_expect(odd, 0)) {
                if constexpr (!PACKED) {
                    for (int down = 0; down < 2; ++down) {
                        b.load_values(p.values + at, lane);
                        clear_values(b.v, token0, first_min, pos_max);
#pragma unroll
                        for (int n = 0; n < S::LOADS; ++n) b.v[n] = pick(b.v[n], down ? ONES_DOWN : ONES_UP);
                        put_values(b.v);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            const uint32_t pos = in_table(pc.q.cached + row_token[mt]), first = in_table(first_seen(p, pc.q.cached + row_token[mt]));
                            int from = (int)(first - token0) - g * 4, to = (int)(pos - token0) - g * 4;
                            asm volatile("" : "+v"(from), "+v"(to));            // compared here, not held in registers from before the loop
                            union { uint32_t words[4]; bf16x8 v; } seen;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int t = (i >> 1) * 16 + (i & 1) * 2;
                                seen.words[i] = (t >= from && t <= to ? 0x3f80u : 0u) | (t + 1 >= from && t + 1 <= to ? 0x3f800000u : 0u);
                            }
#pragma unroll
                            for (int c = 0; c < S::COLS; ++c) {
                                const f32x4 count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value_operand(c), seen.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (count[i] > 0.f) acc[mt][c][i] += down ? -INFINITY : INFINITY;
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    }
                }
                next();
            }
        };

        if (Q_IN_LDS) __syncthreads();
        for (uint32_t i = 0; i < mine; ++i) {
            if (there) work_on(b, pc.begin + wave + i * 4, at, [&]() __attribute__((always_inline)) { request(i + 1); });
            else request(i + 1);
        }

        // columns c of row tile mt that this lane has, divided by the sum of the weights: four of bf16, sixteen of block floats
        auto store = [&](int mt, int c, const f32x4 *v, float sum) __attribute__((always_inline)) {
            if ((uint32_t)(mt * 16 + x) >= pc.rows) return;
            uint32_t token, column;
            rows.at(pc.row0 + mt * 16 + x, token, column);
            column = (pc.kv * p.group + column) * D;
            const float by = sum == 0.f ? 0.f : 1.f / sum;
            if constexpr (PACKED) {
                const uint32_t d = c * 64 + g * 16;            // 4 i + byte
                if (d >= (uint32_t)D) return;
                uint32_t words[8];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) words[2 * i + h] = f32x2_to_bf16x2_rne(v[2 * h][i] * by, v[2 * h + 1][i] * by);
                u32x4 *const o = reinterpret_cast<u32x4 *>(p.out + row_bytes_at(pc.q.start + token, out_width, column + d, p.tiled));
                o[0] = u32x4{words[0], words[1], words[2], words[3]};
                o[1] = u32x4{words[4], words[5], words[6], words[7]};
            } else {
                *reinterpret_cast<u32x2v *>(p.out + row_bytes_at(pc.q.start + token, out_width, column + c * 16 + g * 4, p.tiled)) =
                    u32x2v{f32x2_to_bf16x2_rne(v[0][0] * by, v[0][1] * by), f32x2_to_bf16x2_rne(v[0][2] * by, v[0][3] * by)};
            }
        };
        // ---- join: wavefronts 2, 3 into 0, 1, then 1 into 0; afterwards wavefront 0 has it all -----------------------------------
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) l[mt] = sum_over_quarters(l[mt]);
        auto take = [&](int mt, float m2, float l2, auto &&other) __attribute__((always_inline)) {
            const float next = fmaxf(m[mt], m2), mine_by = __builtin_amdgcn_exp2f(m[mt] - floor_of(next)), other_by = __builtin_amdgcn_exp2f(m2 - floor_of(next));
            m[mt] = next;
            l[mt] = l[mt] * mine_by + l2 * other_by;
#pragma unroll
            for (int c = 0; c < S::COLS; ++c) acc[mt][c] = acc[mt][c] * mine_by + other(c) * other_by;
        };
        auto join_waves = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int half = 2; half >= 1; half >>= 1) {
                __syncthreads();
                float *const state = reinterpret_cast<float *>(lds) + (wave % half) * (JOIN / 8);
                f32x4 *const quads = reinterpret_cast<f32x4 *>(state) + lane;
                float2 *const ml = reinterpret_cast<float2 *>(state + NACC * 256) + lane;
                if (wave >= half && wave < 2 * half) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        ml[mt * 64] = make_float2(m[mt], l[mt]);
#pragma unroll
                        for (int c = 0; c < S::COLS; ++c) quads[(mt * S::COLS + c) * 64] = acc[mt][c];
                    }
                }
                __syncthreads();
                if (wave < half) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const float2 o = ml[mt * 64];
                        take(mt, o.x, o.y, [&](int c) { return quads[(mt * S::COLS + c) * 64]; });
                    }
                }
            }
        };
        join_waves();
        if (pc.parts > 1) {
            constexpr uint32_t SLOT = (NACC + MT) * 1024;
            const bool fits = pc.slot + pc.parts <= p.slots;       // always: the plan makes fewer than two slots to a piece that it aims at
            if (wave == 0 && fits) {
                uint8_t *const at = p.partial + (uint64_t)(pc.slot + pc.part) * SLOT + lane * 16;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    put_quad(at + mt * 1024, f32x4{m[mt], l[mt], 0.f, 0.f});
#pragma unroll
                    for (int c = 0; c < S::COLS; ++c) put_quad(at + (MT + mt * S::COLS + c) * 1024, acc[mt][c]);
                }
            }
            if (!fits || !last_of(p, pc, &flag)) { __syncthreads(); continue; }
            // A wavefront takes every fourth of the columns that a lane stores at once.  A load from another XCD's stores takes 1.7 us, so as many
            // parts as there are registers for are on their way together; the last part stands in for those behind it
            constexpr int TOGETHER = PACKED ? 4 : 1, PER_TILE = S::COLS / TOGETHER, ITEMS = MT * PER_TILE;
            constexpr int MINE = PACKED || ITEMS <= 4 ? 1 : 2, GROUP = PACKED ? 6 : 8;                   // items, parts at a time
            const uint8_t *const at = p.partial + (uint64_t)pc.slot * SLOT + lane * 16;
#pragma unroll 1
            for (int first = wave; first < ITEMS; first += 4 * MINE) {
                int mt[MINE], column[MINE];
                float top[MINE], sum[MINE];
                f32x4 out[MINE][TOGETHER];
#pragma unroll
                for (int n = 0; n < MINE; ++n) {
                    const int item = min(first + n * 4, ITEMS - 1);
                    mt[n] = item / PER_TILE;
                    column[n] = item % PER_TILE;
                    top[n] = -INFINITY;
                    sum[n] = 0.f;
#pragma unroll
                    for (int t = 0; t < TOGETHER; ++t) out[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll 1
                for (uint32_t part = 0; part < pc.parts; part += GROUP) {
                    float2 ml[GROUP][MINE];
                    f32x4 o[GROUP][MINE][TOGETHER];
#pragma unroll
                    for (int k = 0; k < GROUP; ++k) {
                        const uint8_t *const from = at + (uint64_t)min(part + k, pc.parts - 1) * SLOT;
#pragma unroll
                        for (int n = 0; n < MINE; ++n) {
                            ml[k][n] = *reinterpret_cast<const float2 *>(from + mt[n] * 1024);
#pragma unroll
                            for (int t = 0; t < TOGETHER; ++t) o[k][n][t] = get_quad(from + (MT + (mt[n] * PER_TILE + column[n]) * TOGETHER + t) * 1024);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);          // all of them, before the first is waited for
#pragma unroll
                    for (int n = 0; n < MINE; ++n) {
                        float next = top[n];
#pragma unroll
                        for (int k = 0; k < GROUP; ++k) next = fmaxf(next, ml[k][n].x);
                        const float base = floor_of(next), shrink = __builtin_amdgcn_exp2f(top[n] - base);
                        top[n] = next;
                        sum[n] *= shrink;
#pragma unroll
                        for (int t = 0; t < TOGETHER; ++t) out[n][t] *= shrink;
#pragma unroll
                        for (int k = 0; k < GROUP; ++k) {
                            if (part + k >= pc.parts) break;
                            const float by = __builtin_amdgcn_exp2f(ml[k][n].x - base);
                            sum[n] += ml[k][n].y * by;
#pragma unroll
                            for (int t = 0; t < TOGETHER; ++t) out[n][t] += o[k][n][t] * by;
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < MINE; ++n)
                    if (first + n * 4 < ITEMS) store(mt[n], column[n], out[n], sum[n]);
            }
        } else if (wave == 0) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int c = 0; c < S::COLS / (PACKED ? 4 : 1); ++c) store(mt, c, &acc[mt][c * (PACKED ? 4 : 1)], l[mt]);
        }
        __syncthreads();                                        // LDS is the next piece's
    }
    if (p.zero_rows) clear_rows(p, D, plan.begin, plan.end);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Many rows (chunks, prompts): bound by the vector ALU beside the matrix cores.  Eight wavefronts (four where heads have 256 elements) of 32 rows each share a
// unit and its keys and values, 64 tokens (32) a step, which go through LDS as bf16; block floats are expanded on the way,
// once for all rows of the unit.  v_mfma_f32_32x32x16_bf16.
//   phases   a step is a phase of vector work (masks, softmax, the next tokens into LDS) and one of matrix work (values of this step, then
//            keys of the next).  The two wavefronts of a SIMD are a phase apart, kept there by a barrier after every phase: one has the
//            matrix cores while the other has the vector ALU.  In step, both wait for the same unit: 615 us instead of 527 for two
//            prompts of 5000 tokens (BFLOAT8_B cache, window 4096, 32 heads on 8 key heads), 106 instead of 94 for 512 tokens behind 7680
//            (bf16).  With the wavefronts in their matrix phase not preferred (s_setprio): 560 and 97.  The additions of the
//            weights belong into the matrix phase, although v_dot2_f32_bf16 takes 20 cycles beside products: 566 and 102 us in the other
//   rate     those prompts: 527 us = 0.82 PFLOP/s of what the masks leave (the largest of several cards' rates: 590 us and 0.73 on another, and
//            on any under a profiler), a large product reaches 1.22; matrix cores busy 44 % of the time,
//            vector ALU 66 %: an instruction takes it 8 cycles while the matrix cores work, and a step of 32 products (1024 cycles) has 300
//            of them for each wavefront, 140 for expanding block floats, 32 exponentials among the rest
//   LDS      three buffers each for keys and values.  In vector phase i the keys of step i + 2 and the values of step i + 1 are written, read by
//            either half of the workgroup until the end of the matrix phases i + 1, which are one phase apart
//   keys     16-byte chunk (row r, half h) of a face lies at r * 32 + (h ^ (r / 8)) * 16: what a pass of a ds_read_b128 touches lies
//            in different banks
//   values   read transposed (ds_read_b64_tr_b16); the 128-byte halves of the row groups are exchanged in the right-hand faces, for the
//            same reason
// ---------------------------------------------------------------------------------------------------------------------------------
template <int D, bool PACKED> struct TileShape {
    static constexpr int WAVES = D == 256 ? 4 : 8;              // heads of 256 elements need all the registers of their SIMD
    static constexpr int NB = D == 256 ? 1 : 2;                 // blocks of 32 tokens per step
    static constexpr int BLOCK = D * 64, HALF = NB * BLOCK;     // bytes of a block, and of the keys or the values of a step
    static constexpr int TILE_BYTES = PACKED ? 1088 : 2048, ROW_BYTES = D / 32 * TILE_BYTES;
    // pieces of a step's keys, and of its values: 16 bytes of bf16, or a face row of block floats
    static constexpr int PIECES = PACKED ? NB * 2 * D : NB * D * 4, EACH = (PIECES + WAVES * 64 - 1) / (WAVES * 64);
};

// End of a phase: what this wavefront has written to LDS is there.  Loads from memory stay in flight.
__device__ __forceinline__ void end_phase() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int D, bool PACKED>
__global__ __launch_bounds__((TileShape<D, PACKED>::WAVES * 64)) void paged_attention_tile_kernel(const AttentionDev p) {
    using S = TileShape<D, PACKED>;
    constexpr int WAVES = S::WAVES, THREADS = WAVES * 64, ROWS = WAVES * 32, NB = S::NB, SLABS = D / 16, DB = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[6 * S::HALF];                // keys, then values, three buffers each
    __shared__ uint32_t flag;
    const int lane = threadIdx.x & 63, c = lane & 31, kh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool second = WAVES == 8 && wave >= 4;                // the half that runs a phase behind
    typedef __attribute__((address_space(3))) uint8_t lds_byte;
    const Plan plan = make_plan<ROWS, NB>(p);
    const uint32_t out_width = p.heads * D;

    for (uint32_t index = blockIdx.x; index < plan.pieces; index += gridDim.x) {
        Piece pc;
        if (!piece_at<ROWS>(p, plan, index, pc)) continue;
        const bool idle = (uint32_t)wave * 32 >= pc.rows;       // a wavefront without rows only moves keys and values
        uint32_t row_token, head;
        Rows(pc.token0, p.group).at(pc.row0 + min((uint32_t)(wave * 32 + c), pc.rows - 1), row_token, head);
        head += pc.kv * p.group;
        bf16x8 q[SLABS];
#pragma unroll
        for (int s = 0; s < SLABS; ++s) {
            u32x4 w = *reinterpret_cast<const u32x4 *>(p.rows + row_bytes_at(pc.q.start + row_token, p.width, p.query_column + head * D + s * 16 + kh * 8, p.tiled));
            q[s] = __builtin_bit_cast(bf16x8, w ^ u32x4{p.flip, p.flip, p.flip, p.flip});
        }
        f32x16 acc[DB], s[NB];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
        const uint32_t pos = in_table(pc.q.cached + row_token), first = in_table(first_seen(p, pc.q.cached + row_token));
        // tokens that some row, and that every row, sees: of the unit and of this wavefront
        const uint32_t pos_max = pc.q.cached + pc.token1, first_min = first_seen(p, pc.q.cached + pc.token0);
        const uint32_t unit_pos_min = pc.q.cached + pc.token0, unit_first_max = first_seen(p, pos_max);
        const uint32_t wave_pos_min = pc.q.cached + (pc.row0 + min((uint32_t)wave * 32, pc.rows - 1)) / p.group, wave_pos_max = pc.q.cached + (pc.row0 + min((uint32_t)wave * 32 + 31, pc.rows - 1)) / p.group;
        const uint32_t wave_first_min = first_seen(p, wave_pos_min), wave_first_max = first_seen(p, wave_pos_max);
        const uint32_t steps = (pc.end - pc.begin + NB - 1) / NB;
        auto token_of = [&](uint32_t step) { return (pc.begin + step * NB) * 32; };
        // steps [step_from, step_to) have something for this wavefront
        const uint32_t step_to = idle || wave_pos_max < token_of(0) ? 0 : min((wave_pos_max / 32 - pc.begin) / NB + 1, steps);
        const uint32_t step_from = wave_first_min / 32 > pc.begin ? min((wave_first_min / 32 - pc.begin) / NB, step_to) : 0;
        // rows of the unit see different parts of the step, or one ends in it
        auto uneven = [&](uint32_t step) { return !(token_of(step) >= unit_first_max && token_of(step) + NB * 32 - 1 < unit_pos_min); };

        // ---- keys and values: memory -> registers -> LDS ------------------------------------------------------------------------------
        Blocks<1, S::ROW_BYTES> blocks;
        uint64_t keys_at[NB], values_at[NB];                    // of the step whose keys, and whose values, are asked for next
        uint32_t have = 0;                                      // which blocks of four steps, from the current one on, have pages: bit NB * step + block
        u32x4 kreg[S::EACH], vreg[S::EACH];
        uint32_t kexp[S::EACH], vexp[S::EACH];
        const uint32_t thread = threadIdx.x & (THREADS - 1);    // with its range for the compiler to see
        // piece i of this thread: block of the step, byte in the block's tiles (keys and values alike), token of the block
        auto place = [&](int i, uint32_t &block, uint32_t &from, uint32_t &token, uint32_t &exponent) __attribute__((always_inline)) {
            const uint32_t n = min(thread + i * (uint32_t)THREADS, (uint32_t)S::PIECES - 1), per_block = S::PIECES / NB;
            block = n / per_block;
            const uint32_t within = n % per_block;
            if (PACKED) {
                const uint32_t tile = within >> 6, face = within >> 4 & 3, r = within & 15;
                from = tile * 1088 + 64 + face * 256 + r * 16;
                exponent = tile * 1088 + face * 16 + r;
                token = (face >> 1) * 16 + r;
            } else {
                from = within * 16;
                exponent = 0;
                token = (within >> 6 & 1) * 16 + (within >> 1 & 15);
            }
        };
        auto load = [&](const uint8_t *tensor, const uint64_t (&at)[NB], u32x4 (&v)[S::EACH], uint32_t (&e)[S::EACH]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < S::EACH; ++i) {
                uint32_t block, from, token, exponent;
                place(i, block, from, token, exponent);
                const uint8_t *base = tensor + (NB == 2 && block ? at[NB - 1] : at[0]);
                v[i] = *reinterpret_cast<const u32x4 *>(base + from);
                e[i] = PACKED ? base[exponent] : 0u;
            }
        };
        // where the keys of `step` lie, which is `ahead` of the current one; behind the last step, page 0
        auto refill = [&](uint32_t step) __attribute__((always_inline)) {
            if ((step * NB & 63) == 0) blocks.load(p, pc, pc.begin + step * NB);
        };
        auto look_up = [&](uint32_t step, int ahead) __attribute__((always_inline)) {
            const uint32_t i = step * NB & 63;
            have |= (uint32_t)(blocks.pages >> i & ((1u << NB) - 1)) << (ahead * NB);
#pragma unroll
            for (int b = 0; b < NB; ++b) keys_at[b] = blocks.at(i + b);
        };
        auto put = [&](uint32_t to, const u32x4 (&v)[S::EACH], const uint32_t (&e)[S::EACH], bool values) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < S::EACH; ++i) {
                const uint32_t n = thread + i * (uint32_t)THREADS, block = n / (S::PIECES / NB), within = n % (S::PIECES / NB);
                if (S::PIECES % THREADS && n >= (uint32_t)S::PIECES) break;
                lds_byte *const face_at = (lds_byte *)lds + to + block * S::BLOCK + (PACKED ? within >> 4 : within >> 5) * 512;
                // 16-byte chunk of a face, and where it goes: see above
                auto chunk = [&](uint32_t at, uint32_t face, const u32x4 &w) __attribute__((always_inline)) {
                    const uint32_t where = values ? at ^ ((face & 1) * 8) : (at & ~1u) | ((at & 1) ^ (at >> 4));
                    *(__attribute__((address_space(3))) u32x4 *)(face_at + where * 16) = w;
                };
                if constexpr (PACKED) {
                    const float scale = block_scale(e[i]);
                    chunk((within & 15) * 2, within >> 4, expand8(v[i][0], v[i][1], scale));
                    chunk((within & 15) * 2 + 1, within >> 4, expand8(v[i][2], v[i][3], scale));
                } else {
                    chunk(within & 31, within >> 5, v[i]);
                }
            }
        };
        // bf16 values: zeros for tokens that no row of the unit sees
        auto clear_values = [&](uint32_t token0, uint32_t pages) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < S::EACH; ++i) {
                uint32_t block, from, token, exponent;
                place(i, block, from, token, exponent);
                const uint32_t t = token0 + block * 32 + token;
                if (t < first_min || t > pos_max || !(pages >> block & 1)) vreg[i] = u32x4{0, 0, 0, 0};
            }
        };
        uint32_t odd = 0;                                       // values that are not finite, in uneven steps
        auto put_values = [&](uint32_t to, uint32_t step, int ahead) __attribute__((always_inline)) {
            if constexpr (!PACKED) {
                const uint32_t token0 = token_of(step), pages = have >> (ahead * NB) & ((1u << NB) - 1);
                if (__builtin_expect(!(token0 >= first_min && token0 + NB * 32 - 1 <= pos_max && pages == (1u << NB) - 1), 0)) clear_values(token0, pages);
                if (__builtin_expect(uneven(step), 0)) {
#pragma unroll
                    for (int i = 0; i < S::EACH; ++i) {
                        const u32x4 taken = vreg[i] ^ pick(vreg[i], KEEP_FINITE);
                        vreg[i] ^= taken;
                        odd |= taken[0] | taken[1] | taken[2] | taken[3];
                    }
                }
            }
            put(to, vreg, vexp, true);
        };

        // ---- products -----------------------------------------------------------------------------------------------------------------
        const uint32_t key_at = (c >> 4) * 1024 + (c & 15) * 32 + ((kh ^ (c >> 3 & 1)) * 16);
        const uint32_t fc = lane >> 4 & 1, value_at = 3 * S::HALF + fc * 512 + ((kh * 128 + (lane & 15) * 8) ^ (fc * 128));
        constexpr int N_KEYS = NB * SLABS, N_VALUES = DB * 2 * NB;
        auto key_operand = [&](uint32_t buffer, int i) __attribute__((always_inline)) {
            const int b = i / SLABS, sl = i % SLABS;
            return __builtin_bit_cast(bf16x8, *(__attribute__((address_space(3))) u32x4 *)((lds_byte *)lds + buffer + key_at + b * S::BLOCK + (sl >> 1) * 2048 + (sl & 1) * 512));
        };
        // elements 32 (i / 2 NB) .. + 31, tokens 16 (i % 2 NB) .. + 15 of the step
        auto value_operand = [&](uint32_t buffer, int i) __attribute__((always_inline)) {
            const int d = i / (2 * NB), b = i / 2 % NB, h = i % 2;
            union { s16x4 half[2]; bf16x8 v; } u;
#pragma unroll
            for (int r = 0; r < 2; ++r)
                u.half[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)((lds_byte *)lds + buffer + value_at + b * S::BLOCK + d * 2048 + h * 1024 + r * 256));
            return u.v;
        };
        bf16x8 ring[AHEAD], w[NB][2];
        auto clear_scores = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
        };
        auto multiply_keys = [&](uint32_t buffer) __attribute__((always_inline)) {         // the ring holds the first operands
            clear_scores();
#pragma unroll
            for (int i = 0; i < N_KEYS; ++i) {
                s[i / SLABS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % AHEAD], q[i % SLABS], s[i / SLABS], 0, 0, 0);
                if (i + AHEAD < N_KEYS) ring[i % AHEAD] = key_operand(buffer, i + AHEAD);
                keep_order();
            }
        };
        // ... and is left with the first operands of the keys in `next`
        auto multiply_values = [&](uint32_t buffer, uint32_t next) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < N_VALUES; ++i) {
                acc[i / (2 * NB)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % AHEAD], w[i / 2 % NB][i % 2], acc[i / (2 * NB)], 0, 0, 0);
                ring[i % AHEAD] = i + AHEAD < N_VALUES ? value_operand(buffer, i + AHEAD) : key_operand(next, i + AHEAD - N_VALUES);
                keep_order();
            }
        };
        static_assert(N_VALUES % AHEAD == 0, "the ring starts over with the keys");
        // weights rounded to bf16, or what the rounding took off; their sum goes to l
        auto weights = [&](bool rest) __attribute__((always_inline)) {
            const float base = floor_of(m);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    union { uint32_t words[4]; bf16x8 v; } u;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float e[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(s[b][h * 8 + 2 * i + j], p.scale, -base));
                        uint32_t rounded = f32x2_to_bf16x2_rne(e[0], e[1]);
                        if (rest) rounded = f32x2_to_bf16x2_rne(e[0] - __uint_as_float(rounded << 16), e[1] - __uint_as_float(rounded & 0xffff0000u));
                        u.words[i] = rounded;
                        l = add_pair(rounded, l);
                    }
                    w[b][h] = u.v;
                }
        };

        uint32_t buffer[3] = {0, S::HALF, 2 * S::HALF};         // of the current step, the next one, the one after
        if (steps) {
            u32x4 k1[S::EACH];
            uint32_t e1[S::EACH];
            refill(0);
            look_up(0, 0);
            load(p.keys, keys_at, kreg, kexp);
            load(p.values, keys_at, vreg, vexp);
            look_up(1, 1);
            load(p.keys, keys_at, k1, e1);
#pragma unroll
            for (int b = 0; b < NB; ++b) values_at[b] = keys_at[b];
            put(buffer[0], kreg, kexp, false);
            put_values(buffer[0] + 3 * S::HALF, 0, 0);
            put(buffer[1], k1, e1, false);
            load(p.values, values_at, vreg, vexp);
            look_up(2, 2);
            load(p.keys, keys_at, kreg, kexp);
            __syncthreads();
            if (second) end_phase();
        }
        // what a step does for the steps behind it: in its vector phase, and, once the registers are free, in its matrix phase
        // (unless there are none: then it moves what is not looked at, which is less work than asking)
        auto bring = [&](uint32_t step) __attribute__((always_inline)) {
            refill(step + 3);
            put_values(buffer[1] + 3 * S::HALF, step + 1, 1);
            put(buffer[2], kreg, kexp, false);
        };
        auto ask = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NB; ++b) values_at[b] = keys_at[b];
            load(p.values, values_at, vreg, vexp);
            look_up(step + 3, 3);
            load(p.keys, keys_at, kreg, kexp);
        };
        auto turn = [&]() __attribute__((always_inline)) {
            have >>= NB;
            const uint32_t done = buffer[0];
            buffer[0] = buffer[1]; buffer[1] = buffer[2]; buffer[2] = done;
        };
        uint32_t step = 0;
        auto pass_by = [&](uint32_t to) __attribute__((always_inline)) {                    // steps with nothing for this wavefront
            for (; step < to; ++step) {
                bring(step);
                end_phase();
                ask(step);
                end_phase();
                turn();
            }
        };
        pass_by(step_from);
        if (step_from < step_to) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) ring[i] = key_operand(buffer[0], i);
            multiply_keys(buffer[0]);
        }
        for (; step < step_to; ++step) {
            // ---- vector work ------------------------------------------------------------------------------------------------------------
            const uint32_t token0 = token_of(step), last = token0 + NB * 32 - 1;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) ring[i] = value_operand(buffer[0], i);
            keep_order();
            if (__builtin_expect(!(token0 >= wave_first_max && last <= wave_pos_min && (have & ((1u << NB) - 1)) == (1u << NB) - 1), 0)) {
                // against constants: the tokens' numbers would be held in registers over all steps
                const int from = (int)(first - token0) - kh * 4, to = (int)(pos - token0) - kh * 4;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int t = b * 32 + (i >> 2) * 8 + (i & 3);
                        if (t < from || t > to || !(have >> b & 1)) s[b][i] = -INFINITY;
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
            top = max_over_halves(top) * p.scale;
            if (__ballot(top > m + LAZY || (m == -INFINITY && top > m))) {
                const float next = fmaxf(m, top), shrink = __builtin_amdgcn_exp2f(m - floor_of(next));
                m = next;
                l *= shrink;
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= shrink;
            }
            weights(false);
            // here, and not where they are used, in the other phase
#pragma unroll
            for (int b = 0; b < NB; ++b) asm volatile("" : "+v"(w[b][0]), "+v"(w[b][1]));
            bring(step);
            end_phase();
            // ---- matrix work ------------------------------------------------------------------------------------------------------------
            ask(step);
            __builtin_amdgcn_s_setprio(1);
            multiply_values(buffer[0], buffer[1]);
            if (__builtin_expect(last >= wave_pos_min, 0)) {
                weights(true);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) ring[i] = value_operand(buffer[0], i);
                multiply_values(buffer[0], buffer[1]);
            }
            multiply_keys(buffer[1]);                           // behind the last step: of whatever is there, and nobody looks
            __builtin_amdgcn_s_setprio(0);
            end_phase();
            turn();
        }
        pass_by(steps);
        if (steps && WAVES == 8 && !second) end_phase();        // both halves have passed as many barriers

        if constexpr (!PACKED) {
            if (__builtin_expect(__syncthreads_or(odd != 0), 0)) {
                // once more over the uneven steps: ones in place of the values that were taken out, counted by those who see them
                for (step = 0; step < steps; ++step) {
                    if (!uneven(step)) continue;
                    uint32_t pages = 0;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t block = pc.begin + step * NB + b;
                        int32_t page = block < pc.end ? p.table[(uint64_t)pc.r * p.max_pages + block / p.page_blocks] : -1;
                        pages |= (uint32_t)((uint32_t)page < p.pages) << b;
                        if ((uint32_t)page >= p.pages) page = 0;
                        values_at[b] = (((uint64_t)page * p.kv_heads + pc.kv) * p.page_blocks + block % p.page_blocks) * S::ROW_BYTES;
                    }
                    for (int down = 0; down < 2; ++down) {
                        load(p.values, values_at, vreg, vexp);
                        clear_values(token_of(step), pages);
#pragma unroll
                        for (int i = 0; i < S::EACH; ++i) vreg[i] = pick(vreg[i], down ? ONES_DOWN : ONES_UP);
                        __syncthreads();
                        put(3 * S::HALF, vreg, vexp, true);
                        __syncthreads();
                        if (step < step_from || step >= step_to) continue;
                        int from = (int)(first - token_of(step)) - kh * 4, to = (int)(pos - token_of(step)) - kh * 4;
                        asm volatile("" : "+v"(from), "+v"(to));                // compared here, not held in registers from before the loop
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                union { uint32_t words[4]; bf16x8 v; } seen;
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int t = b * 32 + h * 16 + (i >> 1) * 8 + (i & 1) * 2;
                                    seen.words[i] = (t >= from && t <= to ? 0x3f80u : 0u) | (t + 1 >= from && t + 1 <= to ? 0x3f800000u : 0u);
                                }
#pragma unroll
                                for (int d = 0; d < DB; ++d) {
                                    f32x16 count;
#pragma unroll
                                    for (int i = 0; i < 16; ++i) count[i] = 0.f;
                                    count = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_operand(0, (d * NB + b) * 2 + h), seen.v, count, 0, 0, 0);
#pragma unroll
                                    for (int i = 0; i < 16; ++i)
                                        if (count[i] > 0.f) acc[d][i] += down ? -INFINITY : INFINITY;
                                    __builtin_amdgcn_sched_barrier(0);
                                }
                            }
                    }
                }
            }
        }

        l = sum_over_halves(l);
        if (pc.parts > 1) {
            constexpr uint32_t PART = (DB * 4 + 1) * 1024, SLOT = WAVES * PART;        // of a wavefront, of a workgroup
            const bool fits = pc.slot + pc.parts <= p.slots;   // always: the plan makes fewer than two slots to a piece that it aims at
            if (fits && !idle) {
                uint8_t *const at = p.partial + (uint64_t)(pc.slot + pc.part) * SLOT + wave * PART + lane * 16;
                put_quad(at, f32x4{m, l, 0.f, 0.f});
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) put_quad(at + (1 + d * 4 + i) * 1024, f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]});
            }
            if (!fits || !last_of(p, pc, &flag)) { __syncthreads(); continue; }
            m = -INFINITY; l = 0.f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
            if (!idle) {
                // Two parts on their way together: a load from another XCD's stores takes 1.7 us.  The last part stands in for one behind it
                const uint8_t *const at = p.partial + (uint64_t)pc.slot * SLOT + wave * PART + lane * 16;
                for (uint32_t part = 0; part < pc.parts; part += 2) {
                    f32x4 ml[2], o[2][DB * 4];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint8_t *const from = at + (uint64_t)min(part + k, pc.parts - 1) * SLOT;
                        ml[k] = get_quad(from);
#pragma unroll
                        for (int i = 0; i < DB * 4; ++i) o[k][i] = get_quad(from + (1 + i) * 1024);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    const float next = fmaxf(m, fmaxf(ml[0][0], ml[1][0])), base = floor_of(next), by = __builtin_amdgcn_exp2f(m - base);
                    const float by0 = __builtin_amdgcn_exp2f(ml[0][0] - base), by1 = part + 1 < pc.parts ? __builtin_amdgcn_exp2f(ml[1][0] - base) : 0.f;
                    m = next;
                    l = l * by + ml[0][1] * by0 + ml[1][1] * by1;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] * by + o[0][d * 4 + i / 4][i & 3] * by0 + (part + 1 < pc.parts ? o[1][d * 4 + i / 4][i & 3] * by1 : 0.f);
                }
            }
        }
        // columns 8 (i / 4) + 4 kh + i % 4 of 32: the swap leaves columns 8 kh .. 8 kh + 7 of a face row in each lane
        const float by = l == 0.f ? 0.f : 1.f / l;
        const bool stored = (uint32_t)(wave * 32 + c) < pc.rows;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int i = f * 8;
                const auto w0 = __builtin_amdgcn_permlane32_swap(f32x2_to_bf16x2_rne(acc[d][i] * by, acc[d][i + 1] * by), f32x2_to_bf16x2_rne(acc[d][i + 4] * by, acc[d][i + 5] * by), false, false);
                const auto w1 = __builtin_amdgcn_permlane32_swap(f32x2_to_bf16x2_rne(acc[d][i + 2] * by, acc[d][i + 3] * by), f32x2_to_bf16x2_rne(acc[d][i + 6] * by, acc[d][i + 7] * by), false, false);
                if (stored) *reinterpret_cast<u32x4 *>(p.out + row_bytes_at(pc.q.start + row_token, out_width, head * D + d * 32 + f * 16 + kh * 8, p.tiled)) = u32x4{w0[0], w1[0], w0[1], w1[1]};
            }
        __syncthreads();                                        // LDS is the next piece's
    }
    if (p.zero_rows) clear_rows(p, D, plan.begin, plan.end);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
namespace {
// Which kernels a step needs: the lengths are on the device, the host knows how many tokens there are for how many requests.
constexpr uint32_t TILE_TARGET = 256;      // of the kernel for many rows: one workgroup per CU
struct Route {
    uint32_t mt = 0;                       // row tiles of the kernel for few rows; 0: not launched
    bool tile = false;
    uint32_t few = 0;                      // most rows of a request that go to the kernel for few rows where both are launched
    uint32_t target = 256, grid = 256;     // of the kernel for few rows: pieces to aim at, workgroups that are resident at once
    size_t slot_bytes = 0, slots = 0;
};
Route route_of(uint32_t tokens, uint32_t requests, uint32_t heads, const PagedCache &c) {
    Route r;
    const uint32_t group = heads / c.kv_heads;
    const uint64_t rows = (uint64_t)((tokens + requests - 1) / std::max(requests, 1u)) * group;       // of an average request
    // Row tiles that a wavefront has registers for, and rows up to which the kernel for few rows is the faster one, in units of that many
    // tiles.  16 users x 4000 tokens, 8 key heads, bf16: 64 elements, 64 rows 44 us (many rows: 58); 96 elements, 40 rows in four tiles 70
    // (65); 128 elements, 32 rows 51 (74), 40 rows in four tiles 191 (74); 256 elements, 64 rows 154 (206), 80 rows 199 (218); two tiles of 256 elements, 17 rows 524 (one: 196).
    const uint32_t most = c.head_dim == 64 ? 5 : c.head_dim == 256 ? 1 : 2;
    const uint32_t limit = c.head_dim == 64 ? 80 : c.head_dim == 256 ? 64 : 32;
    auto tiles_for = [&](uint64_t n) { return std::min(n <= 16 ? 1u : n <= 32 ? 2u : 5u, most); };
    // Few rows per request: the kernel for few rows takes them all, in tiles for an average request.  Many: the other takes them all.  In
    // between, and where more than 8 tokens per request come to more than 512 rows, the step is a mixture: single tokens go to the one, and every
    // request that is more than its tile to the other.  31 single tokens behind 2000 and a prompt, 8 key heads, both kernels (few rows alone):
    // 300 rows of 64 elements 45 us (33), of 128 elements 69 (49); 1000 rows of 64 elements 51 (74); 1200 rows 47 (66).  From 256 rows per request on the
    // launch that has nothing to do costs more than single tokens among the prompts: 8 prompts of 500 tokens 54 us (56), 31 single tokens and
    // a prompt of 4000 257 (259).
    // Both rules know averages only.  A chunk beside so many single tokens that it does not show in them goes to the kernel for few rows, which is right
    // for short ones and not for long ones: 128 elements, bf16 (BFLOAT8_B), 64 single tokens behind 2000 and a chunk of 200 120 us (95), both kernels 144
    // (101); 96 and 512 188 (176), both 204 (159); 127 and 895 behind 7680 411 (543), both 352 (295); 255 and 1500 494 (466), both 476 (344).
    r.tile = rows > limit || (requests > 1 && tokens > 8ull * requests && (uint64_t)tokens * group > 512);
    if (!r.tile) r.mt = tiles_for(rows);
    else if (requests > 1 && rows < 256 && group <= limit) r.mt = tiles_for(group);
    r.few = c.head_dim == 256 ? limit : r.mt * 16;
    const bool packed = c.dtype == TTMI_BFLOAT8_B;
    // Two workgroups fit a CU up to 128 elements.  One piece for each CU fills the memory pipes of bf16, and is less to join than two: 32 users x 2000
    // tokens, 128 elements 44 us (two: 50), 64 elements 24 (30).  The expansion of block floats takes both: 8 users x 26000 tokens 102 us (one: 136).
    // The second workgroup stays for steps of more units than CUs: 64 users x 500 tokens 25 us (28 without it).
    if (c.head_dim <= 128) r.grid = 512;
    if (c.head_dim <= 128 && packed) r.target = 512;
    if (r.mt) {
        const size_t cols = packed ? (c.head_dim + 63) / 64 * 4 : c.head_dim / 16;
        r.slot_bytes = (r.mt * cols + r.mt) * 1024;
        r.slots = 2 * (size_t)r.grid * r.slot_bytes;
    }
    if (r.tile) r.slots = std::max(r.slots, 2 * (size_t)TILE_TARGET * (c.head_dim == 256 ? 4 : 8) * ((size_t)c.head_dim / 32 * 4 + 1) * 1024);
    return r;
}

__global__ void clear_counters_kernel(uint32_t *counters) { counters[blockIdx.x * 256 + threadIdx.x] = 0; }
int clear_counters(void *at, hipStream_t st) {
    hipLaunchKernelGGL(clear_counters_kernel, dim3(COUNTERS / 256), dim3(256), 0, st, (uint32_t *)at);
    return check_launch("clear_counters_kernel");
}

template <int D, int MT> void launch_stream(const AttentionDev &p, uint32_t grid, bool packed, hipStream_t st) {
    if (packed) hipLaunchKernelGGL((paged_attention_stream_kernel<D, MT, true>), dim3(grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attention_stream_kernel<D, MT, false>), dim3(grid), dim3(256), 0, st, p);
}
template <int D, int MOST> void launch_stream(const AttentionDev &p, const Route &route, bool packed, hipStream_t st) {
    if (route.mt == 1) launch_stream<D, 1>(p, route.grid, packed, st);
    else if constexpr (MOST > 1) {
        if (MOST == 2 || route.mt == 2) launch_stream<D, 2>(p, route.grid, packed, st);
        else launch_stream<D, MOST>(p, route.grid, packed, st);
    }
}
template <int D> void launch_tile(const AttentionDev &p, bool packed, hipStream_t st) {
    constexpr uint32_t threads = TileShape<D, false>::WAVES * 64;
    if (packed) hipLaunchKernelGGL((paged_attention_tile_kernel<D, true>), dim3(TILE_TARGET), dim3(threads), 0, st, p);
    else hipLaunchKernelGGL((paged_attention_tile_kernel<D, false>), dim3(TILE_TARGET), dim3(threads), 0, st, p);
}
}  // namespace

size_t paged_attention_workspace_bytes(uint32_t tokens, uint32_t requests, uint32_t heads, const PagedCache &cache) {
    return COUNTERS * 4 + route_of(tokens, requests, heads, cache).slots;
}

int paged_attention(const PagedAttentionArgs &x, hipStream_t st) {
    const PagedCache &c = x.cache;
    AttentionDev p{};
    p.rows = (const uint8_t *)x.rows.data; p.keys = (const uint8_t *)x.key_cache; p.values = (const uint8_t *)x.value_cache;
    p.table = x.step.page_table; p.cached = x.step.cached; p.starts = x.step.row_starts; p.out = (uint8_t *)x.out;
    p.tiled = x.rows.layout == TTMI_TILE;
    p.tokens = x.rows.tokens; p.out_rows = p.tiled ? (x.rows.tokens + 31) / 32 * 32 : x.rows.tokens;
    if (!p.out_rows) return TTMI_OK;
    p.width = x.rows.width; p.query_column = x.query_column; p.requests = x.step.requests; p.max_pages = x.step.max_pages;
    p.pages = c.pages; p.kv_heads = c.kv_heads; p.page_blocks = c.page_size / 32;
    p.heads = x.heads; p.group = x.heads / c.kv_heads; p.window = x.window;
    const bool packed = c.dtype == TTMI_BFLOAT8_B;
    // a scale of zero stands for the smallest number there is: -inf, what is masked, has to stay -inf, and the largest score is 2^-21
    p.scale = std::max(std::fabs(x.scale) * 1.4426950408889634f, 0x1p-149f);
    p.flip = x.scale < 0.f ? 0x80008000u : 0u;

    const Route route = route_of(p.tokens, p.requests, p.heads, c);
    // Without requests there are no pieces, hence no counters and no partial results: rows are cleared, and that needs no memory.
    uint8_t *memory = p.requests ? (uint8_t *)x.workspace : nullptr;
    static std::mutex fresh_guard;         // another thread's launch on this stream stays behind the clearing of a new buffer
    if (memory) {
        if (int rc = clear_counters(memory, st)) return rc;
    } else if (p.requests) {
        const size_t bytes = COUNTERS * 4 + route.slots;
        std::lock_guard<std::mutex> lock(fresh_guard);
        // what is recorded may be replayed on any stream beside any other call: the buffer of the stream that is captured is not its own
        if (stream_is_capturing(st)) return fail(TTMI_ERR_UNSUPPORTED, "paged attention: a captured call takes no scratch of the library's, bring a workspace of %zu bytes", bytes);
        bool fresh = false;
        if (int rc = scratch_get(SCRATCH_PAGED, st, bytes, (void **)&memory, &fresh)) return rc;
        if (fresh)
            if (int rc = clear_counters(memory, st)) return rc;
    }
    if (memory) {
        p.counters = (uint32_t *)memory;
        p.partial = memory + COUNTERS * 4;
    }
    p.zero_rows = 1;
    if (route.mt) {
        p.least_rows = 1;
        p.most_rows = route.tile ? route.few : 0xffffffffu;
        p.target = route.target; p.slots = 2 * route.grid;
        switch (c.head_dim) {
            case 64: launch_stream<64, 5>(p, route, packed, st); break;
            case 96: launch_stream<96, 2>(p, route, packed, st); break;
            case 128: launch_stream<128, 2>(p, route, packed, st); break;
            default: launch_stream<256, 1>(p, route, packed, st); break;
        }
        if (int rc = check_launch("paged_attention_stream_kernel")) return rc;
        p.zero_rows = 0;
    }
    if (route.tile) {
        p.least_rows = route.mt ? route.few + 1 : 1;
        p.most_rows = 0xffffffffu;
        p.target = TILE_TARGET; p.slots = 2 * p.target;
        switch (c.head_dim) {
            case 64: launch_tile<64>(p, packed, st); break;
            case 96: launch_tile<96>(p, packed, st); break;
            case 128: launch_tile<128>(p, packed, st); break;
            default: launch_tile<256>(p, packed, st); break;
        }
        if (int rc = check_launch("paged_attention_tile_kernel")) return rc;
    }
    return TTMI_OK;
}

}  // namespace ttmi
