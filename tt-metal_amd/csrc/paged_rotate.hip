// Queries and keys of a step by their positions: the norm of every head and its rotation, the keys and values straight into their pages.
//
// Row row_starts[r] + i of the activations is token p = cached[r] + i of request r.  For each head x of D elements, where a norm is given,
//   y_d = x_d w_d / sqrt(mean(x^2) + epsilon)
// and, of its first R elements, the pairs (a, b) = (y_i, y_(i + R/2)), or neighbours (y_2i, y_(2i+1)), i < R/2,
//   (a, b) -> m (a cos(p f_i) - b sin(p f_i), b cos(p f_i) + a sin(p f_i))
// in fp32 and rounded once: to bf16, or, for keys of a BFLOAT8_B cache, from fp32 to its codes (by way of bf16 they would be off by up to 2^-9 more).
//
// Bound by memory, for few tokens by the launch and three loads that wait for each other (row starts, length, slot): 32 tokens of 32 heads of 128 elements
// 4.6 us with the launch, with keys, values and norms 5.0.  8206 tokens of 71 heads of 64 elements: 33 us = 4.6 TB/s; 8183 tokens of 32 + 8 + 8 heads of 128 elements with
// norms into BFLOAT8_B: 42 us = 4.4 TB/s, 43 without norms into bf16 (4.6 TB/s; a large copy moves 5.1).  Queries alone, 8000 tokens,
// TILE or rows: 16 heads of 256 elements 31 us = 4.2 TB/s, 32 of 128 the same, 32 of 96 25 = 3.9.  The vector ALU is busy for 67 % of the prompts into BFLOAT8_B: 135 instructions
// for two chunks of a head, 75 for each head's share of requests and angles.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bfp_dequant.h"
#include "paged_cache.h"
#include "ttmi_internal.h"

namespace ttmi {

enum { QUERIES = 0, KEYS = 1, VALUES = 2 };
struct RotateDev {
    const uint8_t *rows;
    uint8_t *out, *cache[2];
    const int32_t *cached, *starts, *slots;
    const float *frequencies, *norm[2];        // of queries, of keys
    uint64_t items;
    uint32_t tokens, out_rows, width, requests;
    uint32_t column[3], heads[3], blocks[3];   // of queries, keys, values: first column, heads, items of a band
    uint32_t each;                             // heads of an item
    uint32_t pages, page_size, turning;
    float epsilon, magnitude;
    int tiled;
};

// Position of row t0 + r, r < ROWS, false where it is no request's.  A row belongs to the request before the first start behind it, and
// the request's rows begin at the largest start up to its own: row starts that do not ascend are read through their running maximum.
// 64 requests at a time, from the first one on, in every item: 4096 tokens of 32 + 8 + 8 heads of 128 elements into a bf16 cache (slots in any order) 28 us as one request or
// 64, 29 as 512, 34 as 2048, 44 as 4096 single tokens; 512 tokens 7.1 as one request, 8.5 as 512.
template <uint32_t ROWS> __device__ __forceinline__ bool position_of(const RotateDev &p, uint32_t t0, uint32_t r, uint32_t &position) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t owner = 0xffffffffu, from = 0, top = 0, open = (1u << ROWS) - 1;      // rows whose request is still looked for
    for (uint32_t base = 0; base <= p.requests && open; base += 64) {
        const uint32_t v = base + lane <= p.requests ? min((uint32_t)max(p.starts[base + lane], 0), p.tokens) : 0xffffffffu;
        const uint32_t to = max(running_max(v), top);
        if (__ballot(to > t0))
#pragma unroll
            for (uint32_t i = 0; i < ROWS; ++i) {
                const uint64_t behind = __ballot(to > t0 + i);
                if (!(open >> i & 1) || !behind) continue;
                open &= ~(1u << i);
                const uint32_t first = (uint32_t)__builtin_ctzll(behind), before = first ? (uint32_t)__builtin_amdgcn_readlane(to, first - 1) : top;
                if (r == i && base + first && base + first <= p.requests) {
                    owner = base + first - 1;
                    from = before;
                }
            }
        top = last_lane(to);
    }
    if (owner == 0xffffffffu) return false;
    position = (uint32_t)max(p.cached[owner], 0) + (t0 + r - from);
    return true;
}

// Sum over the lanes of a token, in each of them: lanes 2 ROWS apart and pairs in TILE layout, neighbours in rows.  By DPP and lane swaps: LDS permutes take 4 us
// of 49 for the prompts below.
template <int CTRL> __device__ __forceinline__ float add_lane(float v) { return v + __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, false)); }
template <uint32_t LANES> __device__ __forceinline__ float sum_over_token(float v, int tiled) {
    v = add_lane<0xb1>(v);                                     // the other of a pair
    if (tiled) {
        if (LANES == 16) v = add_lane<0x128>(v);               // 8 lanes on, of 16
        if (LANES >= 8) {
            const auto o = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(o[0]) + __uint_as_float(o[1]);
        }
        const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(o[0]) + __uint_as_float(o[1]);
    }
    v = add_lane<0x4e>(v);                                     // the other pair of four
    if (LANES >= 8) v = add_lane<0x141>(v);                    // mirrored in 8: the other four
    if (LANES == 16) v = add_lane<0x140>(v);                   // mirrored in 16: the other eight
    return v;
}

// Codes of 8 of a face row's 16 numbers, lowest element in the lowest byte.  Ordinary rows (shared exponent 32 <= E < 255, or nothing but zeros):
// floor(v + 1/2) = trunc(fma(|x|, 2^(133 - E), 1/2 - 2^-25)) with v = |x| 2^(133 - E), for every 24-bit mantissa; 2^7 becomes 2^7 - 1, zeros lose their sign.
__device__ __forceinline__ uint32_t ordinary_codes(const float *x, float scale) {
    constexpr uint32_t TOP = 0x80808080u, LOW = 0x7f7f7f7fu;
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m |= (uint32_t)fmaf(fabsf(x[e]), scale, 0.5f - 0x1p-25f) << (8 * e);
    const uint32_t signs = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x0c0c0703u) | __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07030c0cu);
    m -= (m & TOP) >> 7;
    return (signs & (m + LOW) & TOP) | m;
}
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], uint32_t shared, bool ordinary) {
    if (ordinary) {
        const float scale = shared < 32u ? 0.f : __uint_as_float((260u - shared) << 23);
        return make_uint2(ordinary_codes(x, scale), ordinary_codes(x + 4, scale));
    }
    uint32_t words[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) words[i >> 2] |= to_code<7>(__float_as_uint(x[i]), shared) << (8 * (i & 3));
    return make_uint2(words[0], words[1]);
}

// An item is up to `each` heads of a few tokens.  LANES lanes share a token; each has two chunks of 8 elements of a head, chosen such that partners
// of the rotation are in one lane: chunks k and k + R/16, or neighbours (heads of 96 elements: six of eight lanes).  Angles are computed once for all heads of the item.  Registers decide: with all
// heads of a token in four lanes, 256 of them, the 8183 tokens took 136 us; now 82 to 128, four or five wavefronts per SIMD (64 elements into block floats
// without norms: 36 bytes of scratch memory as well).  AHEAD heads are on their
// way: two 58.7 us (with the read-back of the caches), three 57.7, four 59.4.
template <int SLABS, bool NORM, bool INTERLEAVED, bool PACKED>
__global__ __launch_bounds__(256) void paged_rotate_kernel(const RotateDev p) {
    constexpr uint32_t D = SLABS * 32, PAIRS = SLABS * 2, LANES = PAIRS <= 4 ? 4 : PAIRS <= 8 ? 8 : 16, ROWS = 64 / LANES, AHEAD = 3;
    __shared__ uint32_t tops[4][ROWS * 4 * SLABS];             // largest exponent of every chunk
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = p.tiled ? lane >> 1 & (ROWS - 1) : lane / LANES, q = p.tiled ? lane / (2 * ROWS) * 2 + (lane & 1) : lane % LANES;
    const uint32_t per_band = p.blocks[0] + p.blocks[1] + p.blocks[2];
    const bool mine = LANES == PAIRS || q < PAIRS;

    for (uint64_t item = (uint64_t)blockIdx.x * 4 + wave; item < p.items; item += (uint64_t)gridDim.x * 4) {
        const uint32_t band = (uint32_t)(item / per_band);
        uint32_t block = (uint32_t)(item - (uint64_t)band * per_band), kind = QUERIES;
        while (block >= p.blocks[kind]) block -= p.blocks[kind++];
        const uint32_t head0 = block * p.each, head1 = min(head0 + p.each, p.heads[kind]);
        const uint32_t t0 = band * ROWS, t = t0 + r;
        const uint32_t turning16 = kind == VALUES ? 0 : p.turning / 16;
        const bool turns = q < turning16, apart = turns && !INTERLEAVED;
        const uint32_t at[2] = {apart ? q : 2 * q, apart ? q + turning16 : 2 * q + 1};

        // what this lane reads, head by head
        const uint32_t head_step = p.tiled ? SLABS * 2048 : D * 2;
        const bool exists = t < p.tokens && mine;
        const uint8_t *from[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) from[h] = p.rows + row_bytes_at(t, p.width, p.column[kind] + head0 * D + at[h] * 8, p.tiled);
        u32x4 raw[AHEAD][2];
        auto load = [&](u32x4 (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v[h] = exists ? *reinterpret_cast<const u32x4 *>(from[h]) : u32x4{0, 0, 0, 0};
                from[h] += head_step;
            }
        };
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            if (head0 + i < head1) load(raw[i]);
        const float *const norm = NORM && kind != VALUES ? p.norm[kind] : nullptr;
        float weight[2][8], cosine[8], sine[8];
        if (NORM && norm && mine) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 8; ++i) weight[h][i] = norm[at[h] * 8 + i];
        }
        if (turns) {
#pragma unroll
            for (int i = 0; i < 8; ++i) cosine[i] = p.frequencies[q * 8 + i];
        }
        uint32_t position = 0;
        const bool owned = position_of<ROWS>(p, t0, r, position);
        // where this lane's chunks go
        bool stored = t < p.out_rows && mine;
        uint8_t *to[2], *exponent[2];
        uint64_t to_step = head_step;
        if (kind == QUERIES) {
#pragma unroll
            for (int h = 0; h < 2; ++h) to[h] = p.out + row_bytes_at(t, p.heads[QUERIES] * D, head0 * D + at[h] * 8, p.tiled);
        } else {
            const int32_t slot = owned ? p.slots[t] : -1;
            const uint32_t page = (uint32_t)max(slot, 0) / p.page_size, within = (uint32_t)max(slot, 0) - page * p.page_size;
            stored = slot >= 0 && page < p.pages && mine;
            const uint32_t tile_bytes = PACKED ? 1088 : 2048;
            to_step = (uint64_t)(p.page_size / 32) * SLABS * tile_bytes;
            uint8_t *const token = p.cache[kind - KEYS] + ((uint64_t)page * p.heads[kind] + head0) * to_step + (uint64_t)(within / 32) * SLABS * tile_bytes;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t c = at[h], face = (within >> 4 & 1) * 2 + (c >> 1 & 1), row = face * 16 + (within & 15);
                uint8_t *const tile = token + c / 4 * tile_bytes;
                to[h] = tile + (PACKED ? 64 + row * 16 + (c & 1) * 8 : row * 32 + (c & 1) * 16);
                exponent[h] = tile + row;
            }
        }
        if (turns) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                double turn = (double)position * ((double)cosine[i] * 0.15915494309189533577);
                turn -= rint(turn);
                cosine[i] = __builtin_amdgcn_cosf((float)turn) * p.magnitude;
                sine[i] = __builtin_amdgcn_sinf((float)turn) * p.magnitude;
                __builtin_amdgcn_sched_barrier(0);             // one after the other: eight at once are 40 registers more
            }
        }

        auto work = [&](const u32x4 (&v)[2]) __attribute__((always_inline)) {
            if (kind == VALUES && !PACKED) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (stored) *reinterpret_cast<u32x4 *>(to[h]) = v[h];
                return;
            }
            float x[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[h][2 * i] = __uint_as_float(v[h][i] << 16);
                    x[h][2 * i + 1] = __uint_as_float(v[h][i] & 0xffff0000u);
                }
            if (NORM && norm) {
                float sum = 0.f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = fmaf(x[h][i], x[h][i], sum);
                sum = sum_over_token<LANES>(sum, p.tiled);
                const float by = rsqrtf(sum * (1.f / D) + p.epsilon);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[h][i] *= by * weight[h][i];
            }
            if (turns) {
                auto turn = [&](float &a, float &b, int i) __attribute__((always_inline)) {
                    const float c = cosine[i], d = sine[i], old = a;
                    a = fmaf(a, c, -(b * d));
                    b = fmaf(b, c, old * d);
                };
                if (INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) turn(x[i >> 2][(i & 3) * 2], x[i >> 2][(i & 3) * 2 + 1], i);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) turn(x[0][i], x[1][i], i);
                }
            }
            if (kind == QUERIES || !PACKED) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4 rounded = {f32x2_to_bf16x2_rne(x[h][0], x[h][1]), f32x2_to_bf16x2_rne(x[h][2], x[h][3]), f32x2_to_bf16x2_rne(x[h][4], x[h][5]), f32x2_to_bf16x2_rne(x[h][6], x[h][7])};
                    if (stored) *reinterpret_cast<u32x4 *>(to[h]) = owned ? rounded : u32x4{0, 0, 0, 0};
                }
                return;
            }
            // block floats: two neighbouring chunks share an exponent, and lie in one lane or in two
            uint32_t *const top = tops[wave] + r * (4 * SLABS);
            uint32_t shared[2];
            bool odd = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                shared[h] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) shared[h] = max(shared[h], __float_as_uint(x[h][i]) & 0x7fffffffu);
                if (mine) top[at[h]] = shared[h];
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t largest = mine ? max(shared[h], top[at[h] ^ 1]) : 0;
                shared[h] = largest >> 23;
                odd |= (shared[h] < 32u && largest != 0) || shared[h] == 255u;
            }
            const bool ordinary = __ballot(odd) == 0;          // asked once for the wavefront
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint2 codes = codes_of(x[h], shared[h], ordinary);
                if (stored) {
                    *reinterpret_cast<uint2 *>(to[h]) = codes;
                    if (!(at[h] & 1)) *exponent[h] = (uint8_t)shared[h];
                }
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        };
        for (uint32_t head = head0; head < head1; ++head) {
            const u32x4 v[2] = {raw[0][0], raw[0][1]};
#pragma unroll
            for (uint32_t i = 0; i + 1 < AHEAD; ++i) { raw[i][0] = raw[i + 1][0]; raw[i][1] = raw[i + 1][1]; }
            if (head + AHEAD < head1) load(raw[AHEAD - 1]);
            work(v);
#pragma unroll
            for (int h = 0; h < 2; ++h) { to[h] += to_step; exponent[h] += to_step; }
        }
    }
}

template <int SLABS, bool NORM, bool INTERLEAVED> static void launch(const RotateDev &p, bool packed, dim3 grid, hipStream_t st) {
    if (packed) hipLaunchKernelGGL((paged_rotate_kernel<SLABS, NORM, INTERLEAVED, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_rotate_kernel<SLABS, NORM, INTERLEAVED, false>), grid, dim3(256), 0, st, p);
}
template <int SLABS> static void launch(const RotateDev &p, const PagedRotationArgs &x, dim3 grid, hipStream_t st) {
    const bool norm = x.query_norm || x.key_norm, packed = x.key_cache && x.cache.dtype == TTMI_BFLOAT8_B;
    if (norm && x.interleaved) launch<SLABS, true, true>(p, packed, grid, st);
    else if (norm) launch<SLABS, true, false>(p, packed, grid, st);
    else if (x.interleaved) launch<SLABS, false, true>(p, packed, grid, st);
    else launch<SLABS, false, false>(p, packed, grid, st);
}

int paged_rotate(const PagedRotationArgs &x, hipStream_t st) {
    RotateDev p{};
    p.rows = (const uint8_t *)x.rows.data; p.out = (uint8_t *)x.out;
    p.cache[0] = (uint8_t *)x.key_cache; p.cache[1] = (uint8_t *)x.value_cache;
    p.cached = x.step.cached; p.starts = x.step.row_starts; p.slots = x.slots;
    p.frequencies = x.frequencies; p.norm[0] = x.query_norm; p.norm[1] = x.key_norm;
    p.tokens = x.rows.tokens; p.width = x.rows.width; p.requests = x.step.requests;
    p.tiled = x.rows.layout == TTMI_TILE;
    p.out_rows = p.tiled ? (p.tokens + 31) / 32 * 32 : p.tokens;
    if (!p.out_rows) return TTMI_OK;
    p.column[0] = x.query_column; p.column[1] = x.key_column; p.column[2] = x.value_column;
    p.heads[0] = x.heads;
    if (x.key_cache) p.heads[1] = p.heads[2] = x.cache.kv_heads;
    p.pages = x.cache.pages; p.page_size = std::max(x.cache.page_size, 32u);
    p.turning = x.rotary_dim;
    p.epsilon = x.epsilon; p.magnitude = x.magnitude;
    const uint32_t rows = x.head_dim == 64 ? 16 : x.head_dim == 256 ? 4 : 8;       // tokens of an item
    const uint64_t bands = ((uint64_t)p.out_rows + rows - 1) / rows, heads = (uint64_t)p.heads[0] + p.heads[1] + p.heads[2];
    // Heads of an item: many share the angles, few leave enough items to fill the chip.  8183 tokens (with the read-back) and 8206: one 82 and 44 us,
    // two 66 and 35, three 62 and 33, four 59 and 33, eight 60 and 35, sixteen 59 and 38
    p.each = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(bands * heads / 8192, 1), 4);
    for (int k = 0; k < 3; ++k) p.blocks[k] = (p.heads[k] + p.each - 1) / p.each;
    p.items = bands * (p.blocks[0] + p.blocks[1] + p.blocks[2]);
    const dim3 grid((uint32_t)std::min<uint64_t>((p.items + 3) / 4, 1u << 20));
    switch (x.head_dim) {
        case 64: launch<2>(p, x, grid, st); break;
        case 96: launch<3>(p, x, grid, st); break;
        case 128: launch<4>(p, x, grid, st); break;
        default: launch<8>(p, x, grid, st); break;
    }
    return check_launch("paged_rotate_kernel");
}

}  // namespace ttmi
