// Queries and keys of a step by their positions: the norm of every head and its rotation, the keys and values straight into their pages.
//
// Row row_starts[r] + i of the activations is token p = cached[r] + i of request r.  For each head x of D elements, where a norm is given,
//   y_d = x_d w_d / sqrt(mean(x^2) + epsilon)
// and, of its first R elements, the pairs (a, b) = (y_i, y_(i + R/2)), or neighbours (y_2i, y_(2i+1)), i < R/2,
//   (a, b) -> m (a cos(p f_i) - b sin(p f_i), b cos(p f_i) + a sin(p f_i))
// in fp32 and rounded once: to bf16, or, for keys of a BFLOAT8_B cache, from fp32 to its codes.
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
    int tiled, interleaved, packed;
};

// Position of row t0 + r, r = 0 .. 15, false where it is no request's.  A row belongs to the request before the first start behind it, and
// the request's rows begin at the largest start up to its own: row starts that do not ascend are read through their running maximum.
__device__ __forceinline__ bool position_of(const RotateDev &p, uint32_t t0, uint32_t r, uint32_t &position) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t owner = 0xffffffffu, from = 0, top = 0, open = 0xffffu;      // rows whose request is still looked for
    for (uint32_t base = 0; base <= p.requests && open; base += 64) {
        const uint32_t v = base + lane <= p.requests ? min((uint32_t)max(p.starts[base + lane], 0), p.tokens) : 0xffffffffu;
        const uint32_t to = max(running_max(v), top);
        if (__ballot(to > t0))
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
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

// An item is up to `each` heads of 16 tokens.  Four lanes share a token; a lane has SLOTS pairs of chunks of 8 elements, chosen such that partners of
// the rotation are in one lane: chunks k and k + R/16, or neighbours.
template <int SLABS, bool NORM>
__global__ __launch_bounds__(256) void paged_rotate_kernel(const RotateDev p) {
    constexpr uint32_t D = SLABS * 32, PAIRS = SLABS * 2, SLOTS = (PAIRS + 3) / 4;
    __shared__ uint32_t tops[4][16 * 4 * SLABS];               // largest exponent of every chunk
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = p.tiled ? lane >> 1 & 15 : lane >> 2, q = p.tiled ? (lane >> 5) * 2 + (lane & 1) : lane & 3;
    const uint32_t per_band = p.blocks[0] + p.blocks[1] + p.blocks[2];

    for (uint64_t item = (uint64_t)blockIdx.x * 4 + wave; item < p.items; item += (uint64_t)gridDim.x * 4) {
        const uint32_t band = (uint32_t)(item / per_band);
        uint32_t block = (uint32_t)(item - (uint64_t)band * per_band), kind = QUERIES;
        while (block >= p.blocks[kind]) block -= p.blocks[kind++];
        const uint32_t head0 = block * p.each, head1 = min(head0 + p.each, p.heads[kind]);
        const uint32_t t0 = band * 16, t = t0 + r, column = p.column[kind];
        const uint32_t turning16 = kind == VALUES ? 0 : p.turning / 16;

        uint32_t at[SLOTS][2];                                 // chunks of a head; this lane has none where the first is past the head
#pragma unroll
        for (uint32_t s = 0; s < SLOTS; ++s) {
            const uint32_t k = s * 4 + q;
            const bool apart = k < turning16 && !p.interleaved;
            at[s][0] = apart ? k : 2 * k;
            at[s][1] = apart ? k + turning16 : 2 * k + 1;
        }
        u32x4 raw[SLOTS][2];
        auto load = [&](uint32_t head) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    raw[s][h] = t < p.tokens && s * 4 + q < PAIRS ? *reinterpret_cast<const u32x4 *>(p.rows + row_bytes_at(t, p.width, column + head * D + at[s][h] * 8, p.tiled)) : u32x4{0, 0, 0, 0};
        };
        load(head0);
        uint32_t position = 0;
        const bool owned = position_of(p, t0, r, position);

        // where this lane's token goes
        uint32_t page = 0, within = 0;
        bool stored = t < p.out_rows;
        if (kind != QUERIES) {
            const int32_t slot = owned ? p.slots[t] : -1;
            page = (uint32_t)max(slot, 0) / p.page_size;
            within = (uint32_t)max(slot, 0) - page * p.page_size;
            stored = slot >= 0 && page < p.pages;
        }
        float cosine[SLOTS][8], sine[SLOTS][8], weight[SLOTS][2][8];
#pragma unroll
        for (uint32_t s = 0; s < SLOTS; ++s) {
            const uint32_t k = s * 4 + q;
            if (k < turning16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    double turns = (double)position * ((double)p.frequencies[k * 8 + i] * 0.15915494309189533577);
                    turns -= rint(turns);
                    cosine[s][i] = __builtin_amdgcn_cosf((float)turns) * p.magnitude;
                    sine[s][i] = __builtin_amdgcn_sinf((float)turns) * p.magnitude;
                }
            }
            if (NORM && kind != VALUES && p.norm[kind] && k < PAIRS) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) weight[s][h][i] = p.norm[kind][at[s][h] * 8 + i];
            }
        }

        for (uint32_t head = head0; head < head1; ++head) {
            float x[SLOTS][2][8];
            u32x4 kept[SLOTS][2];
#pragma unroll
            for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    kept[s][h] = raw[s][h];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[s][h][2 * i] = __uint_as_float(raw[s][h][i] << 16);
                        x[s][h][2 * i + 1] = __uint_as_float(raw[s][h][i] & 0xffff0000u);
                    }
                }
            if (head + 1 < head1) load(head + 1);
            if (NORM && kind != VALUES && p.norm[kind]) {
                float sum = 0.f;
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum = fmaf(x[s][h][i], x[s][h][i], sum);
                sum += __shfl_xor(sum, 1);
                sum += __shfl_xor(sum, p.tiled ? 32 : 2);
                const float by = rsqrtf(sum * (1.f / D) + p.epsilon);
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[s][h][i] *= by * weight[s][h][i];
            }
#pragma unroll
            for (uint32_t s = 0; s < SLOTS; ++s) {
                if (s * 4 + q >= turning16) continue;
                auto turn = [&](float &a, float &b, int i) __attribute__((always_inline)) {
                    const float c = cosine[s][i], d = sine[s][i], old = a;
                    a = fmaf(a, c, -(b * d));
                    b = fmaf(b, c, old * d);
                };
                if (p.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) turn(x[s][i >> 2][(i & 3) * 2], x[s][i >> 2][(i & 3) * 2 + 1], i);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) turn(x[s][0][i], x[s][1][i], i);
                }
            }
            auto rounded = [&](const float (&v)[8]) __attribute__((always_inline)) {
                return u32x4{f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]), f32x2_to_bf16x2_rne(v[4], v[5]), f32x2_to_bf16x2_rne(v[6], v[7])};
            };
            if (kind == QUERIES) {
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (stored && s * 4 + q < PAIRS)
                            *reinterpret_cast<u32x4 *>(p.out + row_bytes_at(t, p.heads[QUERIES] * D, head * D + at[s][h] * 8, p.tiled)) = owned ? rounded(x[s][h]) : u32x4{0, 0, 0, 0};
                continue;
            }
            uint8_t *const cache = p.cache[kind - KEYS];
            const uint64_t tile0 = (((uint64_t)page * p.heads[kind] + head) * (p.page_size / 32) + within / 32) * SLABS;
            if (!p.packed) {
#pragma unroll
                for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t c = at[s][h];
                        if (stored && s * 4 + q < PAIRS)
                            *reinterpret_cast<u32x4 *>(cache + (tile0 + c / 4) * 2048 + ((within >> 4 & 1) * 2 + (c >> 1 & 1)) * 512 + (within & 15) * 32 + (c & 1) * 16) = kind == VALUES ? kept[s][h] : rounded(x[s][h]);
                    }
                continue;
            }
            // block floats: two neighbouring chunks share an exponent, and lie in one lane or in two
            uint32_t *const top = tops[wave] + r * (4 * SLABS);
            uint32_t own[SLOTS][2];
#pragma unroll
            for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    own[s][h] = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) own[s][h] = max(own[s][h], __float_as_uint(x[s][h][i]) >> 23 & 0xffu);
                    if (s * 4 + q < PAIRS) top[at[s][h]] = own[s][h];
                }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (uint32_t s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t c = at[s][h];
                    if (!stored || s * 4 + q >= PAIRS) continue;
                    const uint32_t shared = max(own[s][h], top[c ^ 1]), face = (within >> 4 & 1) * 2 + (c >> 1 & 1);
                    uint32_t words[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 8; ++i) words[i >> 2] |= to_code<7>(__float_as_uint(x[s][h][i]), shared) << (8 * (i & 3));
                    uint8_t *const to = cache + (tile0 + c / 4) * 1088;
                    *reinterpret_cast<uint2 *>(to + 64 + face * 256 + (within & 15) * 16 + (c & 1) * 8) = make_uint2(words[0], words[1]);
                    if (!(c & 1)) to[face * 16 + (within & 15)] = (uint8_t)shared;
                }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
    }
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
    p.turning = x.rotary_dim; p.interleaved = x.interleaved;
    p.epsilon = x.epsilon; p.magnitude = x.magnitude;
    p.packed = x.cache.dtype == TTMI_BFLOAT8_B;
    const uint64_t bands = ((uint64_t)p.out_rows + 15) / 16, heads = (uint64_t)p.heads[0] + p.heads[1] + p.heads[2];
    p.each = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(bands * heads / 8192, 1), 8);
    for (int k = 0; k < 3; ++k) p.blocks[k] = (p.heads[k] + p.each - 1) / p.each;
    p.items = bands * (p.blocks[0] + p.blocks[1] + p.blocks[2]);
    const dim3 grid((uint32_t)std::min<uint64_t>((p.items + 3) / 4, 1u << 20));
    const bool norm = x.query_norm || x.key_norm;
    auto launch = [&](auto plain, auto normed) { hipLaunchKernelGGL(norm ? normed : plain, grid, dim3(256), 0, st, p); };
    switch (x.head_dim) {
        case 64: launch(paged_rotate_kernel<2, false>, paged_rotate_kernel<2, true>); break;
        case 96: launch(paged_rotate_kernel<3, false>, paged_rotate_kernel<3, true>); break;
        case 128: launch(paged_rotate_kernel<4, false>, paged_rotate_kernel<4, true>); break;
        default: launch(paged_rotate_kernel<8, false>, paged_rotate_kernel<8, true>); break;
    }
    return check_launch("paged_rotate_kernel");
}

}  // namespace ttmi
