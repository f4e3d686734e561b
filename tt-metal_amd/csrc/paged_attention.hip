// Attention of new tokens over a paged key/value cache (paged_cache.hip says how one is laid out).
//
// Request r has cached_r tokens from before and n_r = row_starts[r + 1] - row_starts[r] new ones, all of them in the cache.  Row
// row_starts[r] + i of the activations is token p = cached_r + i.  For each of its heads, with the key head that its group shares,
//   out = sum_j softmax_j(scale q . k_j) v_j    over the tokens p - window < j <= p that have a page
// and zeros where nothing is left.  Slots behind a request's last token hold whatever was there before, infinities and NaN
// among it, and never count.
//
// One wavefront per row and query head: 64 keys at a time, one to a lane, the running maximum and sum of the softmax in fp32, then
// each lane adds up its elements of the 64 values.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bfp_dequant.h"
#include "paged_cache.h"
#include "ttmi_internal.h"

namespace ttmi {

struct AttentionDev {
    const uint8_t *rows;
    const uint8_t *keys, *values;
    const int32_t *table, *cached, *starts;
    uint8_t *out;
    uint32_t tokens, width, query_column, requests, max_pages;
    uint32_t pages, kv_heads, page_size, head_dim, heads, group, window;
    float scale;                           // times log2(e)
    int tiled, packed;
};

__device__ __forceinline__ float bf16_at(const uint8_t *p) { return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16); }

// element d of a token that lies in row `at` of a head's page
__device__ __forceinline__ float cached_element(const uint8_t *head_page, uint32_t at, uint32_t d, uint32_t head_dim, int packed) {
    const uint64_t tile = (uint64_t)(at / 32) * (head_dim / 32) + d / 32;
    const uint32_t face = (at >> 4 & 1) * 2 + (d >> 4 & 1), row = at & 15, e = d & 15;
    if (!packed) return bf16_at(head_page + tile * 2048 + face * 512 + row * 32 + e * 2);
    const uint8_t *t = head_page + tile * 1088;
    const uint32_t code = t[64 + face * 256 + row * 16 + e];
    const float v = (float)(code & 127u) * row_scale(t[face * 16 + row]) * Wfmt<7>::unscale;
    return code & 128u ? -v : v;
}

__global__ __launch_bounds__(64) void paged_attention_rows_kernel(const AttentionDev p) {
    const uint32_t lane = threadIdx.x;
    const uint32_t t = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
    const uint64_t out_width = p.heads * p.head_dim;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};                       // elements lane, lane + 64, ... of the head
    float sum = 0.f, top = -INFINITY;
    uint32_t low = 0, high = p.requests;
    if (t < p.tokens && t < (uint32_t)max(p.starts[p.requests], 0)) {
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if ((uint32_t)max(p.starts[mid], 0) <= t) low = mid; else high = mid;
        }
        const uint32_t r = low;
        const uint64_t position = (uint64_t)max(p.cached[r], 0) + (t - (uint32_t)max(p.starts[r], 0));
        const uint64_t first = p.window && position + 1 > p.window ? position + 1 - p.window : 0;
        const uint64_t end = min(position + 1, (uint64_t)p.max_pages * p.page_size);
        const uint64_t page_bytes = (uint64_t)(p.page_size / 32) * (p.head_dim / 32) * (p.packed ? 1088 : 2048);
        const uint32_t kv = h / p.group;
        for (uint64_t j0 = first / 64 * 64; j0 < end; j0 += 64) {
            const uint64_t j = j0 + lane;
            int32_t page = -1;
            if (j >= first && j < end) page = p.table[(uint64_t)r * p.max_pages + j / p.page_size];
            const bool there = (uint32_t)page < p.pages;
            const uint32_t at = (uint32_t)(j % p.page_size);
            const uint64_t head_page = ((uint64_t)page * p.kv_heads + kv) * page_bytes;
            float score = -INFINITY;
            if (there) {
                float dot = 0.f;
                for (uint32_t d = 0; d < p.head_dim; ++d)
                    dot += bf16_at(p.rows + row_bytes_at(t, p.width, p.query_column + h * p.head_dim + (d & ~7u), p.tiled) + (d & 7) * 2) *
                           cached_element(p.keys + head_page, at, d, p.head_dim, p.packed);
                score = dot * p.scale;
            }
            float most = score;
            for (int s = 32; s; s >>= 1) most = fmaxf(most, __shfl_xor(most, s));
            most = fmaxf(most, top);
            const float from = most == -INFINITY ? 0.f : most, shrink = __builtin_amdgcn_exp2f(top - from);
            const float weight = there ? __builtin_amdgcn_exp2f(score - from) : 0.f;
            float all = weight;
            for (int s = 32; s; s >>= 1) all += __shfl_xor(all, s);
            sum = sum * shrink + all;
            top = most;
            for (int i = 0; i < 4; ++i) acc[i] *= shrink;
            for (int l = 0; l < 64; ++l) {
                const float w = __shfl(weight, l);
                if (!__shfl((int)there, l)) continue;          // the whole wavefront
                const uint32_t at_l = __shfl(at, l);
                const uint64_t page_l = ((uint64_t)__shfl(page, l) * p.kv_heads + kv) * page_bytes;
                for (uint32_t i = 0, d = lane; d < p.head_dim; ++i, d += 64) acc[i] += w * cached_element(p.values + page_l, at_l, d, p.head_dim, p.packed);
            }
        }
    }
    const float share = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    for (uint32_t i = 0, d = lane; d < p.head_dim; ++i, d += 64) {
        const uint32_t column = h * p.head_dim + d;
        *reinterpret_cast<uint16_t *>(p.out + row_bytes_at(t, (uint32_t)out_width, column & ~7u, p.tiled) + (column & 7) * 2) = (uint16_t)f32x2_to_bf16x2_rne(sum == 0.f ? 0.f : acc[i] * share, 0.f);
    }
}

size_t paged_attention_workspace_bytes(uint32_t, uint32_t, uint32_t, const PagedCache &) { return 0; }

int paged_attention(const PagedAttentionArgs &x, hipStream_t st) {
    const uint32_t rows = x.rows.layout == TTMI_TILE ? (x.rows.tokens + 31) / 32 * 32 : x.rows.tokens;
    if (!rows) return TTMI_OK;
    AttentionDev p{};
    p.rows = (const uint8_t *)x.rows.data; p.keys = (const uint8_t *)x.key_cache; p.values = (const uint8_t *)x.value_cache;
    p.table = x.step.page_table; p.cached = x.step.cached; p.starts = x.step.row_starts; p.out = (uint8_t *)x.out;
    p.tokens = x.rows.tokens; p.width = x.rows.width; p.query_column = x.query_column; p.requests = x.step.requests; p.max_pages = x.step.max_pages;
    p.pages = x.cache.pages; p.kv_heads = x.cache.kv_heads; p.page_size = x.cache.page_size; p.head_dim = x.cache.head_dim;
    p.heads = x.heads; p.group = x.heads / x.cache.kv_heads; p.window = x.window;
    p.scale = x.scale * 1.4426950408889634f;
    p.tiled = x.rows.layout == TTMI_TILE; p.packed = x.cache.dtype == TTMI_BFLOAT8_B;
    hipLaunchKernelGGL(paged_attention_rows_kernel, dim3(rows * x.heads), dim3(64), 0, st, p);
    return check_launch("paged_attention_rows_kernel");
}

}  // namespace ttmi
