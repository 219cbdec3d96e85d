// What the two kernels of the paged attention share: arithmetic, the tile of
// a block, and the tensor maps of the cache.
#pragma once

#include "kk_common.cuh"
#include "kk_kernels.h"

#include <cuda.h>

namespace kk {

__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The weights of the product with V are 2^(s - m + kLift): half has 2^-14 as
// its smallest normal number, and weights that are small fractions of the
// largest one count where the keys are many. m is at most 8 behind the
// maximum, so half's reach 2^15 (its largest is 2^16 - 32), and they are
// normal from 2^-21 of the largest on. The factor is in the sums too and
// leaves with the division; bfloat16 has the range of 32 bits and needs none.
template <typename T>
constexpr float kLift = 0.f;
template <>
constexpr float kLift<__half> = 7.f;

// 2^x, results below 2^-126 as 0 (weights are at most 2^15 and rounded to 16
// bits, or relative to a largest one)
__device__ __forceinline__ float pow2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 1 / l; 0 for a row that saw no key, and a NaN sum stays one
__device__ __forceinline__ float paged_inverse(float l) { return l > 0.f ? 1.f / l : l == 0.f ? 0.f : l; }

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// Keys that a request's table can hold; positions and steps past them fit 32
// bits.
__device__ __forceinline__ int64_t paged_capacity(const PagedAttnArgs &a) {
    return min((int64_t)a.max_pages * a.cache.page_size, (int64_t)INT32_MAX - 1023);
}

// The tile `w` of a launch, `unit` rows (query, head of the group) each.
// Request r's tiles begin at floor(cu[r] * group / unit) + r: consecutive
// requests are at least as far apart as request r has tiles, so the request
// is found from cu_new alone, and at most
// floor(n_tokens * group / unit) + n_seqs indices are in use.
struct RowTile {
    int r;         // request, -1: no such tile
    int row0;      // first row (query * group + head of the group) in the request
    int rows;      // rows of the request
    int64_t tok0;  // its first token's row in q and out
    int n;         // its new tokens (those that n_tokens covers)
    int base;      // position of its first new token
};

__device__ __forceinline__ int64_t first_tile(const PagedAttnArgs &a, int group, int unit, int r) {
    return min((int64_t)max(a.cu_new[r], 0), a.n_tokens) * group / unit + r;
}

__device__ __forceinline__ RowTile find_tile(const PagedAttnArgs &a, int group, int unit, int64_t w) {
    RowTile t;
    // the last request that begins at or before tile w, 32 candidates a round
    // (every warp of the block by itself)
    const int lane = threadIdx.x & 31;
    int x = 0, n = a.n_seqs;  // among [x, x + n)
    while (n > 1) {
        const int step = (n + 31) / 32, i = lane * step;
        const uint32_t before = __ballot_sync(0xffffffffu, i < n && first_tile(a, group, unit, x + i) <= w);
        const int k = before ? 31 - __clz(before) : 0;
        x += k * step;
        n = min(step, n - k * step);
    }
    t.r = x;
    t.tok0 = min((int64_t)max(a.cu_new[x], 0), a.n_tokens);
    const int64_t tok1 = min((int64_t)max(a.cu_new[x + 1], 0), a.n_tokens);
    t.n = tok1 > t.tok0 ? (int)(tok1 - t.tok0) : 0;
    t.base = a.seq_len[x] - max(a.cu_new[x + 1] - a.cu_new[x], 0);
    const int64_t row0 = (w - first_tile(a, group, unit, x)) * unit, rows = (int64_t)t.n * group;
    if (row0 < 0 || row0 >= rows) t.r = -1;
    t.row0 = (int)row0;
    t.rows = rows > INT32_MAX ? INT32_MAX : (int)rows;
    return t;
}

// Maps of k and v as (dim, token, head, page), boxes of 64 dims and
// min(page_size, keys) tokens, 128-byte swizzle; what lies outside reads as 0.
cudaError_t paged_cache_maps(const PagedCacheView &c, int keys, CUtensorMap *k, CUtensorMap *v);
// rows of q as (dim, head, token), boxes of 64 x heads x tokens
cudaError_t paged_q_map(const PagedAttnArgs &a, int heads, int tokens, CUtensorMap *m);
// tensor-map strides are below 2^40 bytes and not 0
bool paged_strides_mappable(const PagedCacheView &c);

}  // namespace kk
