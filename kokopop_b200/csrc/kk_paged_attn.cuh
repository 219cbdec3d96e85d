// What the two kernels of the paged attention share: the rounding of a pair
// to the cache's type and the tile of a block.
#pragma once

#include "kk_common.cuh"
#include "kk_kernels.h"

namespace kk {

__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The tile `w` of a launch, `unit` rows (query, head of the group) each.
// Request r's tiles begin at floor(cu[r] * group / unit) + r: consecutive
// requests are at least as far apart as request r has tiles, so the request
// is found by bisection of cu_new alone, and at most
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
    int x = 0, y = a.n_seqs - 1;
    while (x < y) {
        const int mid = (x + y + 1) >> 1;
        if (first_tile(a, group, unit, mid) <= w)
            x = mid;
        else
            y = mid - 1;
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

}  // namespace kk
