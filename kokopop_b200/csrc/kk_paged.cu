// The paged key / value cache (sm_100a): pages and slots of the new tokens
// from the request lengths, and the new tokens' rows into their slots.
#include "../../include/kokopop_b200.h"
#include "kk_common.cuh"
#include "kk_kernels.h"

namespace kk {

// ---------------------------------------------------------------------------
// Page tables. Request r has c = ctx_len[r] tokens in the cache and takes
// m = new_len[r] more (negative lengths count as 0). It holds
// old = ceil(c / P) pages and needs
//   need = max(0, min(ceil((c + m) / P), max_pages) - old)
// further ones: the entries table[r][old + j], j < need, are
// free_pages[head + first_r + j], first_r the sum of `need` over the requests
// before r, or -1 from `end` on. A new token at position p = c + t lies in
// slot table[r][p / P] P + p % P, or -1 without a page.
//
// All of it is integer work on 12 bytes written per new token, so what counts
// is that it is one launch without a workspace: every block scans the lengths
// itself (kPtChunk requests at a time, so that any number of requests
// passes), then writes its share of the tokens, 32 of a warp, which find their
// requests by searching the scanned offsets in shared memory. The token at
// the start of a new page writes the table entry, so no block reads what
// another writes. Measured on B200: 64 requests of one token 10 us a call, the
// host's (5.6 on the device); 2048 requests with 1.05 M tokens 14.5 us (13 MB, 2
// us of traffic: the scan in every block, the searches and each token's loads,
// one after another, bound it).
// ---------------------------------------------------------------------------
constexpr int kPtThreads = 1024;
constexpr int kPtPer = 4;
constexpr int kPtChunk = kPtThreads * kPtPer;

__device__ __forceinline__ int clamp_i32(int64_t v) { return v > INT32_MAX ? INT32_MAX : (int)v; }

// pages of n tokens
__device__ __forceinline__ int64_t pages_of(int64_t n, int64_t P, int size_bits) {
    return size_bits >= 0 ? (n + P - 1) >> size_bits : (n + P - 1) / P;
}

// The last of the n ascending offsets cu that is at most t (cu[0] is), for a
// whole warp, 32 candidates a round.
__device__ __forceinline__ int last_at_or_before(const int *cu, int n, int64_t t, int lane) {
    int x = 0;
    while (n > 1) {
        const int step = (n + 31) / 32, i = lane * step;
        const uint32_t before = __ballot_sync(0xffffffffu, i < n && cu[x + i] <= t);
        const int k = before ? 31 - __clz(before) : 0;
        x += k * step;
        n = min(step, n - k * step);
    }
    return x;
}

__global__ void __launch_bounds__(kPtThreads) k_page_tables(PageTablesArgs a) {
    __shared__ int cu_s[kPtChunk + 1];     // first token of each request of the chunk
    __shared__ int first_s[kPtChunk];      // first new page of each request
    __shared__ int64_t wsum[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t P = a.page_size;
    const int size_bits = (a.page_size & (a.page_size - 1)) == 0 ? 31 - __clz(a.page_size) : -1;
    const int64_t t_per = (a.n_tokens + gridDim.x - 1) / gridDim.x;
    const int64_t t0 = blockIdx.x * t_per, t1 = t0 + t_per < a.n_tokens ? t0 + t_per : a.n_tokens;
    const bool writer = blockIdx.x == gridDim.x - 1;
    const int64_t head = a.free_range[0], end = min((int64_t)a.free_range[1], a.free_cap);
    int64_t base_t = 0, base_p = 0;  // tokens and pages of the chunks before
    for (int r0 = 0; r0 < a.n_seqs; r0 += kPtChunk) {
        int64_t m[kPtPer], need[kPtPer], st = 0, sp = 0;
#pragma unroll
        for (int j = 0; j < kPtPer; ++j) {
            const int r = r0 + tid * kPtPer + j;
            m[j] = need[j] = 0;
            if (r < a.n_seqs) {
                const int64_t c = max(a.ctx_len[r], 0);
                m[j] = max(a.new_len[r], 0);
                const int64_t old = pages_of(c, P, size_bits);
                need[j] = max(min(pages_of(c + m[j], P, size_bits), (int64_t)a.max_pages) - old, (int64_t)0);
                if (writer) a.seq_len[r] = clamp_i32(c + m[j]);
            }
            st += m[j];
            sp += need[j];
        }
        // exclusive sums over the block
        int64_t it = st, ip = sp;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, it, o), y = __shfl_up_sync(0xffffffffu, ip, o);
            if (lane >= o) it += x, ip += y;
        }
        if (lane == 31) wsum[0][warp] = it, wsum[1][warp] = ip;
        __syncthreads();
        // every warp sums the 32 warps' totals
        int64_t wt = wsum[0][lane], wp = wsum[1][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, wt, o), y = __shfl_up_sync(0xffffffffu, wp, o);
            if (lane >= o) wt += x, wp += y;
        }
        const int64_t all_t = base_t + __shfl_sync(0xffffffffu, wt, 31),
                      all_p = base_p + __shfl_sync(0xffffffffu, wp, 31);
        const int64_t prev_t = __shfl_sync(0xffffffffu, wt, (warp + 31) & 31),
                      prev_p = __shfl_sync(0xffffffffu, wp, (warp + 31) & 31);
        int64_t tt = base_t + (warp > 0 ? prev_t : 0) + it - st, pp = base_p + (warp > 0 ? prev_p : 0) + ip - sp;
#pragma unroll
        for (int j = 0; j < kPtPer; ++j) {
            const int i = tid * kPtPer + j;
            cu_s[i] = clamp_i32(tt);
            first_s[i] = clamp_i32(pp);
            if (writer && r0 + i < a.n_seqs) a.cu_new[r0 + i] = clamp_i32(tt);
            tt += m[j];
            pp += need[j];
        }
        if (tid == 0) cu_s[kPtChunk] = clamp_i32(all_t);
        __syncthreads();
        const int n = min(kPtChunk, a.n_seqs - r0);
        // a warp takes a run of tokens, 32 at a time: their requests lie between
        // that of the first and that of the last, mostly the same one
        const int64_t lo = max(t0, base_t), hi_all = min(t1, all_t);
        const int64_t run = (max(hi_all - lo, (int64_t)0) + kPtThreads - 1) / kPtThreads * 32;
        const int64_t hi = min(lo + (warp + 1) * run, hi_all);
        int first = -1;
        for (int64_t tw = lo + warp * run; tw < hi; tw += 32) {
            const int64_t t = tw + lane, last = min(tw + 31, hi - 1);
            if (first < 0 || (first + 1 < n && cu_s[first + 1] <= tw)) first = last_at_or_before(cu_s, n, tw, lane);
            int x = first, y = first;
            if (first + 1 < n && cu_s[first + 1] <= last) y = last_at_or_before(cu_s, n, last, lane);
            if (t >= hi) continue;
            while (x < y) {
                const int mid = (x + y + 1) >> 1;
                if (cu_s[mid] <= t)
                    x = mid;
                else
                    y = mid - 1;
            }
            const int r = r0 + x;
            // positions are below 2^32: two lengths of 31 bits
            const uint32_t c = (uint32_t)max(a.ctx_len[r], 0), pos = c + (uint32_t)(t - cu_s[x]), size = a.page_size;
            const uint32_t col = size_bits >= 0 ? pos >> size_bits : pos / size, off = pos - col * size;
            const uint32_t whole = size_bits >= 0 ? c >> size_bits : c / size, old = whole + (whole * size != c);
            int page = -1;
            if (col < (uint32_t)a.max_pages) {
                int32_t *entry = a.table + (int64_t)r * a.max_pages + col;
                if (col < old) {
                    page = *entry;
                } else {
                    const int64_t i = head + first_s[x] + (col - old);
                    if (i >= 0 && i < end) page = a.free_pages[i];
                    if (off == 0) *entry = page;
                }
            }
            a.slots[t] = page >= 0 ? page * P + off : -1;
            if (a.positions) a.positions[t] = clamp_i32(pos);
        }
        base_t = all_t;
        base_p = all_p;
        __syncthreads();  // the offsets are read before the next chunk's are written
    }
    // rows past the last new token
    for (int64_t t = max(t0, base_t) + tid; t < t1; t += kPtThreads) {
        a.slots[t] = -1;
        if (a.positions) a.positions[t] = -1;
    }
    if (writer && tid == 0) {
        a.cu_new[a.n_seqs] = clamp_i32(base_t);
        const int64_t have = max(end - max(head, (int64_t)0), (int64_t)0), took = min(base_p, have);
        a.status[0] = clamp_i32(head + took);
        a.status[1] = a.free_range[1];
        a.status[2] = clamp_i32(base_p - took);
    }
}

cudaError_t page_tables(const PageTablesArgs &a, cudaStream_t st) {
    const int64_t want = (a.n_tokens + kPtThreads - 1) / kPtThreads;
    const int64_t grid = want < 1 ? 1 : want > 148 ? 148 : want;
    k_page_tables<<<(unsigned)grid, kPtThreads, 0, st>>>(a);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Append: row t of k and v (n_kv_heads x head_dim values, rows apart by their
// strides) to the cache row of slots[t]; a slot outside the cache is skipped.
// A copy: bytes bound it (16381 tokens of 12 heads of 64, F32 to F16, 151 MB
// in 27.4 us, 5.5 TB/s). A thread moves 8 values of K and the same 8 of V,
// 16-byte stores into the cache and 16- or 32-byte loads from the source.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const T *h = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&v)[8]) {
    const float4 x = *reinterpret_cast<const float4 *>(p), y = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
}

__device__ __forceinline__ void narrow(float x, __half &o) { o = __float2half_rn(x); }
__device__ __forceinline__ void narrow(float x, __nv_bfloat16 &o) { o = __float2bfloat16_rn(x); }

template <typename S, typename D>
__global__ void __launch_bounds__(256) k_cache_append(const S *__restrict__ k, const S *__restrict__ v,
                                                      int64_t k_stride, int64_t v_stride,
                                                      const int64_t *__restrict__ slots, int64_t n_tokens,
                                                      PagedCacheView c) {
    const int per_head = c.head_dim / 8, per_row = per_head * c.n_kv_heads;
    const int64_t n = n_tokens * per_row;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t t = i / per_row;
        const int j = (int)(i - t * per_row), head = j / per_head, d = (j - head * per_head) * 8;
        const int64_t slot = slots[t];
        if (slot < 0 || slot >= c.n_pages * c.page_size) continue;
        const int64_t page = slot / c.page_size;
        const int64_t dst = page * c.page_stride + (slot - page * c.page_size) * c.token_stride +
                            head * c.head_stride + d;
        float x[8], y[8];
        load8(k + t * k_stride + head * c.head_dim + d, x);
        load8(v + t * v_stride + head * c.head_dim + d, y);
        __align__(16) D a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) narrow(x[e], a[e]), narrow(y[e], b[e]);
        *reinterpret_cast<uint4 *>((D *)c.k + dst) = *reinterpret_cast<const uint4 *>(a);
        *reinterpret_cast<uint4 *>((D *)c.v + dst) = *reinterpret_cast<const uint4 *>(b);
    }
}

template <typename S, typename D>
static void launch_append(const CacheAppendArgs &a, cudaStream_t st) {
    const int64_t n = a.n_tokens * (a.cache.head_dim / 8) * a.cache.n_kv_heads;
    const int64_t want = (n + 255) / 256, grid = want > 148 * 8 ? 148 * 8 : want;
    k_cache_append<S, D><<<(unsigned)grid, 256, 0, st>>>((const S *)a.k, (const S *)a.v, a.k_stride, a.v_stride,
                                                         a.slots, a.n_tokens, a.cache);
}

template <typename D>
static void launch_append_from(const CacheAppendArgs &a, cudaStream_t st) {
    if (a.dtype == KK_DTYPE_F32)
        launch_append<float, D>(a, st);
    else if (a.dtype == KK_DTYPE_F16)
        launch_append<__half, D>(a, st);
    else
        launch_append<__nv_bfloat16, D>(a, st);
}

cudaError_t cache_append(const CacheAppendArgs &a, cudaStream_t st) {
    if (a.cache.bf16)
        launch_append_from<__nv_bfloat16>(a, st);
    else
        launch_append_from<__half>(a, st);
    return cudaGetLastError();
}

}  // namespace kk
