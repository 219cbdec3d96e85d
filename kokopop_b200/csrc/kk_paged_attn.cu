// Attention of a chunk of new tokens over a paged key / value cache (sm_100a).
//
// Request r has len = seq_len[r] tokens in the cache, the last n = cu_new[r+1]
// - cu_new[r] of which are the new ones whose queries are given: query t sits
// at position p = len - n + t and sees the keys j with max(0, p - window + 1)
// <= j <= p (window 0: from 0) whose page exists. For query head h on key
// head h / group:
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q . k_j,
//   m = max_j s_j,  and 0 for a query that sees no key.
// Scores, maxima, sums and the output are 32-bit; the weights e^(s - m) are
// rounded once to the cache's 16-bit type, which is what the tensor cores
// multiply (their relative error, 2^-8 or 2^-11 at most, is that of the
// rounded output; in half, weights below 2^-21 of the largest are rounded to
// multiples of 2^-31 of it), while the sum in the denominator takes them
// unrounded.
//
// k_paged_attn_row: for one or a few queries per key head, bytes bound it:
// every key and value of the request is read once for the `group` heads that
// share it. A block takes 8 or 16 rows (query, head of the group) of one key
// head and one piece of the key axis; each of its 4 warps walks blocks of 16
// keys of its own, with its own ring of copies in flight (no block barrier in
// the loop) and its own running maximum and sum. The products are transposed,
// S^T = K Q^T and O^T = V^T P^T, so that the 16 keys (or 16 dims) are the M
// side of mma.sync.m16n8k16 and the few rows its N side: nothing is computed
// for rows that do not exist beyond the next multiple of 8. The maximum is
// followed lazily as in kk_paged_chunk.cu, so most steps exchange nothing
// between lanes but one vote. Pages whose size is 8 or a multiple of 16 come
// by tensor copies (one lane issues a block's copy of 64 dims), others by
// 16-byte asynchronous copies. The warps are joined in shared memory, the
// pieces in global memory by the block that arrives last, in the order of the
// pieces, so that the result does not depend on which one that is.
//
// Measured on B200, 32 heads of 128 on 8, one token each: 7 requests of
// 30011-65000 keys 216 us, 6.8 TB/s of cache read (the copy rate is 6.55); 64
// requests of 17-4099 keys 97 us, 5.3 TB/s, where blocks start and end unevenly.
// In one piece, as under capture, the long ones take 686 us: 56 blocks.
#include "kk_paged_attn.cuh"
#include "kk_ptx.cuh"

#include <cuda.h>

#include <atomic>
#include <cstring>

namespace kk {

namespace {

constexpr int kKeys = 16;   // keys of a warp's step
constexpr int kWarps = 4;
constexpr int kFewRows = 16;  // query rows up to which a call takes this kernel
constexpr int kMaxPieces = 256;
constexpr float kGrow = 8.0f;  // base-2 growth of a maximum that is left alone

template <int DP, int NB>
struct RowCfg {
    static constexpr int ROWS = 8 * NB;
    // steps of a warp's ring: 96 KB a block, or 32 KB, which leaves room for
    // more blocks (heads of 64, 64 requests: 84 us with three steps, 78 with two)
    static constexpr int STAGES = DP > 64 ? 3 : 2;
    static constexpr int HALF_BYTES = kKeys * 128;   // 64 dims of a block of keys
    static constexpr int TILE = kKeys * DP * 2;      // K or V of one step
    static constexpr int RING = kWarps * STAGES * 2 * TILE;
    static constexpr int OS = DP + 4;                // row stride of the join: no bank twice
    static constexpr int JOIN = (kWarps * ROWS * (OS + 2) + ROWS * (kMaxPieces + 1)) * 4;
    static constexpr int SMEM = (RING > JOIN ? RING : JOIN) + 1024 /*align*/;
};

// 16 bytes of global memory, or zeros (live 0; src is then not read)
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int OFF>
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a), "n"(OFF)
                 : "memory");
}
template <int OFF>
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a), "n"(OFF)
                 : "memory");
}

// An 8 x 8 matrix of 16-bit values over the lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// 4 values of an output row, divided by the sum of its weights
template <typename T>
__device__ __forceinline__ void put_row4(T *out, float4 v, float l) {
    const float inv = paged_inverse(l);
    *reinterpret_cast<uint2 *>(out) =
        make_uint2(pack2(v.x * inv, v.y * inv, T()), pack2(v.z * inv, v.w * inv, T()));
}

}  // namespace

template <typename T, int DP, int NB, bool TMA>
__global__ void __launch_bounds__(kWarps * 32)
    k_paged_attn_row(PagedAttnArgs a, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v) {
    using C = RowCfg<DP, NB>;
    constexpr int KC = DP / 16;      // k-steps of a score, m-tiles of an output
    constexpr int HALVES = DP / 64;
    constexpr int CH = DP / 8;       // 16-byte chunks of a key
    extern __shared__ __align__(1024) unsigned char sm_raw[];
    unsigned char *sm = (unsigned char *)(((uintptr_t)sm_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bar_s[kWarps][C::STAGES];
    __shared__ uint32_t seen_s[kWarps][C::STAGES];
    __shared__ unsigned last_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const int group = a.n_heads / a.cache.n_kv_heads, kvh = blockIdx.y;
    const RowTile t = find_tile(a, group, C::ROWS, blockIdx.x);
    if (t.r < 0) return;  // the whole block
    const int D = a.cache.head_dim, page_size = a.cache.page_size;

    // the rows' positions and key ranges; the block's range and piece
    const int rows_here = min(C::ROWS, t.rows - t.row0);
    const int pos_first = t.base + t.row0 / group, pos_last = t.base + (t.row0 + rows_here - 1) / group;
    const int64_t cap = paged_capacity(a);
    // (a window wholly past the table leaves the block no key: k0 = k1, and no
    // step of the ring lies past 2^31)
    const int64_t lo = a.window > 0 ? min(max((int64_t)pos_first - a.window + 1, (int64_t)0), cap) : 0;
    const int64_t kbeg = lo / kKeys * kKeys, kend = lo < cap ? max(min((int64_t)pos_last + 1, cap), kbeg) : kbeg;
    // pieces: at most `splits`, of split_keys keys or more, then of one size
    const int64_t most = max((kend - kbeg + a.splits - 1) / a.splits, (int64_t)a.split_keys);
    const int64_t parts = max((kend - kbeg + most - 1) / most, (int64_t)1);
    const int64_t piece = max(((kend - kbeg + parts - 1) / parts + 63) / 64 * 64, (int64_t)64);
    const int n_pieces = (int)max((kend - kbeg + piece - 1) / piece, (int64_t)1);
    const int sp = blockIdx.z;
    if (sp >= n_pieces) return;
    // keys are below 2^31: positions are 32-bit
    const int k0 = (int)(kbeg + sp * piece), k1 = (int)min((int64_t)k0 + piece, kend);

    // this warp's steps: blocks of kKeys keys, kWarps apart
    unsigned char *ring = sm + warp * C::STAGES * 2 * C::TILE;
    const uint32_t ring_u = smem_u32(ring), bars = smem_u32(bar_s[warp]);
    const T *kc = (const T *)a.cache.k + kvh * a.cache.head_stride;
    const T *vc = (const T *)a.cache.v + kvh * a.cache.head_stride;
    const int32_t *table = a.table + (int64_t)t.r * a.max_pages;
    if (TMA) {
        if (lane == 0) {
            for (int i = 0; i < C::STAGES; ++i) mbar_init(bars + 8 * i, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
    }

    // TMA: the copy of this lane, 64 dims of one box of a page's tokens, of K or V
    const int boxes = page_size < kKeys ? 2 : 1, box = page_size < kKeys ? 8 : kKeys;
    const int part = lane & (boxes - 1), half = (lane >> (boxes - 1)) & (HALVES - 1),
              kv = lane >> (boxes - 1) >> (HALVES - 1);
    const uint32_t copy_to = ring_u + kv * C::TILE + half * C::HALF_BYTES + part * box * 128;
    const CUtensorMap *copy_map = kv ? &map_v : &map_k;
    const int page_bits = (page_size & (page_size - 1)) == 0 ? 31 - __clz(page_size) : -1;
    auto page_col = [&](int key) { return page_bits >= 0 ? key >> page_bits : key / page_size; };
    int next_key = k0 + warp * kKeys, next_stage = 0;  // of the next block to copy
    auto issue = [&] {
        if (next_key < k1) {
            const int key0 = next_key, st = next_stage;
            if (TMA) {
                const int key = key0 + part * box;
                int page = -1, off = 0;
                if (kv < 2 && key < k1) {
                    const int col = page_col(key);
                    page = table[col];
                    off = key - col * page_size;
                    if (page < 0 || page >= a.cache.n_pages) page = -1;
                }
                const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
                if (lane == 0) {
                    seen_s[warp][st] = boxes == 1 ? (have & 1 ? 0xffffu : 0u)
                                                  : (have & 1 ? 0xffu : 0u) | (have & 2 ? 0xff00u : 0u);
                    mbar_expect_tx(bars + 8 * st, 2 * C::TILE);
                }
                __syncwarp();
                if (kv < 2) tma_load_4d(copy_to + st * 2 * C::TILE, copy_map, bars + 8 * st, 64 * half, off, kvh, page);
            } else {
                // lane = key: where its row lies
                int64_t at = -1;
                const int key = key0 + (lane & (kKeys - 1));
                if (key < k1 && key >= lo) {
                    const int col = page_col(key), page = table[col];
                    if (page >= 0 && page < a.cache.n_pages)
                        at = page * a.cache.page_stride + (key - col * page_size) * a.cache.token_stride;
                }
                const uint32_t seen = __ballot_sync(0xffffffffu, at >= 0) & ((1u << kKeys) - 1);
                if (lane == 0) seen_s[warp][st] = seen;
#pragma unroll
                for (int i = lane; i < kKeys * CH; i += 32) {
                    const int row = i / CH, ch = i % CH;
                    const int64_t off = __shfl_sync(0xffffffffu, at, row);
                    const bool live = off >= 0 && ch * 8 < D;
                    const int64_t e = live ? off + ch * 8 : 0;
                    const uint32_t dst = ring_u + st * 2 * C::TILE + (ch >> 3) * C::HALF_BYTES + row * 128 +
                                         (((ch ^ row) & 7) * 16);
                    cp16(dst, kc + e, live);
                    cp16(dst + C::TILE, vc + e, live);
                }
            }
        }
        if (!TMA) cp_commit();
        next_key += kWarps * kKeys;
        next_stage = next_stage + 1 == C::STAGES ? 0 : next_stage + 1;
    };
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) issue();

    // Q^T fragments: columns (rows of Q) gid and, NB 2, gid + 8
    uint32_t qf[KC][NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int row = t.row0 + gid + 8 * b;
        const bool live = gid + 8 * b < rows_here;
        const T *q = (const T *)a.q + (t.tok0 + row / group) * a.q_stride + (int64_t)(kvh * group + row % group) * D;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const int d = k * 16 + tig * 2;
            qf[k][b][0] = live && d < D ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
            qf[k][b][1] = live && d + 8 < D ? *reinterpret_cast<const uint32_t *>(q + d + 8) : 0u;
        }
    }
    // the keys that this lane's columns (rows of Q 2 tig, 2 tig + 1) see
    int see_hi[NB][2], see_lo[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = 8 * b + 2 * tig + e, pos = t.base + (t.row0 + i) / group;
            see_hi[b][e] = i < rows_here ? pos : -1;
            see_lo[b][e] = i < rows_here && a.window > 0 ? pos - a.window + 1 : 0;
        }

    float o[KC][NB][4], mx[NB][2], sum[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        mx[b][0] = mx[b][1] = -INFINITY;
        sum[b][0] = sum[b][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KC; ++i) o[i][b][0] = o[i][b][1] = o[i][b][2] = o[i][b][3] = 0.f;
    }
    const float scale2 = a.scale * 1.4426950408889634f;  // scores in base 2
    // keys that every row sees need no mask
    const int all_lo = a.window > 0 ? pos_last - a.window + 1 : 0, all_hi = min(pos_first, k1 - 1);
    // lane's part of the fragments: K rows (m) and V rows (k, transposed)
    // their 16-byte chunk is XORed by the row, chunk 2 k + c of a half in two
    // steps: (c ^ row) 16 here, 2 k 16 where it is read
    const uint32_t k_at = ((lane & 7) + (lane & 8)) * 128 + ((lane >> 4 ^ lane) & 7) * 16;
    const uint32_t v_at = ((lane & 7) + (lane >> 4 << 3)) * 128 + ((lane >> 3 & 1 ^ lane) & 7) * 16;
    bool ok = true;
    int st = 0, phase = 0, key0 = k0 + warp * kKeys;
    for (; key0 < k1; key0 += kWarps * kKeys) {
        issue();
        if (TMA) {
            ok = mbar_wait_tight(bars + 8 * st, phase, a.err, kErrPagedWait);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
        } else {
            cp_wait<C::STAGES - 1>();
            __syncwarp();
        }
        const uint32_t kt = ring_u + st * 2 * C::TILE, vt = kt + C::TILE;
        const uint32_t seen = seen_s[warp][st];
        if (TMA && (key0 < lo || key0 + kKeys > k1)) {
            // values of tokens outside the range may be anything, and 0 times
            // a NaN is one: their rows become 0
            for (int i = lane; i < kKeys * CH; i += 32) {
                const int row = i / CH, ch = i % CH;
                if (key0 + row < lo || key0 + row >= k1)
                    *reinterpret_cast<uint4 *>(ring + (st * 2 + 1) * C::TILE + (ch >> 3) * C::HALF_BYTES + row * 128 +
                                               (ch & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async();  // before the next copy into this stage
            __syncwarp();
        }
        float sc[NB][4], sd[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
            sd[b][0] = sd[b][1] = sd[b][2] = sd[b][3] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < KC; k += 2) {  // two chains of products
            uint32_t f[4], g[4];
            const uint32_t at = (kt + k_at) ^ (k % 4 * 32), next = (kt + k_at) ^ ((k + 1) % 4 * 32);
            if (k < 4) {
                ldsm4<0>(at, f);
                ldsm4<0>(next, g);
            } else {
                ldsm4<C::HALF_BYTES>(at, f);
                ldsm4<C::HALF_BYTES>(next, g);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                mma16<T>(sc[b], f, qf[k][b][0], qf[k][b][1]);
                mma16<T>(sd[b], g, qf[k + 1][b][0], qf[k + 1][b][1]);
            }
        }
        bool grow = false;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[b][e] = (sc[b][e] + sd[b][e]) * scale2;
        if (key0 < all_lo || key0 + kKeys - 1 > all_hi || seen != (1u << kKeys) - 1) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = gid + 8 * (e >> 1), key = key0 + i;
                    if (!(seen >> i & 1) || key > see_hi[b][e & 1] || key < see_lo[b][e & 1] || key >= k1)
                        sc[b][e] = -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) grow |= fmaxf(sc[b][e], sc[b][e + 2]) > mx[b][e] + kGrow;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float corr[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = fmaxf(fmaxf(sc[b][e], sc[b][e + 2]), mx[b][e]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    corr[e] = m == mx[b][e] ? 1.f : pow2(mx[b][e] - m);
                    mx[b][e] = m;
                    sum[b][e] *= corr[e];
                }
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    o[i][b][0] *= corr[0], o[i][b][1] *= corr[1];
                    o[i][b][2] *= corr[0], o[i][b][3] *= corr[1];
                }
            }
        }
        uint32_t p[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float r0 = (mx[b][0] == -INFINITY ? 0.f : mx[b][0]) - kLift<T>,
                        r1 = (mx[b][1] == -INFINITY ? 0.f : mx[b][1]) - kLift<T>;
            const float x0 = pow2(sc[b][0] - r0), x1 = pow2(sc[b][1] - r1);
            const float y0 = pow2(sc[b][2] - r0), y1 = pow2(sc[b][3] - r1);
            sum[b][0] += x0 + y0;
            sum[b][1] += x1 + y1;
            // [key gid][row 2 tig, + 1] to [row gid][key 2 tig, + 1]
            p[b][0] = transpose8(pack2(x0, x1, T()));
            p[b][1] = transpose8(pack2(y0, y1, T()));
        }
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            uint32_t f[4];
            if (i < 4)
                ldsm4t<0>((vt + v_at) ^ (i % 4 * 32), f);
            else
                ldsm4t<C::HALF_BYTES>((vt + v_at) ^ (i % 4 * 32), f);
#pragma unroll
            for (int b = 0; b < NB; ++b) mma16<T>(o[i][b], f, p[b][0], p[b][1]);
        }
        __syncwarp();  // the stage is read before its next copies are issued
        st = st + 1 == C::STAGES ? (phase ^= 1, 0) : st + 1;
    }
    if (TMA) {
        if (!ok)  // the copies still in flight land before the block ends
            for (; key0 < min(next_key, k1); key0 += kWarps * kKeys) {
                mbar_wait(bars + 8 * st, phase, a.err, kErrPagedWait, TC_DRAIN_NS);
                st = st + 1 == C::STAGES ? (phase ^= 1, 0) : st + 1;
            }
    } else {
        cp_wait<0>();
    }
    __syncthreads();

    // join the warps: [warp][row][dim] values, then the maxima and sums
    float *jo = reinterpret_cast<float *>(sm);
    float *jm = jo + kWarps * C::ROWS * C::OS, *jl = jm + kWarps * C::ROWS, *jf = jl + kWarps * C::ROWS;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = sum[b][e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int row = warp * C::ROWS + 8 * b + 2 * tig + e;
            if (gid == 0) jm[row] = mx[b][e], jl[row] = l;
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                jo[row * C::OS + i * 16 + gid] = o[i][b][e];
                jo[row * C::OS + i * 16 + gid + 8] = o[i][b][e + 2];
            }
        }
    __syncthreads();
    // a thread takes 4 dims of a row at a time
    const int per_row = D / 4, items = rows_here * per_row;
    for (int it = tid; it < items; it += kWarps * 32) {
        const int row = it / per_row, d = (it - row * per_row) * 4, g = t.row0 + row;
        const int64_t tok = t.tok0 + g / group;
        const int head = kvh * group + g % group;
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, jm[w * C::ROWS + row]);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = pow2(jm[w * C::ROWS + row] - ref);
            l += f * jl[w * C::ROWS + row];
            const float4 x = *reinterpret_cast<const float4 *>(jo + (w * C::ROWS + row) * C::OS + d);
            acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
        }
        if (n_pieces > 1) {
            const int64_t part = (tok * a.n_heads + head) * a.splits + sp;
            *reinterpret_cast<float4 *>(a.part_o + part * D + d) = acc;
            if (d == 0) a.part_ml[part] = make_float2(m, l);
        } else {
            put_row4((T *)a.out + tok * a.out_stride + (int64_t)head * D + d, acc, l);
        }
    }
    if (n_pieces == 1) return;
    __threadfence();
    __syncthreads();
    unsigned *count = a.count + (int64_t)blockIdx.x * gridDim.y + kvh;
    if (tid == 0) last_s = atomicAdd(count, 1u) == (unsigned)n_pieces - 1;
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    if (tid == 0) *count = 0;
    // the factors of the pieces and the sum of each row, a warp per row
    for (int row = warp; row < rows_here; row += kWarps) {
        const int g = t.row0 + row;
        const int64_t part = ((t.tok0 + g / group) * a.n_heads + kvh * group + g % group) * a.splits;
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < n_pieces; i += 32) m = fmaxf(m, __ldcg(&a.part_ml[part + i]).x);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
        const float ref = m == -INFINITY ? 0.f : m;
        for (int i = lane; i < n_pieces; i += 32) {
            const float2 ml = __ldcg(&a.part_ml[part + i]);
            const float f = pow2(ml.x - ref);
            jf[row * (kMaxPieces + 1) + 1 + i] = f;
            l += f * ml.y;
        }
        l = warp_sum(l);
        if (lane == 0) jf[row * (kMaxPieces + 1)] = l;
    }
    __syncthreads();
    for (int it = tid; it < items; it += kWarps * 32) {
        const int row = it / per_row, d = (it - row * per_row) * 4, g = t.row0 + row;
        const int64_t tok = t.tok0 + g / group;
        const int head = kvh * group + g % group;
        const float *f = jf + row * (kMaxPieces + 1) + 1;
        const float *src = a.part_o + (tok * a.n_heads + head) * a.splits * D + d;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int i = 0; i < n_pieces; ++i) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(src + (int64_t)i * D));
            acc.x += f[i] * x.x, acc.y += f[i] * x.y, acc.z += f[i] * x.z, acc.w += f[i] * x.w;
        }
        put_row4((T *)a.out + tok * a.out_stride + (int64_t)head * D + d, acc, f[-1]);
    }
}

// Block of kKeys keys in whole boxes of a page, strides a tensor map takes.
static bool row_by_tensor(const PagedCacheView &c) {
    return (c.page_size == 8 || c.page_size % kKeys == 0) && paged_strides_mappable(c);
}

template <typename T, int DP, int NB, bool TMA>
static cudaError_t launch_row(const PagedAttnArgs &a, int64_t tiles, cudaStream_t st) {
    static std::atomic<bool> attr[64];
    using C = RowCfg<DP, NB>;
    cudaError_t e = dynamic_smem_once(k_paged_attn_row<T, DP, NB, TMA>, C::SMEM, attr);
    if (e != cudaSuccess) return e;
    CUtensorMap mk, mv;
    memset(&mk, 0, sizeof mk);
    memset(&mv, 0, sizeof mv);
    if (TMA) {
        e = paged_cache_maps(a.cache, kKeys, &mk, &mv);
        if (e != cudaSuccess) return e;
    }
    const dim3 grid((unsigned)tiles, (unsigned)a.cache.n_kv_heads, (unsigned)a.splits);
    k_paged_attn_row<T, DP, NB, TMA><<<grid, kWarps * 32, C::SMEM, st>>>(a, mk, mv);
    return cudaGetLastError();
}

template <typename T, int DP>
static cudaError_t launch_row_of(const PagedAttnPlan &p, const PagedAttnArgs &a, cudaStream_t st) {
    const bool tma = row_by_tensor(a.cache);
    if (p.unit == 8)
        return tma ? launch_row<T, DP, 1, true>(a, p.tiles, st) : launch_row<T, DP, 1, false>(a, p.tiles, st);
    return tma ? launch_row<T, DP, 2, true>(a, p.tiles, st) : launch_row<T, DP, 2, false>(a, p.tiles, st);
}

// Chunks of queries take the chunk kernel, whose blocks read the keys once for
// 256 rows but start and end slowly (about 5 us). Up to 48 rows over at most
// 1024 keys in many requests, the row kernel's smaller blocks are done sooner
// although they read the keys once per 16 rows. Measured on B200, row against
// chunk kernel, 300 and 1184 pairs of request and key head:
//   heads of 64   48 rows, 1024 keys 37 / 47 and 110 / 171 us; 17-41 rows, 410
//                 keys (608 pairs) 29 / 54 us
//   heads of 128  32 rows, 410 keys (608 pairs) 49 / 62, 1024 keys 80 / 98 us;
//                 18-41 rows, 30 on average, 1024 keys 88 / 93; 33 rows, 1024
//                 keys 102 / 93; 48 rows 69 / 52 and 233 / 187 us
// so that heads above 64 take it up to 32 rows on average. With less than two
// rounds of chunk blocks it loses: 148 pairs, 20 rows, 300 keys 17 / 15 and
// (heads of 128) 27 / 17 us.
PagedAttnPlan paged_attn_plan(const PagedCacheView &c, int n_heads, int64_t n_tokens, int n_seqs, int max_new,
                              int64_t keys) {
    const int group = n_heads / c.n_kv_heads;
    const int64_t most = n_tokens < max_new ? n_tokens : max_new, rows = most * group;
    // one request has `most` new tokens, each other busy one at least one
    const int64_t others = n_tokens - (most > 0 ? most : 1);
    PagedAttnPlan p;
    p.busy = others + 1 < n_seqs ? others + 1 : n_seqs;
    const bool short_rows = rows <= 48 && keys <= 1024 && p.busy * c.n_kv_heads >= 2 * 148 &&
                            (c.head_dim <= 64 || n_tokens * group <= 32 * p.busy);
    p.chunk = rows > kFewRows && !short_rows && paged_chunk_serves(c, n_heads);
    p.unit = p.chunk ? paged_chunk_unit(group) : rows > 8 ? 16 : 8;
    p.tiles = n_tokens * group / p.unit + n_seqs;
    return p;
}

cudaError_t paged_attn(const PagedAttnPlan &p, const PagedAttnArgs &a, cudaStream_t st) {
    if (p.chunk) return paged_chunk_attn(a, st);
    if (a.cache.head_dim <= 64)
        return a.cache.bf16 ? launch_row_of<__nv_bfloat16, 64>(p, a, st) : launch_row_of<__half, 64>(p, a, st);
    return a.cache.bf16 ? launch_row_of<__nv_bfloat16, 128>(p, a, st) : launch_row_of<__half, 128>(p, a, st);
}

}  // namespace kk
