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
// rounded output), while the sum in the denominator takes them unrounded.
//
// k_paged_attn_row: for one or a few queries per key head, bytes bound it:
// every key and value of the request is read once for the `group` heads that
// share it. A block takes 16 rows (query, head of the group) of one key head
// as the M = 16 side of mma.sync.m16n8k16, so that a single token of a group
// of up to 16 heads reads its keys once; one piece of the key axis per block
// keeps all SMs reading when there are few rows. Each of the 4 warps walks its
// own blocks of 16 keys with its own ring of asynchronous 16-byte copies (no
// block barrier in the loop) and its own running maximum and sum; the warps
// are joined in shared memory, the pieces in global memory by the block that
// arrives last, in the order of the pieces, so that the result does not
// depend on which one that is.
#include "kk_paged_attn.cuh"

#include <atomic>

namespace kk {

namespace {

constexpr int kRows = 16;   // query rows of a block
constexpr int kKeys = 16;   // keys of a warp's step
constexpr int kWarps = 4;
constexpr int kStages = 3;

template <int DP>
struct RowCfg {
    static constexpr int ROW_BYTES = DP * 2;
    static constexpr int TILE = kKeys * ROW_BYTES;  // K or V of one step
    static constexpr int RING = kWarps * kStages * 2 * TILE;
    static constexpr int JOIN = kWarps * kRows * (DP + 2) * 4;
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes of global memory, or zeros (live 0; src is then not read)
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                     uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace

template <typename T, int DP>
__global__ void __launch_bounds__(kWarps * 32) k_paged_attn_row(PagedAttnArgs a) {
    using C = RowCfg<DP>;
    constexpr int KC = DP / 16;      // k-steps of a score
    constexpr int NT = DP / 8;       // n-tiles of an output row
    constexpr int CH = DP / 8;       // 16-byte chunks of a key
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ uint32_t seen_s[kWarps][kStages];
    __shared__ unsigned last_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const int group = a.n_heads / a.cache.n_kv_heads, kvh = blockIdx.y;
    const RowTile t = find_tile(a, group, kRows, blockIdx.x);
    if (t.r < 0) return;  // the whole block
    const int D = a.cache.head_dim;

    // the rows' positions and key ranges; the block's range
    const int base = t.base;
    const int rows_here = min(kRows, t.rows - t.row0);
    const int pos_first = base + t.row0 / group, pos_last = base + (t.row0 + rows_here - 1) / group;
    int64_t kend = min((int64_t)pos_last + 1, (int64_t)a.max_pages * a.cache.page_size);
    int64_t kbeg = a.window > 0 ? max((int64_t)pos_first - a.window + 1, (int64_t)0) : 0;
    kbeg = kbeg / kKeys * kKeys;
    if (kend < kbeg) kend = kbeg;
    // pieces: at least split_keys keys each, so that splits of them reach the end
    int64_t piece = (kend - kbeg + a.splits - 1) / a.splits;
    piece = max((piece + 63) / 64 * 64, (int64_t)a.split_keys);
    const int n_pieces = (int)max((kend - kbeg + piece - 1) / piece, (int64_t)1);
    const int sp = blockIdx.z;
    if (sp >= n_pieces) return;
    const int64_t k0 = kbeg + sp * piece, k1 = min(k0 + piece, kend);

    // Q fragments: rows gid and gid + 8
    uint32_t qf[KC][4];
    int lim_hi[2], lim_lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = t.row0 + gid + 8 * i;
        const bool live = gid + 8 * i < rows_here;
        const int tok = row / group, head = kvh * group + row % group;
        lim_hi[i] = live ? base + tok : -1;
        lim_lo[i] = live && a.window > 0 ? base + tok - a.window + 1 : 0;
        const T *q = (const T *)a.q + (t.tok0 + tok) * a.q_stride + (int64_t)head * D;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const int d = k * 16 + tig * 2;
            qf[k][i] = live && d < D ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
            qf[k][2 + i] = live && d + 8 < D ? *reinterpret_cast<const uint32_t *>(q + d + 8) : 0u;
        }
    }

    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

    // this warp's steps: blocks of kKeys keys, kWarps apart
    const int n_blocks = (int)((k1 - k0 + kKeys - 1) / kKeys);
    const int n_steps = n_blocks > warp ? (n_blocks - warp + kWarps - 1) / kWarps : 0;
    unsigned char *ring = sm + warp * kStages * 2 * C::TILE;
    const T *kc = (const T *)a.cache.k + kvh * a.cache.head_stride;
    const T *vc = (const T *)a.cache.v + kvh * a.cache.head_stride;
    const int32_t *table = a.table + (int64_t)t.r * a.max_pages;

    auto issue = [&](int s) {
        if (s < n_steps) {
            const int64_t key0 = k0 + (int64_t)(warp + s * kWarps) * kKeys;
            // lane = key: where its row lies
            int64_t at = -1;
            const int64_t key = key0 + (lane & (kKeys - 1));
            if (key < k1) {
                const int64_t col = key / a.cache.page_size;
                const int page = table[col];
                if (page >= 0 && page < a.cache.n_pages)
                    at = page * a.cache.page_stride + (key - col * a.cache.page_size) * a.cache.token_stride;
            }
            const uint32_t seen = __ballot_sync(0xffffffffu, at >= 0) & ((1u << kKeys) - 1);
            unsigned char *kt = ring + (s % kStages) * 2 * C::TILE;
            if (lane == 0) seen_s[warp][s % kStages] = seen;
#pragma unroll
            for (int i = lane; i < kKeys * CH; i += 32) {
                const int row = i / CH, ch = i % CH;
                const int64_t off = __shfl_sync(0xffffffffu, at, row);
                const bool live = off >= 0 && ch * 8 < D;
                const int64_t e = live ? off + ch * 8 : 0;
                const uint32_t dst = smem_addr(kt) + row * C::ROW_BYTES + ((ch ^ (row & 7)) * 16);
                cp16(dst, kc + e, live);
                cp16(dst + C::TILE, vc + e, live);
            }
        }
        cp_commit();
    };

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    const float scale2 = a.scale * 1.4426950408889634f;  // scores in base 2
    for (int s = 0; s < n_steps; ++s) {
        issue(s + kStages - 1);
        cp_wait<kStages - 1>();
        __syncwarp();
        const uint32_t kt = smem_addr(ring + (s % kStages) * 2 * C::TILE), vt = kt + C::TILE;
        const uint32_t seen = seen_s[warp][s % kStages];
        const int64_t key0 = k0 + (int64_t)(warp + s * kWarps) * kKeys;
        float sc[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            // 16 keys x 16 dims: matrices (keys 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
            const int row = (lane & 7) + ((lane >> 4) << 3), ch = 2 * k + ((lane >> 3) & 1);
            uint32_t b[4];
            ldsm4(kt + row * C::ROW_BYTES + ((ch ^ (row & 7)) * 16), b);
            mma16<T>(sc[0], qf[k], b[0], b[1]);
            mma16<T>(sc[1], qf[k], b[2], b[3]);
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = i * 8 + tig * 2 + (e & 1), h = e >> 1;
                const int64_t key = key0 + col;
                const bool live = (seen >> col & 1) && key <= lim_hi[h] && key >= lim_lo[h];
                sc[i][e] = live ? sc[i][e] * scale2 : -INFINITY;
                top[h] = fmaxf(top[h], sc[i][e]);
            }
        uint32_t p[4];
        float corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            const float m = fmaxf(mx[h], top[h]);
            const float ref = m == -INFINITY ? 0.f : m;  // no key so far: every weight 0
            corr[h] = exp2f(mx[h] - ref);
            mx[h] = m;
            float add = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float x = exp2f(sc[i][2 * h] - ref), y = exp2f(sc[i][2 * h + 1] - ref);
                add += x + y;
                p[2 * i + h] = pack2(x, y, T());
            }
            sum[h] = sum[h] * corr[h] + add;
        }
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
            // 16 keys x 16 dims of V, transposed: (keys 0-7, d 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
            const int row = (lane & 15), ch = 2 * j + (lane >> 4);
            uint32_t b[4];
            ldsm4t(vt + row * C::ROW_BYTES + ((ch ^ (row & 7)) * 16), b);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float(&c)[4] = o[2 * j + i];
                c[0] *= corr[0], c[1] *= corr[0], c[2] *= corr[1], c[3] *= corr[1];
                mma16<T>(c, p, b[2 * i], b[2 * i + 1]);
            }
        }
        __syncwarp();  // the stage is read before its next copies are issued
    }
    cp_wait<0>();
    __syncthreads();

    // join the warps: [warp][row][DP] values, then the maxima and sums
    float *jo = reinterpret_cast<float *>(sm);
    float *jm = jo + kWarps * kRows * DP, *jl = jm + kWarps * kRows;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        const int row = warp * kRows + gid + 8 * h;
        if (tig == 0) jm[row] = mx[h], jl[row] = sum[h];
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<float2 *>(jo + row * DP + j * 8 + tig * 2) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
    }
    __syncthreads();
    constexpr int PER = kRows * DP / (kWarps * 32);  // values of a thread: PER of one row
    const int row = tid * PER / DP, d0 = tid * PER % DP;
    const bool live = row < rows_here;
    const int g = t.row0 + row;
    const int64_t tok = t.tok0 + g / group;
    const int head = kvh * group + g % group;
    float m = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, jm[w * kRows + row]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const float f = exp2f(jm[w * kRows + row] - ref);
        l += f * jl[w * kRows + row];
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] += f * jo[(w * kRows + row) * DP + d0 + i];
    }
    if (n_pieces > 1) {
        const int64_t part = (tok * a.n_heads + head) * a.splits;
        if (live) {
            for (int i = 0; i < PER; ++i)
                if (d0 + i < D) a.part_o[(part + sp) * D + d0 + i] = acc[i];
            if (d0 == 0) a.part_ml[part + sp] = make_float2(m, l);
        }
        __threadfence();
        __syncthreads();
        unsigned *count = a.count + (int64_t)blockIdx.x * gridDim.y + kvh;
        if (tid == 0) last_s = atomicAdd(count, 1u) == (unsigned)n_pieces - 1;
        __syncthreads();
        if (!last_s) return;
        __threadfence();
        if (tid == 0) *count = 0;
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = 0.f;
        if (live) {
            for (int s = 0; s < n_pieces; ++s) m = fmaxf(m, __ldcg(&a.part_ml[part + s]).x);
            const float all = m == -INFINITY ? 0.f : m;
            for (int s = 0; s < n_pieces; ++s) {
                const float2 ml = __ldcg(&a.part_ml[part + s]);
                const float f = exp2f(ml.x - all);
                l += f * ml.y;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (d0 + i < D) acc[i] += f * __ldcg(&a.part_o[(part + s) * D + d0 + i]);
            }
        }
    }
    if (live) {
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // a NaN sum stays one
        T *out = (T *)a.out + tok * a.out_stride + (int64_t)head * D;
#pragma unroll
        for (int i = 0; i < PER; i += 2)
            if (d0 + i < D) *reinterpret_cast<uint32_t *>(out + d0 + i) = pack2(acc[i] * inv, acc[i + 1] * inv, T());
    }
}

template <typename T, int DP>
static cudaError_t launch_row(const PagedAttnArgs &a, int64_t tiles, cudaStream_t st) {
    static std::atomic<bool> attr[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!attr[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(k_paged_attn_row<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 RowCfg<DP>::SMEM);
        if (e != cudaSuccess) return e;
        attr[dev].store(true, std::memory_order_release);
    }
    const dim3 grid((unsigned)tiles, (unsigned)a.cache.n_kv_heads, (unsigned)a.splits);
    k_paged_attn_row<T, DP><<<grid, kWarps * 32, RowCfg<DP>::SMEM, st>>>(a);
    return cudaGetLastError();
}

PagedAttnPlan paged_attn_plan(const PagedCacheView &c, int n_heads, int64_t n_tokens, int n_seqs, int max_new) {
    const int group = n_heads / c.n_kv_heads;
    const int64_t rows = (n_tokens < max_new ? n_tokens : max_new) * (int64_t)group;
    PagedAttnPlan p;
    p.chunk = rows > kRows && paged_chunk_serves(c, n_heads);
    p.unit = p.chunk ? paged_chunk_unit(group) : kRows;
    p.tiles = n_tokens * group / p.unit + n_seqs;
    return p;
}

cudaError_t paged_attn(const PagedAttnPlan &p, const PagedAttnArgs &a, cudaStream_t st) {
    if (p.chunk) return paged_chunk_attn(a, st);
    if (a.cache.head_dim <= 64)
        return a.cache.bf16 ? launch_row<__nv_bfloat16, 64>(a, p.tiles, st) : launch_row<__half, 64>(a, p.tiles, st);
    return a.cache.bf16 ? launch_row<__nv_bfloat16, 128>(a, p.tiles, st) : launch_row<__half, 128>(a, p.tiles, st);
}

}  // namespace kk
