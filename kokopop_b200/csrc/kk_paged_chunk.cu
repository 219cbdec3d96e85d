// Attention of chunks of new tokens over the paged cache on the 5th-generation
// tensor cores (sm_100a); the definition is in kk_paged_attn.cu. With many
// query rows per key head the arithmetic bounds it: 4 head_dim operations per
// (row, key), and one exponential, of which an SM does 16 a clock.
//
// A block takes two tiles of up to 128 rows (query, head of the group) of one
// key head and one piece of the key axis, 128 keys a step:
//   S = Q K^T      128 x 128 x head_dim, into tensor memory
//   P = e^(S - m)  by 128 threads (thread = row = lane of tensor memory), which
//                  hold a row of S in registers, back as 16 bits
//   O += P V       P from tensor memory, V as it lies (keys x dims)
// No row needs a reduction between threads. Tensor memory holds one S, which
// the tiles use in turn: as soon as a tile's threads have read theirs, the
// other tile's is computed, so that no product waits for a softmax nor for
// another product; P has columns of its own. (With an S for each tile and P
// over it, the next S waited for the product that reads P: 485 us where this
// takes 444.) m follows the running maximum lazily: O is rescaled only when the
// maximum has grown by more than 8 in base 2 (the weights stay below 2^8, or
// 2^15 in half, see kLift), which after the first steps is rare; the result
// does not depend on m but for rounding.
//
// Roles: warps 0-3 and 4-7 softmax and output of the two tiles, warp 8 issues
// the products with K, warp 10 those with V, warp 9 the copies (11 only fills
// its warpgroup). Keys and values come page by page through 4-D tensor maps
// (dim, token, head, page) into 128-byte swizzled tiles, so any stride order
// of the cache is served; pages that are missing or hold no key of the tile
// are fetched from outside the tensor and read as zeros. Values of tokens
// outside the block's key range may be anything, and 0 times a NaN is one:
// their rows are zeroed in shared memory in the steps at the two ends.
//
// Measured on B200: 3 requests, 1590-2048 new tokens at the end of 5890-7300,
// 32 heads of 128 on 8, 476 GFLOP under the masks: 444 us, 1.07 PFLOP/s, in
// short loops (0.65 of the measured burst rate), 495 us, 0.96 PFLOP/s, in long
// ones at the power limit (0.70 of the sustained rate). The softmax bounds it:
// without its exponentials 385 us in short loops. Head dims between 64 and 128
// cost what 128 does: both products run over the padded tile.
#include "kk_paged_attn.cuh"
#include "kk_ptx.cuh"

#include <cudaTypedefs.h>

#include <atomic>

namespace kk {

namespace {

constexpr int kTile = 128;       // rows of a tile, keys of a step
constexpr int kStages = 2;       // pairs of a V tile and the next step's K tile
constexpr int kThreads = 384;
// registers of a thread: 168 at launch (3 warpgroups), moved from the copy and
// MMA warpgroup to the two that hold a row of scores: 72 + 2 x 216 = 3 x 168
constexpr int kRegsFew = 72, kRegsMany = 216;
constexpr int kScoreWarp = 8, kCopyWarp = 9, kValueWarp = 10;
constexpr float kGrow = 8.0f;    // base-2 growth of a maximum that is left alone

template <int DP>
struct ChunkCfg {
    static constexpr int TILE_BYTES = kTile * DP * 2;
    static constexpr int HALF_BYTES = kTile * 128;   // 64 dims of a tile
    static constexpr int SMEM = (2 + 2 * kStages) * TILE_BYTES + 1024 /*barriers*/ + 1024 /*align*/;
    // tensor memory columns: S of either tile in turn, P and O of both
    static constexpr int S0 = 0, P0 = kTile, O0 = 2 * kTile;
    static constexpr int COLS = 512;
};
static_assert(ChunkCfg<128>::SMEM <= 227 * 1024, "shared memory");

// Shared-memory matrix descriptors, 128-byte swizzle, as two words: the upper
// one (SBO 1024 bytes between blocks of 8 rows, version 1 at bit 46, swizzle
// mode 2 in [61,64)) is the same for all, the lower one is start >> 4 and
// LBO >> 4 at bit 16, so that a step in shared memory is one 32-bit addition.
constexpr uint32_t kDescHi = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
    return (addr >> 4 & 0x3FFFu) | (lbo >> 4) << 16;
}

// Instruction descriptor, kind::f16: D F32, A and B half (0) or bfloat16 (1)
// at bits 7 and 10, B transposed (its rows are the sum's axis) at bit 16.
__device__ __forceinline__ constexpr uint32_t idesc_of(int bf16, int b_rows, int n) {
    return idesc_f16(kTile, n) | (uint32_t)bf16 << 7 | (uint32_t)bf16 << 10 | (uint32_t)b_rows << 16;
}

// one lane of the warp, the same in every call
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}

// Whether v holds in any of the 256 softmax threads (named barrier 1).
__device__ __forceinline__ bool any_of_barrier(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v)
        : "memory");
    return r != 0;
}

// D[tmem] (+)= A[shared] B[shared]
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
        : "memory");
}

// D[tmem] (+)= A[tmem] B[shared]
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
        : "memory");
}

#define KK_R32(r) \
    "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), \
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), \
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), \
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
// 32 columns of this thread's lane, without the wait
__device__ __forceinline__ void tmem_get32(uint32_t taddr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : KK_R32(r)
        : "r"(taddr));
}
#undef KK_R32
__device__ __forceinline__ void tmem_get_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_put32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
}  // namespace

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_paged_attn_chunk(PagedAttnArgs a, const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using C = ChunkCfg<DP>;
    constexpr int HALVES = DP / 64;
    constexpr int BF16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.n_heads / a.cache.n_kv_heads, kvh = blockIdx.y, D = a.cache.head_dim;
    const int tile_tok = kTile / group;  // tokens of a tile
    // the last tiles of a request see the most keys: first
    const RowTile t = find_tile(a, group, 2 * tile_tok * group, gridDim.x - 1 - blockIdx.x);
    if (t.r < 0) return;  // the whole block

    // the tiles' tokens and key ranges, the block's piece of the keys
    const int64_t cap = paged_capacity(a);
    const int tok_first = t.row0 / group;
    int tok[2], n_tok[2], n_step[2];
    int64_t hi[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        tok[x] = tok_first + x * tile_tok;
        n_tok[x] = max(min(t.n - tok[x], tile_tok), 0);
        hi[x] = n_tok[x] > 0 ? max(min((int64_t)t.base + tok[x] + n_tok[x], cap), (int64_t)0) : 0;
    }
    // (a window wholly past the table leaves the block no key: k0 = k1)
    const int64_t lo = a.window > 0 ? min(max((int64_t)t.base + tok_first - a.window + 1, (int64_t)0), cap) : 0;
    const int64_t kbeg = lo / kTile * kTile, kend = lo < cap ? max(max(hi[0], hi[1]), kbeg) : kbeg;
    // pieces: at most `splits`, of split_keys keys or more, then of one size
    const int64_t most = max((kend - kbeg + a.splits - 1) / a.splits, (int64_t)a.split_keys);
    const int64_t parts = max((kend - kbeg + most - 1) / most, (int64_t)1);
    const int64_t piece = max(((kend - kbeg + parts - 1) / parts + kTile - 1) / kTile * kTile, (int64_t)kTile);
    const int n_pieces = (int)max((kend - kbeg + piece - 1) / piece, (int64_t)1);
    const int sp = blockIdx.z;
    if (sp >= n_pieces) return;
    const int64_t k0 = kbeg + sp * piece, k1 = min(k0 + piece, kend);
#pragma unroll
    for (int x = 0; x < 2; ++x) n_step[x] = (int)((max(min(k1, hi[x]) - k0, (int64_t)0) + kTile - 1) / kTile);
    const int steps = max(n_step[0], n_step[1]);
    const int32_t *table = a.table + (int64_t)t.r * a.max_pages;
    const int page_size = a.cache.page_size;

    uint8_t *sQ = smem, *sKV = smem + 2 * C::TILE_BYTES;
    const uint32_t bars = smem_u32(sKV + 2 * kStages * C::TILE_BYTES);
    const uint32_t bQ = bars, bFull = bars + 16, bEmpty = bFull + 8 * kStages, bS = bEmpty + 8 * kStages,
                   bP = bS + 16, bPV = bP + 32, bDrain = bPV + 16, bFree = bDrain + 16;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bQ + 8 * i, 1);
            mbar_init(bS + 8 * i, 1);
            mbar_init(bP + 16 * i, 4);      // the four warps of a tile, keys 0-63
            mbar_init(bP + 16 * i + 8, 4);  // keys 64-127
            mbar_init(bPV + 8 * i, 1);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(bFull + 8 * i, 1);
            mbar_init(bEmpty + 8 * i, 2);  // both issuers
        }
        mbar_init(bDrain, 1);
        mbar_init(bDrain + 8, 1);
        mbar_init(bFree, 4);  // the softmax warps of the tile whose scores they are
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kScoreWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                     "r"(C::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_s;

    // The roles part here for good: each side has its own register budget, and
    // they meet once more at the block barrier that frees tensor memory.
    if (warp >= kScoreWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
        if (warp == kCopyWarp) {
            // Q of both tiles, then pair i = (V of step i - 1, K of step i) into
            // stage i % kStages; the first has no V, the last no K
            if (lane == 0)
                for (int x = 0; x < 2; ++x)
                    if (n_step[x] > 0) {
                        mbar_expect_tx(bQ + 8 * x, (uint32_t)(tile_tok * group * 128 * HALVES));
                        for (int h = 0; h < HALVES; ++h)
                            tma_load_3d(smem_u32(sQ + x * C::TILE_BYTES + h * C::HALF_BYTES), &map_q, bQ + 8 * x,
                                        64 * h, kvh * group, (int)(t.tok0 + tok[x]));
                    }
            const int box = min(page_size, kTile);           // tokens of a copy
            const int boxes = kTile / box;                   // copies of 64 dims of a tile
            const int part = lane % boxes, half = lane / boxes;
            const int pairs = steps > 0 ? steps + 1 : 0;
            int page = -1, off = 0;  // of the K of the pair before, the V of this one
            bool ok = true;
            int i = 0;
            for (; i < pairs; ++i) {
                const int page_v = page, off_v = off;
                const int64_t key = k0 + (int64_t)i * kTile + part * box;
                page = -1;
                if (half < HALVES && key < k1 && key + box > lo) {
                    const int col = (int)key / page_size;
                    page = table[col];
                    off = (int)key - col * page_size;
                    if (page < 0 || page >= a.cache.n_pages) page = -1;
                }
                const int s = i % kStages;
                const uint32_t bar = bFull + 8 * s, at = smem_u32(sKV + 2 * s * C::TILE_BYTES);
                if (lane == 0) {
                    if (i >= kStages) ok = mbar_wait_tight(bEmpty + 8 * s, (i / kStages - 1) & 1, a.err, kErrPagedWait);
                    if (ok) mbar_expect_tx(bar, (i > 0 && i < steps ? 2 : 1) * C::TILE_BYTES);
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                if (!ok) break;
                if (half < HALVES) {
                    const uint32_t to = at + half * C::HALF_BYTES + part * box * 128;
                    if (i > 0) tma_load_4d(to, &map_v, bar, 64 * half, off_v, kvh, page_v);
                    if (i < steps) tma_load_4d(to + C::TILE_BYTES, &map_k, bar, 64 * half, off, kvh, page);
                }
            }
            // the last copy into each stage has landed (consumed already, unless
            // a wait ran out)
            if (lane == 0) {
                for (int c = max(i - kStages, 0); c < i; ++c)
                    mbar_wait(bFull + 8 * (c % kStages), (c / kStages) & 1, a.err, kErrPagedWait, TC_DRAIN_NS);
                for (int x = 0; x < 2; ++x)
                    if (n_step[x] > 0) mbar_wait(bQ + 8 * x, 0, a.err, kErrPagedWait, TC_DRAIN_NS);
            }
            __syncwarp();
        } else if (warp == kScoreWarp || warp == kValueWarp) {
            // One warp issues the products with K, the other those with V.
            // Both walk the steps whole, so that every operand of an MMA is
            // the same in all lanes and sits in a uniform register; one
            // elected lane issues. (Issued from code of one lane, an MMA of 64
            // clocks cost 75-105 clocks of issue.)
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
            const int n0 = __shfl_sync(0xffffffffu, n_step[0], 0), n1 = __shfl_sync(0xffffffffu, n_step[1], 0);
            const int all = max(n0, n1);
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity) {
                ok = __all_sync(0xffffffffu, mbar_wait_tight(bar, parity, a.err, kErrPagedWait));
                return ok;
            };
            if (warp == kScoreWarp) {
                constexpr uint32_t id = idesc_of(BF16, 0, kTile);
                const uint32_t dq = desc_lo(base, 16), dk = desc_lo(base + 3 * C::TILE_BYTES, 16);
                int turn = 0;  // of the scores' columns
                for (int j = 0; j < all && ok; ++j) {
                    const int s = j % kStages;  // K of step j is in pair j
                    if (!wait(bFull + 8 * s, j / kStages & 1)) break;
                    const uint32_t k = dk + 2 * s * (C::TILE_BYTES >> 4);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (j >= (x ? n1 : n0)) continue;
                        if (j == 0 && !wait(bQ + 8 * x, 0)) break;
                        // the scores before have been read
                        if (turn > 0 && !wait(bFree, (turn - 1) & 1)) break;
                        ++turn;
                        fence_after_sync();
                        if (elect_one()) {
#pragma unroll
                            for (int d = 0; d < DP / 16; ++d) {
                                const uint32_t at = (d / 4 * C::HALF_BYTES + d % 4 * 32) >> 4;
                                mma_ss(tm + C::S0, dq + (x * C::TILE_BYTES >> 4) + at, k + at, id, d > 0);
                            }
                            mma_commit(bS + 8 * x);
                        }
                        __syncwarp();
                    }
                    if (ok && elect_one()) mma_commit(bEmpty + 8 * s);
                    __syncwarp();
                }
            } else {
                constexpr uint32_t id = idesc_of(BF16, 1, DP);
                const uint32_t dv = desc_lo(base + 2 * C::TILE_BYTES, C::HALF_BYTES);
                if (all > 0) {  // pair 0 has no V
                    if (elect_one()) mbar_arrive(bEmpty);
                    __syncwarp();
                }
                const int r_lo = (int)max(min(lo - k0, (int64_t)kTile), (int64_t)0);  // rows of step 0 below the keys
                for (int j = 0; j < all && ok; ++j) {
                    const int s = (j + 1) % kStages;  // V of step j is in pair j + 1
                    if (!wait(bFull + 8 * s, (j + 1) / kStages & 1)) break;
                    // the rows of V outside the block's keys become 0
                    const int r_hi = (int)min(k1 - k0 - (int64_t)j * kTile, (int64_t)kTile);
                    if ((j == 0 && r_lo > 0) || r_hi < kTile) {
                        uint8_t *v = sKV + 2 * s * C::TILE_BYTES;
                        for (int e = lane; e < kTile * HALVES * 8; e += 32) {
                            const int row = (e >> 3) % kTile, h = e / (kTile * 8);
                            if ((j == 0 && row < r_lo) || row >= r_hi)
                                *reinterpret_cast<uint4 *>(v + h * C::HALF_BYTES + row * 128 + (e & 7) * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                    const uint32_t v = dv + 2 * s * (C::TILE_BYTES >> 4);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (j >= (x ? n1 : n0)) continue;
                        // O += P V, the first 64 keys as soon as their weights are there
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (!wait(bP + 16 * x + 8 * h, j & 1)) break;
                            fence_after_sync();
                            if (elect_one()) {
#pragma unroll
                                for (int k = 4 * h; k < 4 * h + 4; ++k)
                                    mma_ts(tm + C::O0 + x * DP, tm + C::P0 + x * (kTile / 2) + k * 8,
                                           v + (k * 2048 >> 4), id, j > 0 || k > 0);
                                if (h == 1) mma_commit(bPV + 8 * x);
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                    }
                    if (ok && elect_one()) mma_commit(bEmpty + 8 * s);
                    __syncwarp();
                }
            }
            // every MMA issued has completed before tensor memory is freed
            const uint32_t drain = bDrain + (warp == kValueWarp ? 8 : 0);
            if (elect_one()) mma_commit(drain);
            __syncwarp();
            mbar_wait(drain, 0, a.err, kErrPagedWait, TC_DRAIN_NS);
        }
        asm volatile("bar.sync 0;" ::: "memory");
        if (warp == kScoreWarp) {
            fence_after_sync();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
        const int x = warp >> 2, row = tid & (kTile - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
        const uint32_t tS = tmem + C::S0 + lanes, tO = tmem + C::O0 + x * DP + lanes,
                       tP = tmem + C::P0 + x * (kTile / 2) + lanes;
        const int i = row / group;
        const bool live = i < n_tok[x] && row < tile_tok * group;
        const int64_t tq = t.tok0 + tok[x] + i;
        const int head = kvh * group + row % group;
        // the keys this row sees, [see_lo, see_hi), counted from k0
        const int64_t pos = (int64_t)t.base + tok[x] + i;
        const int see_hi = live ? (int)(min(min(pos + 1, cap), k1) - k0) : 0;
        const int see_lo = a.window > 0 ? (int)(pos - a.window + 1 - k0) : 0;
        // scores in base 2; a negative scale is the positive one of -S, and a
        // scale of 0 a tiny one (masked scores are -inf, and 0 inf is a NaN)
        const float sc = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
        const bool flip = a.scale < 0.f;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const int n = x ? n_step[1] : n_step[0];
        // whether a page of the block's keys is missing, looked up while the
        // first copies are under way (k0 is at most the table's end: without a
        // key the loop reads nothing, or a column of the table)
        bool gone = false;
        for (int64_t key = k0 / page_size * page_size + (int64_t)tid * page_size; key < k1;
             key += (int64_t)2 * kTile * page_size) {
            const int page = table[(int)key / page_size];
            gone |= page < 0 || page >= a.cache.n_pages;
        }
        const bool any_missing = any_of_barrier(gone);
        for (int j = 0; j < n && ok; ++j) {
            const int c0 = see_lo - j * kTile, c1 = see_hi - j * kTile;  // the columns seen, [c0, c1)
            ok = mbar_wait_tight(bS + 8 * x, j & 1, a.err, kErrPagedWait);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after_sync();
            float s[kTile];
#pragma unroll
            for (int c = 0; c < kTile; c += 32) tmem_get32(tS + c, s + c);
            tmem_get_wait();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bFree);
            if (flip) {
#pragma unroll
                for (int c = 0; c < kTile; ++c) s[c] = -s[c];
            }
            // masked scores
            if (c0 > 0 || c1 < kTile || any_missing) {
#pragma unroll
                for (int c = 0; c < kTile; ++c)
                    if (c < c0 || c >= c1) s[c] = -INFINITY;
                if (any_missing) {
#pragma unroll
                    for (int w = 0; w < kTile; w += 32) {
                        uint32_t hide = 0;  // pages are whole blocks of 8 keys
                        const int key = (int)k0 + j * kTile + w;
                        for (int c = 0; c < 32 && key + c < k1; c += 8) {
                            const int page = table[(key + c) / page_size];
                            if (page < 0 || page >= a.cache.n_pages) hide |= 0xffu << c;
                        }
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (hide >> c & 1) s[w + c] = -INFINITY;
                    }
                }
            }
            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < kTile; ++c) top[c & 3] = fmaxf(top[c & 3], s[c]);
            const float m_new = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m);
            // P and O of the step before have been read and written
            if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait_tight(bPV + 8 * x, (j - 1) & 1, a.err, kErrPagedWait));
                if (!ok) break;
                fence_after_sync();
            }
            if (j == 0) {
                m = m_new;
            } else if (__any_sync(0xffffffffu, (m_new - m) * sc > kGrow)) {
                const float f = m_new == m ? 1.f : pow2((m - m_new) * sc);
                m = m_new;
                l *= f;
#pragma unroll
                for (int c = 0; c < DP; c += 32) {
                    float o[32];
                    tmem_get32(tO + c, o);
                    tmem_get_wait();
                    uint32_t u[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(o[e] * f);
                    tmem_put32(tO + c, u);
                }
            }
            float ref = m == -INFINITY ? 0.f : -m * sc;
            if constexpr (kLift<T> != 0.f) ref += kLift<T>;  // an addition of 0 would stay in the code
            const float2 sc2 = make_float2(sc, sc), ref2 = make_float2(ref, ref);
            float2 add = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kTile; c += 64) {
                uint32_t u[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float2 y = f2fma(make_float2(s[c + 2 * e], s[c + 2 * e + 1]), sc2, ref2);
                    const float2 p = make_float2(pow2(y.x), pow2(y.y));
                    add = f2add(add, p);
                    u[e] = pack2(p.x, p.y, T());
                }
                tmem_put32(tP + c / 2, u);
                tmem_put_wait();
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bP + 16 * x + c / 8);
            }
            l += add.x + add.y;
        }
        if (n > 0 && ok) ok = mbar_wait_tight(bPV + 8 * x, (n - 1) & 1, a.err, kErrPagedWait);
        ok = __all_sync(0xffffffffu, ok);
        fence_after_sync();
        const float inv = paged_inverse(l);
        const int64_t part = (tq * a.n_heads + head) * a.splits + sp;
        if (a.splits > 1 && live && sp == 0) a.part_n[tq * a.n_heads + head] = n_pieces;
        if (n_pieces > 1 && live && ok) a.part_ml[part] = make_float2(n > 0 ? m * sc : -INFINITY, l);
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
            float o[32];
            if (n > 0 && ok) {
                tmem_get32(tO + c, o);
                tmem_get_wait();
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
            }
            if (!live || !ok) continue;
            if (n_pieces > 1) {
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    if (c + e < D)
                        *reinterpret_cast<float4 *>(a.part_o + part * D + c + e) =
                            make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else {
                T *out = (T *)a.out + tq * a.out_stride + (int64_t)head * D + c;
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    if (c + e < D)
                        *reinterpret_cast<uint4 *>(out + e) =
                            make_uint4(pack2(o[e] * inv, o[e + 1] * inv, T()),
                                       pack2(o[e + 2] * inv, o[e + 3] * inv, T()),
                                       pack2(o[e + 4] * inv, o[e + 5] * inv, T()),
                                       pack2(o[e + 6] * inv, o[e + 7] * inv, T()));
            }
        }
        fence_before_sync();
        asm volatile("bar.sync 0;" ::: "memory");
    }
}

// Joins the pieces of the chunk kernel, a warp per (token, head), in the order
// of the pieces. Rows that one block finished have n = 1 and are left.
template <typename T>
__global__ void __launch_bounds__(256) k_paged_join(PagedAttnArgs a) {
    const int lane = threadIdx.x & 31, D = a.cache.head_dim;
    const int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5), tok = row / a.n_heads;
    if (tok >= min((int64_t)a.cu_new[a.n_seqs], a.n_tokens)) return;
    const int n = min(a.part_n[row], a.splits);
    if (n <= 1) return;
    const int64_t part = row * a.splits;
    float top = -INFINITY;
    for (int s = lane; s < n; s += 32) top = fmaxf(top, a.part_ml[part + s].x);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float ref = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const float2 ml = a.part_ml[part + s];
        const float f = pow2(ml.x - ref);
        l += f * ml.y;
        if (lane * 4 < D) {
            const float4 o = *(reinterpret_cast<const float4 *>(a.part_o + (part + s) * D) + lane);
            acc.x += f * o.x, acc.y += f * o.y, acc.z += f * o.z, acc.w += f * o.w;
        }
    }
    const float inv = paged_inverse(l);
    if (lane * 4 < D)
        *reinterpret_cast<uint2 *>((T *)a.out + tok * a.out_stride + (row - tok * a.n_heads) * D + lane * 4) =
            make_uint2(pack2(acc.x * inv, acc.y * inv, T()), pack2(acc.z * inv, acc.w * inv, T()));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> g_encode{nullptr};

cudaError_t tensor_map_encoder(PFN_cuTensorMapEncodeTiled_v12000 *out) {
    *out = g_encode.load(std::memory_order_acquire);
    if (*out) return cudaSuccess;
    cudaDriverEntryPointQueryResult q;
    void *fn = nullptr;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q);
    if (e != cudaSuccess) return e;
    if (q != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
    *out = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    g_encode.store(*out, std::memory_order_release);
    return cudaSuccess;
}

bool paged_strides_mappable(const PagedCacheView &c) {
    const int64_t most = (int64_t)1 << 39;
    return c.token_stride > 0 && c.token_stride < most && c.head_stride > 0 && c.head_stride < most &&
           c.page_stride > 0 && c.page_stride < most;
}

static CUtensorMapDataType map_type(int bf16) {
    return bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

cudaError_t paged_cache_maps(const PagedCacheView &c, int keys, CUtensorMap *k, CUtensorMap *v) {
    PFN_cuTensorMapEncodeTiled_v12000 encode;
    const cudaError_t e = tensor_map_encoder(&encode);
    if (e != cudaSuccess) return e;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.n_kv_heads,
                                (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.token_stride * 2, (cuuint64_t)c.head_stride * 2,
                                   (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(c.page_size < keys ? c.page_size : keys), 1, 1};
    const cuuint32_t step[4] = {1, 1, 1, 1};
    for (int i = 0; i < 2; ++i)
        if (encode(i ? v : k, map_type(c.bf16), 4, i ? c.v : c.k, dims, strides, box, step,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    return cudaSuccess;
}

cudaError_t paged_q_map(const PagedAttnArgs &a, int heads, int tokens, CUtensorMap *m) {
    PFN_cuTensorMapEncodeTiled_v12000 encode;
    const cudaError_t e = tensor_map_encoder(&encode);
    if (e != cudaSuccess) return e;
    const cuuint64_t dims[3] = {(cuuint64_t)a.cache.head_dim, (cuuint64_t)a.n_heads, (cuuint64_t)a.n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)a.cache.head_dim * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens};
    const cuuint32_t step[3] = {1, 1, 1};
    return encode(m, map_type(a.cache.bf16), 3, (void *)a.q, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

// Swizzled tiles are made of blocks of 8 rows: a step's 128 keys are whole
// pages of 8, 16, 32, 64 or 128 tokens, or lie in one page of a multiple of
// 128.
bool paged_chunk_serves(const PagedCacheView &c, int n_heads) {
    const bool page = c.page_size >= 8 && (kTile % c.page_size == 0 || c.page_size % kTile == 0);
    return page && n_heads / c.n_kv_heads <= kTile && paged_strides_mappable(c);
}

int paged_chunk_unit(int group) { return 2 * (kTile / group) * group; }

template <typename T, int DP>
static cudaError_t launch_chunk(const PagedAttnArgs &a, cudaStream_t st) {
    static std::atomic<bool> attr[64];
    cudaError_t e = dynamic_smem_once(k_paged_attn_chunk<T, DP>, ChunkCfg<DP>::SMEM, attr);
    if (e != cudaSuccess) return e;
    const int group = a.n_heads / a.cache.n_kv_heads, tile_tok = kTile / group;
    CUtensorMap q, k, v;
    e = paged_q_map(a, group, tile_tok, &q);
    if (e == cudaSuccess) e = paged_cache_maps(a.cache, kTile, &k, &v);
    if (e != cudaSuccess) return e;
    const int64_t tiles = a.n_tokens / (2 * tile_tok) + a.n_seqs;
    const dim3 grid((unsigned)tiles, (unsigned)a.cache.n_kv_heads, (unsigned)a.splits);
    k_paged_attn_chunk<T, DP><<<grid, kThreads, ChunkCfg<DP>::SMEM, st>>>(a, q, k, v);
    e = cudaGetLastError();
    if (e != cudaSuccess || a.splits == 1) return e;
    const int64_t rows = a.n_tokens * a.n_heads;
    k_paged_join<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(a);
    return cudaGetLastError();
}

cudaError_t paged_chunk_attn(const PagedAttnArgs &a, cudaStream_t st) {
    if (a.cache.head_dim <= 64)
        return a.cache.bf16 ? launch_chunk<__nv_bfloat16, 64>(a, st) : launch_chunk<__half, 64>(a, st);
    return a.cache.bf16 ? launch_chunk<__nv_bfloat16, 128>(a, st) : launch_chunk<__half, 128>(a, st);
}

}  // namespace kk
