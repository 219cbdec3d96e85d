// Products of a few rows with a 4-bit weight matrix (sm_100a):
//   out[r][n] = sum_k x[r][k] (q[n][k] - 8) s[n][k / group] (+ bias[n])
// q in [0, 15], two to a byte (element 2 i in the low nibble of byte i), s
// half, x and out of one type. Sums are 32-bit; the products are exact:
// q - 8 fits the 16-bit types, and a 32-bit x is split into three bfloat16
// parts (8 + 8 + 8 significant bits, its whole range). Bfloat16 weights are
// unpacked as (q - 8) 2^-11 and the scales multiplied by 2^11, so that a
// group's sum of up to 128 x 8 times the largest x stays finite until its
// scale is applied. (The last of 24 bits of an x below 2^-115 then fall below
// the smallest float.)
//
// The weights are read once, n_out n_in / 2 bytes, but their unpacking bounds
// it: 7 integer operations for 8 weights and its latencies. A warp takes 16
// outputs as the M side of mma.sync.m16n8k16 and 8 or 16 rows of x as its N
// side, so a row more costs no further work on the weights. The order of k
// within a product is free as long as both sides agree: a lane takes 8
// consecutive k (one 32-bit word of weights, whose nibbles i and i + 4 are
// the two halves of one masked word), so nothing is moved between lanes. The
// products of one group are summed by the tensor cores, then scaled once per
// output in 32 bits.
//
// The weights come as tensor copies of 256 k (128 bytes, swizzled, so that the
// words of 8 rows lie in different banks) into a ring of each warp, one lane
// issuing. x is brought to shared memory a chunk of k at a time by the whole
// block, split and ordered as the lanes read it, 16 bytes each without a bank
// twice. The 8 warps of a block lie along the outputs (WR) and along k; the
// latter are joined in shared memory, in the order of the warps.
//
// Measured on B200, 8192 -> 24576, groups of 128, bfloat16: one row 35 us (3.0
// TB/s), 8 rows 43 us, 16 rows 66 us, and 391 us for 128, each 16 rows reading
// and unpacking the weights again. 25, 29 and 35 instructions a word of weights,
// the integer pipe half busy; the bytes alone are 16 us.
#include "../../include/kokopop_b200.h"
#include "kk_common.cuh"
#include "kk_kernels.h"
#include "kk_ptx.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <type_traits>

namespace kk {

namespace {

constexpr int kQ4Warps = 8;

// mma16 from a sum of 0.
template <typename T>
__device__ __forceinline__ void mma16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    c[0] = c[1] = c[2] = c[3] = 0.f;
    mma16<T>(c, a, b0, b1);
}

// The 8 weights of a word as 4 pairs (nibbles i and i + 4) of values q - 8.
// The nibbles are placed in the mantissa of 128 (bfloat16) or 1024 (half),
// whose last place is 1, and 128 + 8 or 1024 + 8 is subtracted by a fused
// multiply-add; half has room for them 4 places up too, as 1024 + 16 q. All of
// it is exact.
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));  // (w & mask) | bits
    return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c, __half) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c, __nv_bfloat16) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&v)[4], __half t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t u = w >> (8 * i);
        v[2 * i] = fma2(mask_or(u, 0x000f000fu, 0x64006400u), 0x3c003c00u, 0xe408e408u, t);      // 1, -1032
        v[2 * i + 1] = fma2(mask_or(u, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u, t);  // 1 / 16, -72
    }
}
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&v)[4], __nv_bfloat16 t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = fma2(mask_or(w >> (4 * i), 0x000f000fu, 0x43004300u), 0x3a003a00u, 0xbd88bd88u, t);  // 2^-11 (1, -136)
}

// a weight over its unpacked value
template <typename M>
constexpr float kUnpacked = 2048.f;
template <>
constexpr float kUnpacked<__half> = 1.f;

// The type multiplied for x of type T, and the parts of one value.
template <typename T>
struct XType {
    using M = T;
    static constexpr int PARTS = 1;
};
template <>
struct XType<float> {
    using M = __nv_bfloat16;
    static constexpr int PARTS = 3;
};

// 8 consecutive x as 16-bit parts in the lane's order of k: words (0, 4),
// (1, 5), (2, 6), (3, 7).
template <typename T>
__device__ __forceinline__ void load_x(const T *p, uint32_t (&b)[1][4]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    b[0][0] = __byte_perm(u.x, u.z, 0x5410);
    b[0][1] = __byte_perm(u.x, u.z, 0x7632);
    b[0][2] = __byte_perm(u.y, u.w, 0x5410);
    b[0][3] = __byte_perm(u.y, u.w, 0x7632);
}
__device__ __forceinline__ void load_x(const float *p, uint32_t (&b)[3][4]) {
    const float4 lo = *reinterpret_cast<const float4 *>(p), hi = *reinterpret_cast<const float4 *>(p + 4);
    float v[8] = {lo.x, hi.x, lo.y, hi.y, lo.z, hi.z, lo.w, hi.w};
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // the upper 16 bits: rounded towards zero, so nothing overflows
            b[s][i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float &x = v[2 * i + e];
                x = fabsf(x) == INFINITY ? 0.f : x - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
            }
        }
}

__device__ __forceinline__ void put(float v, float *p) { *p = v; }
__device__ __forceinline__ void put(float v, __half *p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(float v, __nv_bfloat16 *p) { *p = __float2bfloat16_rn(v); }

}  // namespace

// One block of 256 k of 16 outputs: c = the sum over a group of PG x 32 k,
// then acc += scale c. at: the lane's word of row gid in the first 16 bytes
// of the block, w8 its row; x: the lane's 16 bytes of the first 32 k for each
// tile of rows, x_group and x_part bytes further for the next 32 k and the
// next part (0 where the lane's row does not exist: it then stays on 16 bytes
// of zeros); fa: the scales of outputs gid and gid + 8, times kUnpacked.
template <typename M, int NB, int PARTS, int PG>
__device__ __forceinline__ void q4_block(uint32_t at, uint32_t w8, const uint32_t (&x0)[NB],
                                         const uint32_t (&x_group)[NB], const uint32_t (&x_part)[NB],
                                         const float (&fa)[2][8 / PG], float (&acc)[NB][4]) {
    float c[NB][4];
    uint32_t x[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) x[b] = x0[b];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        uint32_t v[NB][PARTS][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(v[b][p][0]), "=r"(v[b][p][1]), "=r"(v[b][p][2]), "=r"(v[b][p][3])
                             : "r"(x[b] + p * x_part[b])
                             : "memory");
            x[b] += x_group[b];
        }
        const uint32_t w = at + ((g * 16) ^ w8);
        uint32_t ua, ub, fu[4], fv[4];
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(ua) : "r"(w) : "memory");
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(ub) : "r"(w + 1024) : "memory");
        unpack(ua, fu, M());
        unpack(ub, fv, M());
        const uint32_t lo[4] = {fu[0], fv[0], fu[1], fv[1]}, hi[4] = {fu[2], fv[2], fu[3], fv[3]};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int p = PARTS - 1; p >= 0; --p) {
                if (g % PG == 0 && p == PARTS - 1)
                    mma16_first<M>(c[b], lo, v[b][p][0], v[b][p][1]);
                else
                    mma16<M>(c[b], lo, v[b][p][0], v[b][p][1]);
                mma16<M>(c[b], hi, v[b][p][2], v[b][p][3]);
            }
        if (g % PG == PG - 1)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[b][e] = fmaf(fa[e >> 1][g / PG], c[b][e], acc[b][e]);
    }
}

// WR warps along the outputs, 16 each, the others along k; NB tiles of 8 rows
// of x.
template <typename T, int NB, int WR>
struct Q4Cfg {
    static constexpr int WK = kQ4Warps / WR;
    static constexpr int ROWS = 16 * WR;
    static constexpr int STAGES = 3;
    static constexpr int TILE = 16 * 128;                              // a block of 256 k
    static constexpr int CTAS = NB == 1 ? 3 : 2;                       // of an SM
    static constexpr int X_BYTES = (NB == 1 ? 24 : 48) * 1024;         // of x at a time
    static constexpr int SMEM = kQ4Warps * STAGES * TILE + X_BYTES + 1024 /*align*/;
};

template <typename T, int NB, int WR>
__global__ void __launch_bounds__(kQ4Warps * 32, (Q4Cfg<T, NB, WR>::CTAS))
    k_q4_matvec(const __grid_constant__ Q4MatvecArgs a, const __grid_constant__ CUtensorMap map_w) {
    using C = Q4Cfg<T, NB, WR>;
    using M = typename XType<T>::M;
    constexpr int PARTS = XType<T>::PARTS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *sX = smem + kQ4Warps * C::STAGES * C::TILE;
    __shared__ __align__(8) uint64_t bar_s[kQ4Warps][C::STAGES];
    __shared__ __align__(16) uint4 zero_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const int wr = warp / C::WK, wk = warp % C::WK;
    const int n0 = blockIdx.x * C::ROWS + wr * 16;
    const int64_t r0 = (int64_t)blockIdx.y * (8 * NB);
    const int shift = 31 - __clz(a.group), groups = a.n_in >> shift, blocks = (a.n_in + 255) / 256;
    const int rows = (int)min(a.n_rows - r0, (int64_t)(8 * NB));
    const uint32_t ring = smem_u32(smem + warp * C::STAGES * C::TILE), bars = smem_u32(bar_s[warp]);
    if (lane == 0) {
        for (int i = 0; i < C::STAGES; ++i) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // the warp's first blocks of 256 k: wk, wk + WK, ...
        for (int i = 0; i < C::STAGES - 1; ++i)
            if (wk + i * C::WK < blocks) {
                mbar_expect_tx(bars + 8 * i, C::TILE);
                tma_load_2d(ring + i * C::TILE, &map_w, bars + 8 * i, (wk + i * C::WK) * 128, n0);
            }
    }
    __syncwarp();

    // scales of this lane's outputs; outputs past the last are not written
    const __half *sa = a.scales + (int64_t)min(n0 + gid, a.n_out - 1) * groups;
    const __half *sb = a.scales + (int64_t)min(n0 + 8 + gid, a.n_out - 1) * groups;
    // the lane's word in row gid of a block; its 16-byte chunk is XORed by the row
    const uint32_t at0 = ring + gid * 128 + tig * 4;
    float acc[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0.f;

    // x in shared memory: [group of 32 k][part][row][8 k of lane tig]; 16
    // bytes of zeros for the rows that do not exist
    const uint32_t part = rows * 64, step = part * PARTS;
    // a warp brings a row, or a power of two of the warps share it
    const int row_bits = min(32 - __clz(rows - 1), 3), xk = (warp >> row_bits) * 32 + lane,
              xk_step = kQ4Warps * 32 >> row_bits;
    const int chunk = min(C::X_BYTES / (int)step / 8 * 256, blocks * 256);
    if (tid == 0) zero_s = make_uint4(0u, 0u, 0u, 0u);
    uint32_t x_at[NB], x_group[NB], x_part[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int r = 8 * b + gid;
        x_at[b] = r < rows ? smem_u32(sX) + r * 64 + tig * 16 : smem_u32(&zero_s);
        x_group[b] = r < rows ? step : 0;
        x_part[b] = r < rows ? part : 0;
    }

    bool ok = true;
    int blk = wk;
    uint32_t st = 0, phase = 0;  // stage and phase of the warp's block
    for (int c0 = 0; c0 < a.n_in; c0 += chunk) {
        const int c1 = min(c0 + chunk, a.n_in);
        // x of [c0, c1), 8 values of a row at a time and 0 up to the next
        // multiple of 256: the weights there read as 0, which stands for -8
        if (c0 > 0) __syncthreads();
        const int per_row = (c1 - c0 + 255) / 256 * 32;
        constexpr int BATCH = PARTS == 1 ? 6 : 3;  // loads in flight of a thread
        for (int xr = warp & ((1 << row_bits) - 1); xr < rows; xr += 8) {
            const T *x = (const T *)a.x + (r0 + xr) * a.x_stride + c0;
            for (int k8 = xk; k8 < per_row; k8 += BATCH * xk_step) {
                uint32_t v[BATCH][PARTS][4];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int k = (k8 + j * xk_step) * 8;
                    if (c0 + k < c1) {
                        load_x(x + k, v[j]);
                    } else {
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) v[j][p][0] = v[j][p][1] = v[j][p][2] = v[j][p][3] = 0u;
                    }
                }
                // xk_step is a multiple of 4: k8 % 4 stays
                uint8_t *to = sX + (k8 >> 2) * step + xr * 64 + (k8 & 3) * 16;
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    if (k8 + j * xk_step < per_row)
#pragma unroll
                        for (int p = 0; p < PARTS; ++p)
                            *reinterpret_cast<uint4 *>(to + j * (xk_step >> 2) * step + p * part) =
                                make_uint4(v[j][p][0], v[j][p][1], v[j][p][2], v[j][p][3]);
            }
        }
        __syncthreads();
        for (; ok && blk * 256 < c1; blk += C::WK) {
            const uint32_t bar = bars + 8 * st, at = at0 + st * C::TILE;
            const int next = blk + (C::STAGES - 1) * C::WK;
            if (lane == 0 && next < blocks) {
                const uint32_t to = st == 0 ? C::STAGES - 1 : st - 1;
                mbar_expect_tx(bars + 8 * to, C::TILE);
                tma_load_2d(ring + to * C::TILE, &map_w, bars + 8 * to, next * 128, n0);
            }
            uint32_t x[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) x[b] = x_at[b] + ((blk * 256 - c0) >> 5) * x_group[b];
            auto run = [&](auto pg) {
                constexpr int PG = decltype(pg)::value, NS = 8 / PG;
                // the block's scales: loaded before its weights are waited for
                float fa[2][NS];
                const int s0 = blk * NS;
#pragma unroll
                for (int g = 0; g < NS; ++g) {
                    fa[0][g] = s0 + g < groups ? kUnpacked<M> * __half2float(__ldg(sa + s0 + g)) : 0.f;
                    fa[1][g] = s0 + g < groups ? kUnpacked<M> * __half2float(__ldg(sb + s0 + g)) : 0.f;
                }
                ok = __all_sync(0xffffffffu, mbar_wait_tight(bar, phase, a.err, kErrQ4Wait));
                if (ok) q4_block<M, NB, PARTS, PG>(at, gid * 16, x, x_group, x_part, fa, acc);
            };
            if (shift == 5)
                run(std::integral_constant<int, 1>());
            else if (shift == 6)
                run(std::integral_constant<int, 2>());
            else
                run(std::integral_constant<int, 4>());
            if (!ok) break;
            __syncwarp();  // the stage is read before its next copy is issued
            st = st + 1 == C::STAGES ? (phase ^= 1, 0) : st + 1;
        }
    }
    if (!ok)  // copies in flight land before the block ends
        for (int j = 0; j < C::STAGES && blk + j * C::WK < blocks; ++j) {
            mbar_wait(bars + 8 * st, phase, a.err, kErrQ4Wait, TC_DRAIN_NS);
            st = st + 1 == C::STAGES ? (phase ^= 1, 0) : st + 1;
        }
    __syncthreads();
    // join: [wk][output][row]
    float *join = reinterpret_cast<float *>(smem);
    constexpr int COLS = 8 * NB, LEN = C::ROWS * COLS;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            join[wk * LEN + (wr * 16 + 8 * (e >> 1) + gid) * COLS + 8 * b + 2 * tig + (e & 1)] = acc[b][e];
    __syncthreads();
    for (int it = tid; it < LEN; it += kQ4Warps * 32) {
        const int n = blockIdx.x * C::ROWS + it % C::ROWS, r = it / C::ROWS;
        if (n < a.n_out && r < rows) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < C::WK; ++w) v += join[w * LEN + it % C::ROWS * COLS + r];
            if (a.bias) v += a.bias[n];
            put(v, (T *)a.out + (r0 + r) * a.out_stride + n);
        }
    }
}

// the weights as bytes, boxes of 128 bytes x 16 outputs, swizzled; outside reads as 0
static cudaError_t weight_map(const Q4MatvecArgs &a, CUtensorMap *m) {
    PFN_cuTensorMapEncodeTiled_v12000 encode;
    const cudaError_t e = tensor_map_encoder(&encode);
    if (e != cudaSuccess) return e;
    const cuuint64_t dims[2] = {(cuuint64_t)a.n_in / 2, (cuuint64_t)a.n_out};
    const cuuint64_t strides[1] = {(cuuint64_t)a.n_in / 2};
    const cuuint32_t box[2] = {128, 16}, step[2] = {1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)a.w, dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

template <typename T, int NB, int WR>
static cudaError_t launch_q4(const Q4MatvecArgs &a, cudaStream_t st) {
    using C = Q4Cfg<T, NB, WR>;
    static std::atomic<bool> attr[64];
    cudaError_t e = dynamic_smem_once(k_q4_matvec<T, NB, WR>, C::SMEM, attr);
    if (e != cudaSuccess) return e;
    CUtensorMap m;
    e = weight_map(a, &m);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)((a.n_out + C::ROWS - 1) / C::ROWS), (unsigned)((a.n_rows + 8 * NB - 1) / (8 * NB)));
    k_q4_matvec<T, NB, WR><<<grid, kQ4Warps * 32, C::SMEM, st>>>(a, m);
    return cudaGetLastError();
}

template <typename T, int NB>
static cudaError_t launch_q4_rows(const Q4MatvecArgs &a, cudaStream_t st) {
    // Warps along the outputs: more of them share x in shared memory, fewer
    // make more blocks. 8 rows of 8192, with 1, 2, 4, 8: 24576 outputs 98, 70,
    // 51, 60 us; 8192 outputs (4 rows) 30, 22, 25, 36 us.
    if (a.n_out >= 16384) return launch_q4<T, NB, 4>(a, st);
    if (a.n_out >= 32 * 148) return launch_q4<T, NB, 2>(a, st);
    return launch_q4<T, NB, 1>(a, st);
}

template <typename T>
static cudaError_t launch_q4_of(const Q4MatvecArgs &a, cudaStream_t st) {
    return a.n_rows <= 8 ? launch_q4_rows<T, 1>(a, st) : launch_q4_rows<T, 2>(a, st);
}

cudaError_t q4_matvec(const Q4MatvecArgs &a, cudaStream_t st) {
    if (a.dtype == KK_DTYPE_F32) return launch_q4_of<float>(a, st);
    if (a.dtype == KK_DTYPE_F16) return launch_q4_of<__half>(a, st);
    return launch_q4_of<__nv_bfloat16>(a, st);
}

}  // namespace kk
