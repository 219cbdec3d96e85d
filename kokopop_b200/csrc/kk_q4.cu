// Products of a few rows with a 4-bit weight matrix (sm_100a):
//   out[r][n] = sum_k x[r][k] (q[n][k] - 8) s[n][k / group] (+ bias[n])
// q in [0, 15], two to a byte (element 2 i in the low nibble of byte i), s
// half, x and out of one type. Sums are 32-bit; the products are exact:
// q - 8 fits the 16-bit types, and a 32-bit x is split into three bfloat16
// parts (8 + 8 + 8 significant bits, its whole range).
//
// The weights are read once, n_out n_in / 2 bytes, and bound it. A warp takes
// 16 outputs as the M side of mma.sync.m16n8k16 and up to 8 rows of x as its
// N side, so a row more costs no further work on the weights. The order of k
// within a product is free as long as both sides agree: a lane takes 8
// consecutive k (one 32-bit word of weights, whose nibbles i and i + 4 are
// the two halves of one masked word), so nothing is moved between lanes. The
// products of one group are summed by the tensor cores, then scaled once per
// output in 32 bits. The warps of a block share the k axis and are joined in
// shared memory, in the order of the warps.
#include "../../include/kokopop_b200.h"
#include "kk_common.cuh"
#include "kk_kernels.h"

namespace kk {

namespace {

constexpr int kQ4Warps = 8;

template <typename T>
__device__ __forceinline__ void mma_q4(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_q4<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_q4<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                      uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// nibbles i and i + 4 of w (i = 0 after the shift) as a pair of values q - 8:
// placed in the mantissa of 1024 (half) or 128 (bfloat16), whose last place
// is 1, and 1024 + 8 or 128 + 8 subtracted, exactly
__device__ __forceinline__ uint32_t pair_of(uint32_t w, __half) {
    const uint32_t u = (w & 0x000f000fu) | 0x64006400u, b = 0x64086408u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t pair_of(uint32_t w, __nv_bfloat16) {
    const uint32_t u = (w & 0x000f000fu) | 0x43004300u, b = 0x43084308u;
    const __nv_bfloat162 r =
        __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&u), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

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

template <typename T>
__global__ void __launch_bounds__(kQ4Warps * 32) k_q4_matvec(Q4MatvecArgs a) {
    using M = typename XType<T>::M;
    constexpr int PARTS = XType<T>::PARTS;
    __shared__ float join[kQ4Warps][16][8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * 16;
    const int64_t r0 = (int64_t)blockIdx.y * 8;
    const int64_t kb = a.n_in / 2;
    const int groups = a.n_in / a.group;
    // outputs past the last read the last row's weights and are not written
    const int na = min(n0 + gid, a.n_out - 1), nb = min(n0 + gid + 8, a.n_out - 1);
    const uint8_t *wa = a.w + na * kb + tig * 4, *wb = a.w + nb * kb + tig * 4;
    const __half *sa = a.scales + (int64_t)na * groups, *sb = a.scales + (int64_t)nb * groups;
    const bool has_x = r0 + gid < a.n_rows;
    const T *x = (const T *)a.x + (has_x ? r0 + gid : 0) * a.x_stride + tig * 8;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int steps = a.group / 32;
    for (int g = warp; g < groups; g += kQ4Warps) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < steps; ++s) {
            const int64_t k = (int64_t)g * a.group + s * 32;
            const uint32_t ua = *reinterpret_cast<const uint32_t *>(wa + k / 2);
            const uint32_t ub = *reinterpret_cast<const uint32_t *>(wb + k / 2);
            uint32_t b[PARTS][4];
            if (has_x) {
                load_x(x + k, b);
            } else {
#pragma unroll
                for (int p = 0; p < PARTS; ++p) b[p][0] = b[p][1] = b[p][2] = b[p][3] = 0u;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t f[4] = {pair_of(ua >> (8 * h), M()), pair_of(ub >> (8 * h), M()),
                                       pair_of(ua >> (8 * h + 4), M()), pair_of(ub >> (8 * h + 4), M())};
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p) mma_q4<M>(c, f, b[p][2 * h], b[p][2 * h + 1]);
            }
        }
        const float s0 = __half2float(sa[g]), s1 = __half2float(sb[g]);
        acc[0] = fmaf(s0, c[0], acc[0]);
        acc[1] = fmaf(s0, c[1], acc[1]);
        acc[2] = fmaf(s1, c[2], acc[2]);
        acc[3] = fmaf(s1, c[3], acc[3]);
    }
    join[warp][gid][tig * 2] = acc[0];
    join[warp][gid][tig * 2 + 1] = acc[1];
    join[warp][gid + 8][tig * 2] = acc[2];
    join[warp][gid + 8][tig * 2 + 1] = acc[3];
    __syncthreads();
    if (tid < 128) {
        const int n = n0 + (tid & 15), r = tid >> 4;
        if (n < a.n_out && r0 + r < a.n_rows) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kQ4Warps; ++w) v += join[w][tid & 15][r];
            if (a.bias) v += a.bias[n];
            put(v, (T *)a.out + (r0 + r) * a.out_stride + n);
        }
    }
}

cudaError_t q4_matvec(const Q4MatvecArgs &a, cudaStream_t st) {
    const dim3 grid((unsigned)((a.n_out + 15) / 16), (unsigned)((a.n_rows + 7) / 8));
    if (a.dtype == KK_DTYPE_F32)
        k_q4_matvec<float><<<grid, kQ4Warps * 32, 0, st>>>(a);
    else if (a.dtype == KK_DTYPE_F16)
        k_q4_matvec<__half><<<grid, kQ4Warps * 32, 0, st>>>(a);
    else
        k_q4_matvec<__nv_bfloat16><<<grid, kQ4Warps * 32, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace kk
