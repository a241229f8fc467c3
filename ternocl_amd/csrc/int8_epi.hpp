// int8_epi.hpp -- what the engines of ternocl_int8_gemm do to a sum of products.
#pragma once

#include "common.hpp"

namespace tcl {
struct I8Args {
    const int8_t *A;
    const float *SA;
    const int8_t *B;
    const float *SB;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K, postop, out_f32, ksn;
    int *part;      // [ksn][M][N] with ksn > 1
    uint64_t *cnt;  // two words a tile
};
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));


// The whole sum (exact in 32 bits: K below 2^17), rounded to fp32 where it passes 2^24,
// times the channel's scale, then the token's: a token's scale may be as large as its
// activations (2^120 at bf16), and the channel's has brought the sum down before it.
__device__ __forceinline__ float i8_scaled(int acc, float sb, float sa) { return ((float)acc * sb) * sa; }

// The outputs (m, n .. n + 3) of four sums; n % 4 == 0.
template <bool BF16> __device__ __forceinline__ void i8_store4(const I8Args &a, int m, int n, i32x4_t s) {
    const float4 sb = *(const float4 *)(a.SB + n);
    const float sa = a.SA[m];
    const float v[4] = {i8_scaled(s[0], sb.x, sa), i8_scaled(s[1], sb.y, sa), i8_scaled(s[2], sb.z, sa), i8_scaled(s[3], sb.w, sa)};
    epi_dispatch(a.postop, a.out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
        epi_store4_c<BF16, decltype(P_)::value, decltype(F_)::value>(a.C, a.Other, a.Bias, a.N, m, n, v);
    });
}

// Four sums to and from the workspace, past the XCD's own L2.
__device__ __forceinline__ void i8_part_store(int *p, i32x4_t s) {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
        __hip_atomic_store((uint64_t *)(p + i), (uint64_t)(uint32_t)s[i] | ((uint64_t)(uint32_t)s[i + 1] << 32), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ i32x4_t i8_part_load(const int *p) {
    i32x4_t s;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint64_t x = __hip_atomic_load((const uint64_t *)(p + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s[i] = (int)(uint32_t)x;
        s[i + 1] = (int)(uint32_t)(x >> 32);
    }
    return s;
}

}  // namespace
}  // namespace tcl
