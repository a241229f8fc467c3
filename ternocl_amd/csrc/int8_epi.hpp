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

typedef uint32_t i8_u32x2_t __attribute__((ext_vector_type(2)));
typedef float i8_f32x4_t __attribute__((ext_vector_type(4)));

// The epilogue of outputs (m, n .. n + 3), n % 4 == 0, in two parts, so that a lane's loads are in
// flight together, or while the products run: what it reads, as it is stored, then the output.
struct I8Col {
    i8_f32x4_t sb, bias;  // (bias: fp32, or DT pairs in the first two)
};
struct I8Row {
    float sa;
    i8_u32x2_t other;
};
__device__ __forceinline__ I8Col i8_col(const I8Args &a, int n) {
    I8Col c;
    c.sb = *(const i8_f32x4_t *)(a.SB + n);
    if (postop_needs_bias(a.postop)) {
        if (a.out_f32) {
            c.bias = *(const i8_f32x4_t *)((const float *)a.Bias + n);
        } else {
            const i8_u32x2_t t = *(const i8_u32x2_t *)((const uint16_t *)a.Bias + n);
            c.bias = i8_f32x4_t{__uint_as_float(t[0]), __uint_as_float(t[1]), 0.0f, 0.0f};
        }
    }
    return c;
}
__device__ __forceinline__ I8Row i8_row(const I8Args &a, int m, int n) {
    I8Row r;
    r.sa = a.SA[m];
    if (postop_needs_other(a.postop)) r.other = *(const i8_u32x2_t *)(a.Other + (size_t)m * a.N + n);
    return r;
}
template <bool BF16, int P, bool F32>
__device__ __forceinline__ void i8_out(const I8Args &a, int m, int n, i32x4_t s, const I8Col &c, const I8Row &r) {
    auto four = [](uint32_t x, uint32_t y) __attribute__((always_inline)) {
        return i8_f32x4_t{dt2f<BF16>(x & 0xffffu), dt2f<BF16>(x >> 16), dt2f<BF16>(y & 0xffffu), dt2f<BF16>(y >> 16)};
    };
    i8_f32x4_t o = {}, b = {}, v;
    if constexpr (postop_needs_other(P)) o = four(r.other[0], r.other[1]);
    if constexpr (postop_needs_bias(P)) b = F32 ? c.bias : four(__float_as_uint(c.bias[0]), __float_as_uint(c.bias[1]));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = epi_apply_c<P>(i8_scaled(s[i], c.sb[i], r.sa), o[i], b[i]);
    const size_t at = (size_t)m * a.N + n;
    if constexpr (F32) *(i8_f32x4_t *)((float *)a.C + at) = v;
    else *(i8_u32x2_t *)((uint16_t *)a.C + at) = i8_u32x2_t{f2dt<BF16>(v[0]) | (f2dt<BF16>(v[1]) << 16), f2dt<BF16>(v[2]) | (f2dt<BF16>(v[3]) << 16)};
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
