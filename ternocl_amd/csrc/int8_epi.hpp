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

// The epilogue of outputs (m, n .. n + 3), n % 4 == 0, in two parts, so that a lane's loads are in
// flight together: what it reads, then the output.
template <bool BF16, int P, bool F32> struct I8Epi {
    typedef uint32_t U2 __attribute__((ext_vector_type(2)));
    typedef float F4 __attribute__((ext_vector_type(4)));
    const I8Args &a;
    __device__ __forceinline__ I8Epi(const I8Args &a_) : a(a_) {}
    struct Col {
        F4 sb, bias;
    };
    struct Row {
        float sa;
        U2 other;
    };
    static __device__ __forceinline__ F4 four(U2 t) {
        return F4{dt2f<BF16>(t[0] & 0xffffu), dt2f<BF16>(t[0] >> 16), dt2f<BF16>(t[1] & 0xffffu), dt2f<BF16>(t[1] >> 16)};
    }
    __device__ __forceinline__ Col col(int n) const {
        Col c;
        c.sb = *(const F4 *)(a.SB + n);
        if constexpr (postop_needs_bias(P)) c.bias = F32 ? *(const F4 *)((const float *)a.Bias + n) : four(*(const U2 *)((const uint16_t *)a.Bias + n));
        return c;
    }
    __device__ __forceinline__ Row row(int m, int n) const {
        Row r;
        r.sa = a.SA[m];
        if constexpr (postop_needs_other(P)) r.other = *(const U2 *)(a.Other + (size_t)m * a.N + n);
        return r;
    }
    __device__ __forceinline__ void store(int m, int n, i32x4_t s, const Col &c, const Row &r) const {
        F4 o = {}, b = {}, v;
        if constexpr (postop_needs_other(P)) o = four(r.other);
        if constexpr (postop_needs_bias(P)) b = c.bias;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = epi_apply_c<P>(i8_scaled(s[i], c.sb[i], r.sa), o[i], b[i]);
        const size_t at = (size_t)m * a.N + n;
        if constexpr (F32) *(F4 *)((float *)a.C + at) = v;
        else *(U2 *)((uint16_t *)a.C + at) = U2{f2dt<BF16>(v[0]) | (f2dt<BF16>(v[1]) << 16), f2dt<BF16>(v[2]) | (f2dt<BF16>(v[3]) << 16)};
    }
};

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
