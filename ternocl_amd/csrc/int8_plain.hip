// int8_plain.hip -- products of 8-bit integers with a scale for each token and channel
// (ternocl_int8_gemm) for operands that are not 16-byte aligned, which the matrix-core
// engines load 16 bytes at a time: v_dot4 on a lane per column, kPlainRows rows of A per
// pass over the weights.  bf16 with a bias off 16 bytes, plain / matrix cores: 8 x 4096 x 4096 27 / 6.1 us,
// 200 x 5120 x 5120 163 / 16.6, 1024 x 4096 x 14336 1750 / 60.
//
//   C[m,n] = ct(epi(SA[m] SB[n] sum_k A[m,k] B[k,n]))
#include "int8_epi.hpp"

namespace tcl {
namespace {

constexpr int kPlainRows = 8, kPlainWaves = 4;

// Workgroup: 64 columns, kPlainRows rows; its waves take every kPlainWaves-th block of 16
// rows of K.
template <bool BF16>
__global__ void __launch_bounds__(64 * kPlainWaves)
k_int8_plain(const int8_t *__restrict__ A, const float *__restrict__ SA, const int4 *__restrict__ B,
             const float *__restrict__ SB, void *__restrict__ C, const uint16_t *__restrict__ Other,
             const void *__restrict__ Bias, int M, int N, int K, int postop, int out_f32) {
    __shared__ int red[kPlainWaves][kPlainRows][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = blockIdx.x * 64 + lane, nc = min(n, N - 1), m0 = blockIdx.y * kPlainRows;
    int acc[kPlainRows] = {};
    for (int kb = w; kb < K / 16; kb += kPlainWaves) {
        const int4 b = B[(size_t)kb * N + nc];
#pragma unroll
        for (int i = 0; i < kPlainRows; ++i) {
            int x[4];
            __builtin_memcpy(x, A + (size_t)min(m0 + i, M - 1) * K + 16 * kb, 16);
            acc[i] = __builtin_amdgcn_sdot4(x[0], b.x, acc[i], false);
            acc[i] = __builtin_amdgcn_sdot4(x[1], b.y, acc[i], false);
            acc[i] = __builtin_amdgcn_sdot4(x[2], b.z, acc[i], false);
            acc[i] = __builtin_amdgcn_sdot4(x[3], b.w, acc[i], false);
        }
    }
#pragma unroll
    for (int i = 0; i < kPlainRows; ++i) red[w][i][lane] = acc[i];
    __syncthreads();
    if (n >= N) return;
    epi_dispatch(postop, out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
        for (int i = w; i < kPlainRows; i += kPlainWaves) {
            if (m0 + i >= M) break;
            int v = red[0][i][lane];
#pragma unroll
            for (int k = 1; k < kPlainWaves; ++k) v += red[k][i][lane];
            epi_store1_c<BF16, decltype(P_)::value, decltype(F_)::value>(C, Other, Bias, N, m0 + i, n, i8_scaled(v, SB[n], SA[m0 + i]));
        }
    });
}

}  // namespace

// (grid.y holds 65535 row tiles: more rows run in further launches)
ternocl_status int8_plain_run(int dtype, const int8_t *A, const float *SA, const int8_t *B, const float *SB, void *C,
                              const void *Other, const void *Bias, int M, int N, int K, int postop, int out_f32,
                              hipStream_t st) {
    const int step = 65535 * kPlainRows;
    for (int m = 0; m < M; m += step) {
        const int rows = M - m < step ? M - m : step;
        const dim3 g((N + 63) / 64, (rows + kPlainRows - 1) / kPlainRows);
        auto go = [&](auto bf) {
            hipLaunchKernelGGL((k_int8_plain<decltype(bf)::value>), g, dim3(64 * kPlainWaves), 0, st, A + (size_t)m * K, SA + m,
                               (const int4 *)B, SB, (uint8_t *)C + (size_t)m * N * (out_f32 ? 4 : 2),
                               Other ? (const uint16_t *)Other + (size_t)m * N : nullptr, Bias, rows, N, K, postop, out_f32);
        };
        if (dtype == TERNOCL_BF16) go(std::true_type{});
        else go(std::false_type{});
        const ternocl_status s = check_launch();
        if (s != TERNOCL_OK) return s;
        if (M - m <= step) break;
    }
    return TERNOCL_OK;
}

}  // namespace tcl
