// int4_plain.hip -- C = A x (q - Z) S on 4-bit weights (ternocl_int4_gemm) for
// operands that are not 16-byte aligned, which the matrix-core engines load 16 bytes at
// a time: fp32 FMAs, a lane per column, kPlainRows rows of A per pass over the weights.
//
//   C[m,n] = ct(epi(sum_g S[g,n] (sum_{k in g} A[m,k] q[k,n] - Z[g,n] sum_{k in g} A[m,k])))
#include "common.hpp"

namespace tcl {
namespace {

constexpr int kPlainRows = 8, kPlainWaves = 4;

// Workgroup: 64 columns, kPlainRows rows; its waves take every kPlainWaves-th group and
// their sums are added in wave order.
template <bool BF16>
__global__ void __launch_bounds__(64 * kPlainWaves)
k_int4_plain(const uint16_t *__restrict__ A, const uint4 *__restrict__ B, const uint16_t *__restrict__ S,
             const uint16_t *__restrict__ Z, void *__restrict__ C, const uint16_t *__restrict__ Other,
             const void *__restrict__ Bias, int M, int N, int K, int group, int postop, int out_f32) {
    __shared__ float red[kPlainWaves][kPlainRows][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = blockIdx.x * 64 + lane, nc = min(n, N - 1), m0 = blockIdx.y * kPlainRows;
    float acc[kPlainRows] = {};
    for (int g = w; g < K / group; g += kPlainWaves) {
        float p[kPlainRows] = {}, sa[kPlainRows] = {};
        for (int kb = g * group / 32; kb < (g + 1) * group / 32; ++kb) {
            const uint4 b = B[(size_t)kb * N + nc];
            const uint32_t x[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const int nib = (r % 8) / 2 + 4 * (r % 2);
                const float q = (float)((int)(x[r / 8] << (28 - 4 * nib)) >> 28);
#pragma unroll
                for (int i = 0; i < kPlainRows; ++i) {
                    const float v = dt2f<BF16>(A[(size_t)min(m0 + i, M - 1) * K + 32 * kb + r]);
                    p[i] = __builtin_fmaf(v, q, p[i]);
                    sa[i] += v;
                }
            }
        }
        const float s = dt2f<BF16>(S[(size_t)g * N + nc]);
        const float z = Z ? dt2f<BF16>(Z[(size_t)g * N + nc]) : 0.0f;
#pragma unroll
        for (int i = 0; i < kPlainRows; ++i) acc[i] = __builtin_fmaf(s, Z ? __builtin_fmaf(-z, sa[i], p[i]) : p[i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < kPlainRows; ++i) red[w][i][lane] = acc[i];
    __syncthreads();
    if (n >= N) return;
    epi_dispatch(postop, out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
        for (int i = w; i < kPlainRows; i += kPlainWaves) {
            if (m0 + i >= M) break;
            float v = red[0][i][lane];
#pragma unroll
            for (int k = 1; k < kPlainWaves; ++k) v += red[k][i][lane];
            epi_store1_c<BF16, decltype(P_)::value, decltype(F_)::value>(C, Other, Bias, N, m0 + i, n, v);
        }
    });
}

}  // namespace

// (grid.y holds 65535 row tiles: more rows run in further launches)
ternocl_status int4_plain_run(int dtype, const void *A, const uint32_t *B, const void *S, const void *Z, void *C,
                              const void *Other, const void *Bias, int M, int N, int K, int group, int postop,
                              int out_f32, hipStream_t st) {
    const int step = 65535 * kPlainRows;
    for (int m = 0; m < M; m += step) {
        const int rows = M - m < step ? M - m : step;
        const dim3 g((N + 63) / 64, (rows + kPlainRows - 1) / kPlainRows);
        auto go = [&](auto bf) {
            hipLaunchKernelGGL((k_int4_plain<decltype(bf)::value>), g, dim3(64 * kPlainWaves), 0, st,
                               (const uint16_t *)A + (size_t)m * K, (const uint4 *)B, (const uint16_t *)S,
                               (const uint16_t *)Z, (uint8_t *)C + (size_t)m * N * (out_f32 ? 4 : 2),
                               Other ? (const uint16_t *)Other + (size_t)m * N : nullptr, Bias, rows, N, K, group, postop,
                               out_f32);
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
