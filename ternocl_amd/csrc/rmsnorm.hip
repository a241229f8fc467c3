// rmsnorm.hip -- root-mean-square norm of the residual stream with the residual's addition
// and an output in 8 bits (ternocl_rmsnorm), and the 8-bit rows alone (ternocl_quant_rows),
// for gfx950:
//
//   h = x + r,  t = h (woff + w),  s = 1 / sqrt(mean_k h^2 + eps),  n = t s
//   H = DT(h),  Y = DT(n)
//   rows:   SQ[m] = max_k |n| / 127,  q = rne(127 t / max_k |t|)   (= rne(n / SQ): s cancels)
//   groups: quant_a of Y: SQ[g, m] = DT(127 / max(absmax, FLT_EPSILON)), q = sat(rne(Y SQ))
//
// Everything before a rounding to DT or to a code is 64-bit: x + r of two 16-bit values is
// exact there, and a code is the one that the formula gives also where a quotient lies next
// to a half (fp32 is off by up to 2^-16 of a step there).  gfx950 runs a 64-bit FMA at the
// rate of an fp32 one.
#include "common.hpp"

#include <cfloat>

namespace tcl {
namespace {

struct NormArgs {
    const uint16_t *X, *R;
    long ldx, ldr;
    int wtype;
    const void *W;
    float woff, eps;
    uint16_t *H, *Y;
    int quant;  // 0 none, 1 rows, 2 groups
    int8_t *Q;
    void *SQ;
    int M, K;
};

constexpr double kTie = 0.5 - 0x1p-30;  // past this a product with 127 / top may be on the wrong side of a half

__device__ __forceinline__ int row_code(double t, double inv, double top) {
    const double p = t * inv;
    double q = __builtin_rint(p);
    if (__builtin_fabs(p - q) > kTie) q = __builtin_rint(127.0 * t / top);
    return (int)q;
}

__device__ __forceinline__ double weight_of(const NormArgs &a, int k) {
    if (!a.W) return 1.0;
    const float w = a.wtype == TERNOCL_FP32   ? ((const float *)a.W)[k]
                    : a.wtype == TERNOCL_BF16 ? dt2f<true>(((const uint16_t *)a.W)[k])
                                              : dt2f<false>(((const uint16_t *)a.W)[k]);
    return (double)w + (double)a.woff;
}

// Sums and maxima over the workgroup's waves.
struct RowStat {
    double ss, top, bad;  // sum of h^2, max |t| of the finite t, NaN where a t is not finite
};
__device__ __forceinline__ RowStat wave_stat(RowStat s) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        s.ss += __shfl_xor(s.ss, o);
        s.top = fmax(s.top, __shfl_xor(s.top, o));
        s.bad += __shfl_xor(s.bad, o);
    }
    return s;
}

// Rows of any length, pitch and alignment: a workgroup a row, which is read twice, a wave 128
// elements at a time (a scale group).
constexpr int kAnyWaves = 4;
template <bool BF16, bool NORM> __global__ void __launch_bounds__(64 * kAnyWaves) k_rows_any(const NormArgs a) {
    __shared__ RowStat red[kAnyWaves];
    const int m = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6, K = a.K;
    const uint16_t *x = a.X + (size_t)m * a.ldx, *r = a.R ? a.R + (size_t)m * a.ldr : nullptr;
    auto h_of = [&](int k) __attribute__((always_inline)) {
        const double h = dt2f<BF16>(x[k]);
        return NORM && r ? h + (double)dt2f<BF16>(r[k]) : h;
    };
    RowStat s = {0.0, 0.0, 0.0};
    for (long b = 128 * w; b < K; b += 128 * kAnyWaves)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long k = b + lane + 64 * i;
            if (k < K) {
                const double h = h_of(k), t = NORM ? h * weight_of(a, k) : h;
                if (NORM) s.ss = __builtin_fma(h, h, s.ss);
                s.top = fmax(s.top, __builtin_fabs(t));
                s.bad = __builtin_fma(t, 0.0, s.bad);
            }
        }
    s = wave_stat(s);
    if (lane == 0) red[w] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int i = 1; i < kAnyWaves; ++i) {
        s.ss += red[i].ss;
        s.top = fmax(s.top, red[i].top);
        s.bad += red[i].bad;
    }
    const bool bad = s.bad != 0.0;  // (0 or NaN)
    const double rs = NORM ? 1.0 / __builtin_sqrt(s.ss / K + (double)a.eps) : 1.0;
    const double inv = !bad && s.top > 0.0 ? 127.0 / s.top : 0.0;
    if (a.quant == 1 && threadIdx.x == 0) ((float *)a.SQ)[m] = bad ? __builtin_nanf("") : (float)(s.top * rs / 127.0);
    for (long b = 128 * w; b < K; b += 128 * kAnyWaves) {
        uint32_t y[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long k = b + lane + 64 * i;
            if (k < K) {
                const double h = h_of(k), t = NORM ? h * weight_of(a, k) : h;
                if (NORM) {
                    if (a.H) a.H[(size_t)m * K + k] = (uint16_t)f2dt<BF16>((float)h);
                    y[i] = f2dt<BF16>((float)(t * rs));
                    if (a.Y) a.Y[(size_t)m * K + k] = (uint16_t)y[i];
                }
                if (a.quant == 1) a.Q[(size_t)m * K + k] = bad ? (int8_t)0 : (int8_t)row_code(t, inv, s.top);
            }
        }
        if (NORM && a.quant == 2) {  // (K a multiple of 128)
            const float v[2] = {dt2f<BF16>(y[0]), dt2f<BF16>(y[1])};
            float mx = fmaxf(fabsf(v[0]), fabsf(v[1]));
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            const uint32_t sh = f2dt<BF16>(127.0f / fmaxf(mx, FLT_EPSILON));
            const float sc = dt2f<BF16>(sh);
            if (lane == 0) ((uint16_t *)a.SQ)[(size_t)(b >> 7) * ((a.M + 31) & ~31) + m] = (uint16_t)sh;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float p = v[i] * sc;  // (exact)
                a.Q[(size_t)m * K + b + lane + 64 * i] = p == p ? (int8_t)fminf(fmaxf(__builtin_rintf(p), -128.0f), 127.0f) : (int8_t)0;
            }
        }
    }
}

template <bool NORM> ternocl_status rows_run(int dtype, const NormArgs &a, hipStream_t st) {
    if (dtype == TERNOCL_BF16) hipLaunchKernelGGL((k_rows_any<true, NORM>), dim3(a.M), dim3(64 * kAnyWaves), 0, st, a);
    else hipLaunchKernelGGL((k_rows_any<false, NORM>), dim3(a.M), dim3(64 * kAnyWaves), 0, st, a);
    return check_launch();
}

}  // namespace

ternocl_status rmsnorm_run(int dtype, const void *X, long ldx, const void *R, long ldr, int wtype, const void *W, float woff,
                           float eps, void *H, void *Y, int quant, int8_t *Q, void *SQ, int M, int K, hipStream_t st) {
    return rows_run<true>(dtype, {(const uint16_t *)X, (const uint16_t *)R, ldx, ldr, wtype, W, woff, eps, (uint16_t *)H,
                                  (uint16_t *)Y, quant, Q, SQ, M, K}, st);
}

ternocl_status quant_rows_run(int dtype, const void *X, long ldx, int8_t *Q, float *SQ, int M, int K, hipStream_t st) {
    return rows_run<false>(dtype, {(const uint16_t *)X, nullptr, ldx, 0, 0, nullptr, 0.0f, 0.0f, nullptr, nullptr, 1, Q, SQ, M, K}, st);
}

}  // namespace tcl
