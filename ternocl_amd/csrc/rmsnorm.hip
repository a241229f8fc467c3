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
// exact there (bf16 ones some 45 binary orders apart: off by 2^-53), and a code is the one that
// the formula gives also where a quotient lies next to a half (fp32 is off by up to 2^-15 of a step
// there).  gfx950 runs a 64-bit FMA at the rate of an fp32 one.
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
    int m0;  // a launch's first row
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

// Rows of any length: a workgroup a row, which is read twice, a wave 128 elements at a time (a
// scale group), 2 bytes a lane.  Only for rows past 32768: 512 x 53248 bf16 codes 144 us where the
// bytes take 17 at the rate of a large copy, with residual and norm 428 where they take 40.
constexpr int kAnyWaves = 4;
constexpr int kShort = 256;  // threads of a workgroup of short rows
template <bool BF16, bool NORM> __global__ void __launch_bounds__(64 * kAnyWaves) k_rows_any(const NormArgs a) {
    __shared__ RowStat red[kAnyWaves];
    const int m = a.m0 + blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6, K = a.K;
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

__device__ __forceinline__ double max_abs(double m, double t) { return fmax(m, __builtin_fabs(t)); }
__device__ __forceinline__ float max_abs(float m, float t) { return fmaxf(m, __builtin_fabsf(t)); }

// Sums and maxima over each LANES lanes (8, 16, 32 or the wave), by lane moves.
template <int M> __device__ __forceinline__ double lane_xor64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(lane_xor<M>(__uint_as_float((uint32_t)u), lane));
    const uint32_t hi = __float_as_uint(lane_xor<M>(__uint_as_float((uint32_t)(u >> 32)), lane));
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
template <int LANES> __device__ __forceinline__ void lanes_stat(double &ss, double &top, int lane) {
    auto step = [&](auto m) __attribute__((always_inline)) {
        ss += lane_xor64<decltype(m)::value>(ss, lane);
        top = fmax(top, lane_xor64<decltype(m)::value>(top, lane));
    };
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 4>{});
    if constexpr (LANES > 8) step(std::integral_constant<int, 8>{});
    if constexpr (LANES > 16) step(std::integral_constant<int, 16>{});
    if constexpr (LANES > 32) step(std::integral_constant<int, 32>{});
}

// Eight codes.  1.5 2^52 (2^23) added rounds a product to a whole number and leaves it, in two's
// complement, in the sum's low bits.  F is float where t is exact in it (a row of 16-bit values
// without a norm: half the registers, 2047 x 14336 25.0 -> 20.5 us): its products are within 2^-15
// of the quotient, so those closer than 2^-14 to a half, and what leaves its range, are done
// again in 64 bits.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}
template <class F> __device__ __forceinline__ void row_codes(const F t[8], double inv, double top, uint32_t q[2]) {
    constexpr bool D = sizeof(F) == 8;
    const F magic = D ? (F)0x1.8p52 : (F)0x1.8p23, tie = D ? (F)kTie : (F)(0.5 - 0x1p-14), f = (F)inv;
    uint32_t c[8];
    bool close = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const F p = t[j] * f, s = p + magic, d = p - (s - magic);
        if constexpr (D) c[j] = (uint32_t)__builtin_bit_cast(uint64_t, s);
        else c[j] = __builtin_bit_cast(uint32_t, s);
        close |= !((d < 0 ? -d : d) <= tie);  // (NaN too)
    }
    if (close)
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = (uint32_t)row_code((double)t[j], inv, top);
    q[0] = low_bytes(c[0], c[1], c[2], c[3]);
    q[1] = low_bytes(c[4], c[5], c[6], c[7]);
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

template <bool BF16> __device__ __forceinline__ float half_of(const u32x4_t &v, int j) {
    return dt2f<BF16>(j & 1 ? v[j >> 1] >> 16 : v[j >> 1] & 0xffffu);
}

// Vectors of n <= 8 elements from p on; AL: 8, on a multiple of the vector's bytes.  gfx950 loads
// and stores 16 bytes at any address.
typedef u32x4_t __attribute__((aligned(2))) u32x4_any_t;
typedef u32x2_t __attribute__((aligned(1))) u32x2_any_t;
template <bool AL> __device__ __forceinline__ u32x4_t load8(const uint16_t *p, int n) {
    if constexpr (AL) return *(const u32x4_t *)p;
    if (n == 8) return *(const u32x4_any_t *)p;
    u32x4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 7; ++j)
        if (j < n) v[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
    return v;
}
template <bool AL> __device__ __forceinline__ void store8(uint16_t *p, const u32x4_t &v, int n) {
    if constexpr (AL) {
        *(u32x4_t *)p = v;
    } else if (n == 8) {
        *(u32x4_any_t *)p = v;
    } else {
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < n) p[j] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
    }
}
template <bool AL> __device__ __forceinline__ void store8(int8_t *p, const u32x2_t &v, int n) {
    if constexpr (AL) {
        *(u32x2_t *)p = v;
    } else if (n == 8) {
        *(u32x2_any_t *)p = v;
    } else {
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < n) p[j] = (int8_t)(v[j >> 2] >> (8 * (j & 3)));
    }
}

// n <= 8 weights from element k on (the others 0).
template <bool AL> __device__ __forceinline__ void weights_of(const NormArgs &a, int k, int n, float w[8]) {
    if (a.wtype == TERNOCL_FP32) {
        const float *p = (const float *)a.W + k;
        if (AL) {
            const float4 u = *(const float4 *)p, v = *(const float4 *)(p + 4);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = j < n ? p[j] : 0.0f;
        }
    } else {
        const u32x4_t v = load8<AL>((const uint16_t *)a.W + k, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = a.wtype == TERNOCL_BF16 ? half_of<true>(v, j) : half_of<false>(v, j);
    }
}

// Rows of up to 32768 elements, each read once: a workgroup a row, up to C vectors of 8 elements
// a thread; or (C = 1) L < 64 lanes a row.  AL: whole vectors on 16 bytes (codes: 8).
template <bool BF16, bool NORM, bool AL, int C, int L = 64>
__global__ void __launch_bounds__(L < 64 ? kShort : 1024) k_rows_vec(const NormArgs a, double invk) {
    __shared__ double red[16][2];
    __shared__ uint32_t redbad[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = a.m0 + (L < 64 ? blockIdx.x * (kShort / L) + threadIdx.x / L : blockIdx.x), tid = L < 64 ? threadIdx.x % L : threadIdx.x;
    const int nt = blockDim.x, nw = nt >> 6, vecs = (a.K + 7) >> 3;
    auto len = [&](int v) __attribute__((always_inline)) { return AL ? 8 : min(8, a.K - 8 * v); };
    if (L < 64 && m >= a.M) return;  // (a row's lanes leave together, and moves stay among them)
    const uint16_t *x = a.X + (size_t)m * a.ldx, *r = NORM && a.R ? a.R + (size_t)m * a.ldr : nullptr;
    u32x4_t xv[C], rv[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int v = tid + i * nt;
        if (v < vecs) {
            xv[i] = load8<AL>(x + 8 * v, len(v));
            if (r) rv[i] = load8<AL>(r + 8 * v, len(v));
        }
    }
    typedef typename std::conditional<NORM, double, float>::type F;
    F t[C][8], bad = 0, ftop = 0;
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int v = tid + i * nt;
        if (v < vecs) {
            float w[8];
            if (NORM && a.W) weights_of<AL>(a, 8 * v, len(v), w);
            u32x4_t hv;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                F h = half_of<BF16>(xv[i], j);
                if (r) h += (F)half_of<BF16>(rv[i], j);
                if (NORM && a.H) {
                    const uint32_t y = f2dt<BF16>((float)h);
                    if (j & 1) hv[j >> 1] |= y << 16;
                    else hv[j >> 1] = y;
                }
                if (NORM) ss = __builtin_fma(h, h, ss);
                t[i][j] = NORM && a.W ? h * ((F)w[j] + (F)a.woff) : h;
                ftop = max_abs(ftop, t[i][j]);
                bad += t[i][j] * (F)0;
            }
            if (NORM && a.H) store8<AL>(a.H + (size_t)m * a.K + 8 * v, hv, len(v));
        }
    }
    double top = ftop;
    const uint64_t odd = __ballot(bad != 0);  // (0 or NaN)
    bool nan = L < 64 ? (odd >> (lane & ~(L - 1)) & ((1ull << (L & 63)) - 1)) != 0 : odd != 0;
    lanes_stat<L>(ss, top, lane);
    if (L == 64 && nw > 1) {
        if (lane == 0) {
            red[wave][0] = ss;
            red[wave][1] = top;
            redbad[wave] = nan;
        }
        __syncthreads();
        const int l = min(lane & 15, nw - 1);
        const bool real = (lane & 15) < nw;
        ss = real ? red[l][0] : 0.0;
        top = red[l][1];
        nan = __ballot(redbad[l] != 0) != 0;
        lanes_stat<16>(ss, top, lane);
    }
    const double rs = NORM ? 1.0 / __builtin_sqrt(ss * invk + (double)a.eps) : 1.0;
    const double inv = !nan && top > 0.0 ? 127.0 / top : 0.0;
    if (a.quant == 1 && tid == 0) ((float *)a.SQ)[m] = nan ? __builtin_nanf("") : (float)(top * rs * (1.0 / 127.0));
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int v = tid + i * nt;
        if (v >= vecs) break;
        u32x4_t y;
        if (NORM && (a.Y || a.quant == 2)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = f2dt<BF16>((float)(t[i][2 * j] * rs)) | (f2dt<BF16>((float)(t[i][2 * j + 1] * rs)) << 16);
            if (a.Y) store8<AL>(a.Y + (size_t)m * a.K + 8 * v, y, len(v));
        }
        u32x2_t q = {0, 0};
        if (a.quant == 1) {
            if (!nan) {
                uint32_t c[2];
                row_codes<F>(t[i], inv, top, c);
                q = u32x2_t{c[0], c[1]};
            }
        } else if (NORM && a.quant == 2) {
            float mx = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(half_of<BF16>(y, j)));
            mx = fmaxf(mx, lane_xor<1>(mx, lane));
            mx = fmaxf(mx, lane_xor<2>(mx, lane));
            mx = fmaxf(mx, lane_xor<4>(mx, lane));
            mx = fmaxf(mx, lane_xor<8>(mx, lane));
            const uint32_t sh = f2dt<BF16>(127.0f / fmaxf(mx, FLT_EPSILON));
            const float sc = dt2f<BF16>(sh);
            if ((lane & 15) == 0) ((uint16_t *)a.SQ)[(size_t)(v >> 4) * ((a.M + 31) & ~31) + m] = (uint16_t)sh;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = half_of<BF16>(y, j) * sc;  // (exact)
                const int c = p == p ? (int)fminf(fmaxf(__builtin_rintf(p), -128.0f), 127.0f) : 0;
                q[j >> 2] |= (uint32_t)(uint8_t)c << (8 * (j & 3));
            }
        }
        if (a.quant) store8<AL>(a.Q + (size_t)m * a.K + 8 * v, q, len(v));
    }
}

// Rows a.m0 .. a.m0 + rows - 1.
template <bool NORM> ternocl_status rows_launch(int dtype, const NormArgs &a, int rows, hipStream_t st) {
    const bool bf = dtype == TERNOCL_BF16;
    if (a.K > 32768) {
        if (bf) hipLaunchKernelGGL((k_rows_any<true, NORM>), dim3(rows), dim3(64 * kAnyWaves), 0, st, a);
        else hipLaunchKernelGGL((k_rows_any<false, NORM>), dim3(rows), dim3(64 * kAnyWaves), 0, st, a);
        return check_launch();
    }
    const uintptr_t low = (uintptr_t)a.X | (uintptr_t)a.R | (uintptr_t)a.W | (uintptr_t)a.H | (uintptr_t)a.Y | (uintptr_t)(2 * a.K) |
                          (2 * (uintptr_t)a.Q) | (uintptr_t)(a.M > 1 ? 2 * (a.ldx | (a.R ? a.ldr : 0)) : 0);
    const bool al = (low & 15) == 0;
    const int vecs = (a.K + 7) / 8;
    auto pick = [&](auto f) {
        if (bf) al ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
        else al ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
    };
    if (vecs <= 32) {
        auto go = [&](auto l) {
            constexpr int L = decltype(l)::value;
            const dim3 g((rows + kShort / L - 1) / (kShort / L));
            pick([&](auto b, auto w) {
                hipLaunchKernelGGL((k_rows_vec<decltype(b)::value, NORM, decltype(w)::value, 1, L>), g, dim3(kShort), 0, st, a, 1.0 / a.K);
            });
        };
        if (vecs <= 8) go(std::integral_constant<int, 8>{});
        else if (vecs <= 16) go(std::integral_constant<int, 16>{});
        else go(std::integral_constant<int, 32>{});
        return check_launch();
    }
    // Vectors a thread: one where a call is as long as a row's latency (one row of 4096: 3.5 us,
    // with two 3.9), more where workgroups queue (8192 x 5120 rows of codes: one 86.6, two
    // 63.8, four 64.9; without a norm, where a thread holds half as much, 2047 x 14336: two
    // 22.7, four 20.5).  By rows, one / two, codes after a norm: of 4096 at 256 rows 4.9 / 5.1, 384
    // 6.1 / 5.8, 512 6.9 / 6.6, 768 9.8 / 9.3; of 1024 at 512 4.3 / 4.5, 1024 4.6 / 4.8, 1536 6.0 / 5.7.  Without
    // a norm 4096 at 256 3.6 / 3.8, 512 4.8 / 4.2; 14336, two / four: 512 9.8 / 10.1, 1024 14.2 / 14.1, 2048
    // 22.2 / 20.0.
    int c = vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : 4;
    if (a.M > 512) c = vecs > 2048 || (!NORM && vecs > 512) ? 4 : 2;
    const int nt = ((vecs + c - 1) / c + 63) / 64 * 64;
    auto go = [&](auto n) {
        pick([&](auto b, auto w) {
            hipLaunchKernelGGL((k_rows_vec<decltype(b)::value, NORM, decltype(w)::value, decltype(n)::value>), dim3(rows), dim3(nt), 0, st,
                               a, 1.0 / a.K);
        });
    };
    if (c == 1) go(std::integral_constant<int, 1>{});
    else if (c == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
    return check_launch();
}

// (a launch holds 2^32 threads: 2^21 rows of up to 1024 at a time)
template <bool NORM> ternocl_status rows_run(int dtype, NormArgs a, hipStream_t st) {
    constexpr int step = 1 << 21;
    for (a.m0 = 0; a.m0 < a.M; a.m0 += step) {
        const ternocl_status s = rows_launch<NORM>(dtype, a, a.M - a.m0 < step ? a.M - a.m0 : step, st);
        if (s != TERNOCL_OK) return s;
    }
    return TERNOCL_OK;
}

}  // namespace

ternocl_status rmsnorm_run(int dtype, const void *X, long ldx, const void *R, long ldr, int wtype, const void *W, float woff,
                           float eps, void *H, void *Y, int quant, int8_t *Q, void *SQ, int M, int K, hipStream_t st) {
    return rows_run<true>(dtype, {(const uint16_t *)X, (const uint16_t *)R, ldx, ldr, wtype, W, woff, eps, (uint16_t *)H,
                                  (uint16_t *)Y, quant, Q, SQ, M, K, 0}, st);
}

ternocl_status quant_rows_run(int dtype, const void *X, long ldx, int8_t *Q, float *SQ, int M, int K, hipStream_t st) {
    return rows_run<false>(dtype, {(const uint16_t *)X, nullptr, ldx, 0, 0, nullptr, 0.0f, 0.0f, nullptr, nullptr, 1, Q, SQ, M, K, 0}, st);
}

}  // namespace tcl
