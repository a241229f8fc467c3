// int4_gemv.hip -- decode GEMV (M <= 8) on 4-bit weights with group scales for gfx950
// (ternocl_int4_gemm):
//
//   C[m,n] = ct(epi(sum_g S[g,n] * sum_{k in g} A[m,k] (q[k,n] - Z[g,n])))
//
// The call streams the weights once; what it can lose beside that is the work per
// weight.  Both operands go to the int8 matrix cores, whose sums are exact:
//
// * Weights: a nibble in the upper half of a byte is the int8 value 16 q, sign
//   included, so a word of 8 codes becomes two operand dwords by w & 0xf0f0f0f0 and
//   (w << 4) & 0xf0f0f0f0: three operations for 8 weights.
// * Activations: per row and scale group, t = round(a 2^(21 - e)) with e the exponent of
//   the group's largest |a|, |t| <= 2^22, in three balanced base-256 digits t = 65536 d2 +
//   256 d1 + d0.  Each digit is a matrix row of its own (rows 4 m + 0 .. 2), so one
//   instruction multiplies all digits of four activation rows with 16 columns.  fp16
//   values down to 2^-11 and bf16 values down to 2^-14 of their group's largest are t
//   exactly; smaller ones are within 2^-22 of that largest.
// * Per group and column: three int32 sums to one fp32 (exact digits, two roundings),
//   times a sixteenth of the activations' power of two, and S.  Zero points take Z times
//   the group's sum of activations off.  A group with an infinity or NaN gets NaN for its
//   power of two.
//
// Work split: a workgroup stages the activations' digits in LDS once and walks 16-column
// strips; its waves take parts of K, in 128-row steps (one 16-byte load a lane: 16
// columns x 4 blocks of 32 rows), with kDepth steps of weights in flight across strips.
// The waves' sums meet in LDS, added in wave order by one wave while the others go on:
// the same bits on every run, one barrier a strip.
//
// What bounds it is the weight stream: M = 4 K = 4096 N = 151680 fp16, 320 MB, 60.8 us a call,
// 5.3 TB/s (a large copy 4.9); M = 1 K = 5120 N = 34816 bf16, groups of 64 with zero points, 100
// MB, 22.3 us, 4.5 TB/s.  A small call is launch and first loads: M = 1 K = N = 4096 4.9 us
// for 8.7 MB.
#include "common.hpp"

#include <algorithm>

namespace tcl {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t g4_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kDepth = 4;       // steps of weights in flight per wave
constexpr int kMaxWaves = 16;
constexpr int kMaxLds = 160 << 10;

// LDS layout: digits [steps][2][3 M][64] bytes, then (scale, sum) floats [groups][MP],
// then the waves' sums [2][waves][64 RS] floats.
struct G4Lds {
    int digits, scales, sums, red, total;
};
__host__ __device__ inline G4Lds g4_lds(int M, int K, int group, bool zero, int waves) {
    const int mp = M > 4 ? 8 : 4;
    G4Lds l;
    l.digits = 0;
    l.scales = K / 128 * 2 * 3 * M * 64;
    l.sums = l.scales + K / group * mp * 4;
    l.red = l.sums + (zero ? K / group * mp * 4 : 0);
    l.total = l.red + 2 * waves * 64 * (mp / 4) * 4;
    return l;
}

struct G4Args {
    const uint16_t *A;
    const uint32_t *B;
    const uint16_t *S, *Z;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K, postop, out_f32;
};

// The workgroup's LDS writes are done and every wave is here; loads in flight stay so.
__device__ __forceinline__ void g4_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A wave's part of a group sum over the lanes of one group (8 activations a lane)
template <int G, class Op> __device__ __forceinline__ float g4_reduce(float v, int lane, Op op) {
    v = op(v, lane_xor<1>(v, lane));
    v = op(v, lane_xor<2>(v, lane));
    if constexpr (G >= 64) v = op(v, lane_xor<4>(v, lane));
    if constexpr (G >= 128) v = op(v, lane_xor<8>(v, lane));
    return v;
}

// byte j of a, b, c, d in a dword, each with its top bit flipped (offset -> balanced digit)
template <int j> __device__ __forceinline__ uint32_t g4_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0000u | ((4 + j) << 8) | j);
    const uint32_t hi = __builtin_amdgcn_perm(d, c, 0x00000c0cu | ((uint32_t)(4 + j) << 24) | (j << 16));
    return (lo | hi) ^ 0x80808080u;
}

// Variants of 64 registers a lane: two workgroups on a CU, their staging and tails apart (M =
// 1 K = 5120 N = 34816 20.0 -> 18.6 us; the others would spill).
__host__ __device__ constexpr bool g4_two(int rs, int group, bool zero) { return rs == 1 && group == 128 && !zero; }

// Eight activations, task i (i >= tasks: nothing is stored): the lanes of its group are
// adjacent, and all of a wave's are here.
template <bool BF16, int G, bool ZP>
__device__ __forceinline__ void g4_stage8(const G4Args &a, uint8_t *lds, const G4Lds &l, const uint4 &raw, int i, int tasks) {
    const int units = a.K / 8, mp = a.M > 4 ? 8 : 4, lane = threadIdx.x & 63, R = 3 * a.M;
    const int ic = min(i, tasks - 1), m = ic / units, u = ic - m * units;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = dt2f<BF16>(w[j] & 0xffffu);
        f[2 * j + 1] = dt2f<BF16>(w[j] >> 16);
    }
    uint32_t mb = 0;  // the largest |a| by its bits: a NaN is above infinity
#pragma unroll
    for (int j = 0; j < 8; ++j) mb = max(mb, __float_as_uint(f[j]) & 0x7fffffffu);
    mb = __float_as_uint(g4_reduce<G>(__uint_as_float(mb), lane, [](float x, float y) {
        return __uint_as_float(max(__float_as_uint(x), __float_as_uint(y)));
    }));
    const bool bad = mb >= 0x7f800000u;
    const int e = max((int)(mb >> 23), 15) - 127;  // (2^-112 at least: bf16's multiples of 2^-133 are t exactly there)
    uint32_t t[8];
    int sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int q = bad ? 0 : (int)__builtin_rintf(__builtin_ldexpf(f[j], 21 - e));
        sum += q;
        t[j] = (uint32_t)q + 0x808080u;
    }
    if constexpr (ZP)
        sum = __float_as_int(g4_reduce<G>(__int_as_float(sum), lane, [](float x, float y) {
            return __int_as_float(__float_as_int(x) + __float_as_int(y));
        }));
    if (i >= tasks) return;
    const int step = u >> 4, b = (u >> 2) & 3, wd = u & 3;
    const int q = G == 128 ? b : wd, h = (G == 128 ? wd : b) >> 1, half = (G == 128 ? wd : b) & 1;
    uint8_t *p = lds + l.digits + ((step * 2 + h) * R + 3 * m) * 64 + q * 16 + half * 8;
    // odd nibbles' rows 2, 6, 3, 7, then even nibbles' rows 0, 4, 1, 5 (the order of g4_mfma)
    *(uint2 *)(p) = make_uint2(g4_bytes<2>(t[2], t[6], t[3], t[7]), g4_bytes<2>(t[0], t[4], t[1], t[5]));
    *(uint2 *)(p + 64) = make_uint2(g4_bytes<1>(t[2], t[6], t[3], t[7]), g4_bytes<1>(t[0], t[4], t[1], t[5]));
    *(uint2 *)(p + 128) = make_uint2(g4_bytes<0>(t[2], t[6], t[3], t[7]), g4_bytes<0>(t[0], t[4], t[1], t[5]));
    if ((8 * u) % G == 0) {
        const int g = 8 * u / G;
        // (a sixteenth for the weights' 16: nothing on the way to a sum is larger than it is)
        ((float *)(lds + l.scales))[g * mp + m] = bad ? __builtin_nanf("") : __builtin_ldexpf(1.0f, e - 25);
        if constexpr (ZP)
            ((float *)(lds + l.sums))[g * mp + m] = bad ? __builtin_nanf("") : __builtin_ldexpf((float)sum, e - 21);
    }
}

// Stages the digits, powers of two (and sums) of all M rows.  Task i: activations 8 u ..
// 8 u + 7 of a row; 16 tasks a 128-row step, so G / 8 adjacent lanes hold a group.
template <bool BF16, int RS, int G, bool ZP>
__device__ __forceinline__ void g4_stage(const G4Args &a, uint8_t *lds, const G4Lds &l) {
    const int tasks = a.M * (a.K / 8), mp = a.M > 4 ? 8 : 4;
    constexpr int kPass = g4_two(RS, G, ZP) ? 1 : 4;  // passes whose loads are in flight together (registers)
    const int T = blockDim.x;
    for (int i0 = threadIdx.x; i0 - (int)threadIdx.x < tasks; i0 += kPass * T) {
        uint4 raw[kPass];
#pragma unroll
        for (int k = 0; k < kPass; ++k) raw[k] = *(const uint4 *)(a.A + 8 * (size_t)min(i0 + k * T, tasks - 1));
#pragma unroll
        for (int k = 0; k < kPass; ++k)
            if (i0 - (int)threadIdx.x + k * T < tasks) g4_stage8<BF16, G, ZP>(a, lds, l, raw[k], i0 + k * T, tasks);
    }
    // rows M .. mp - 1: nothing
    for (int i = threadIdx.x; i < a.K / G * mp; i += blockDim.x)
        if (i % mp >= a.M) {
            ((float *)(lds + l.scales))[i] = 0.0f;
            if constexpr (ZP) ((float *)(lds + l.sums))[i] = 0.0f;
        }
}

// One step's weights of a lane: block q of its column; and the scales (zeros) of the step's
// groups, value v of its column (S of group v, then Z) in lane q = v: two or four values a
// load, handed round by row moves.
template <bool BF16, int G, bool ZP> struct G4Slot {
    static constexpr int GS = 128 / G, NV = ZP ? 2 * GS : GS, NL = NV > 4 ? 2 : 1;
    g4_u32x4 w;
    uint16_t x[NL];
    // this lane's first value of step 0 and column 0
    static __device__ __forceinline__ void base(const G4Args &a, int q, const uint16_t *(&p)[NL]) {
        if constexpr (NV == 1) p[0] = a.S;
        else if constexpr (NL == 2) p[0] = a.S + (size_t)q * a.N, p[1] = a.Z + (size_t)q * a.N;
        else if constexpr (!ZP) p[0] = a.S + (size_t)(q % GS) * a.N;
        else p[0] = ((q / GS) & 1 ? a.Z : a.S) + (size_t)(q % GS) * a.N;
    }
    __device__ __forceinline__ void load(const G4Args &a, const uint16_t *const (&p)[NL], int step, int n, int q) {
        w = __builtin_nontemporal_load((const g4_u32x4 *)(a.B + ((size_t)(4 * step + q) * a.N + n) * 4));
#pragma unroll
        for (int i = 0; i < NL; ++i) x[i] = p[i][(size_t)(step * GS) * a.N + n];
    }
    // every value of the lane's column: S, then Z, by group
    __device__ __forceinline__ void values(float (&v)[NV]) const {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t f = __float_as_uint(dt2f<BF16>(x[i]));
            if constexpr (NV == 1) {
                v[0] = __uint_as_float(f);
            } else {
                const auto r = __builtin_amdgcn_permlane16_swap(f, f, false, false);  // even, odd rows' values
                if constexpr (NV == 2) {
                    v[0] = __uint_as_float(r[0]);
                    v[1] = __uint_as_float(r[1]);
                } else {
                    const auto e = __builtin_amdgcn_permlane32_swap(r[0], r[0], false, false);  // rows 0, 2
                    const auto o = __builtin_amdgcn_permlane32_swap(r[1], r[1], false, false);  // rows 1, 3
                    v[4 * i] = __uint_as_float(e[0]);
                    v[4 * i + 1] = __uint_as_float(o[0]);
                    v[4 * i + 2] = __uint_as_float(e[1]);
                    v[4 * i + 3] = __uint_as_float(o[1]);
                }
            }
        }
    }
};

// RS: sets of four activation rows.
template <bool BF16, int RS, int G, bool ZP>
__global__ void __launch_bounds__(64 * kMaxWaves, g4_two(RS, G, ZP) ? 8 : 4) k_int4_gemv(const G4Args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int GS = 128 / G, MP = 4 * RS;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const int W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int steps = a.K / 128, strips = a.N / 16, R = 3 * a.M;
    const G4Lds l = g4_lds(a.M, a.K, G, ZP, W);
    const int s0 = steps * w / W, s1 = steps * (w + 1) / W;  // (W <= steps: at least one)
    // XCD x (workgroups x, x + 8, ...) takes runs of eight strips in a row: four strips share a
    // 128-byte line of S and Z, which every XCD that reads of it fetches whole (strips dealt
    // round, M = 1 K = 5120 N = 34816: groups of 64 with zero points 26.0 -> 23.9 us, groups of
    // 32 33.4 -> 29.1)
    const int j8 = blockIdx.x >> 3, first = ((j8 >> 3) * 8 + (blockIdx.x & 7)) * 8 + (j8 & 7);
    if (first >= strips) return;  // (whole workgroup)
    // the loads run kDepth steps ahead of the products, across strips
    int ls = first, lt = s0;
    typedef G4Slot<BF16, G, ZP> Slot;
    Slot slot[kDepth];
    const uint16_t *sp[Slot::NL];
    Slot::base(a, q, sp);
    auto fetch = [&](int d) __attribute__((always_inline)) {
        if (ls >= strips) return;  // (uniform)
        slot[d].load(a, sp, lt, 16 * ls + c, q);
        if (++lt == s1) {
            lt = s0;
            ls += gridDim.x;
        }
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch(d);
    g4_stage<BF16, RS, G, ZP>(a, lds, l);
    g4_barrier();

    // matrix row r = lane % 16: digit r % 4 (3: unused) of activation row r / 4
    const uint8_t *arow[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        const int m = 4 * s + (c >> 2);
        arow[s] = lds + l.digits + (m < a.M ? 3 * m + min(c & 3, 2) : 0) * 64 + q * 16;
    }
    const float *scales = (const float *)(lds + l.scales) + q, *sums = (const float *)(lds + l.sums) + q;
    float *red = (float *)(lds + l.red);
    float acc[RS] = {};
    int strip = first, t = s0, it = 0;
    auto item = [&](int d) __attribute__((always_inline)) {
        uint32_t w4[4] = {slot[d].w[0], slot[d].w[1], slot[d].w[2], slot[d].w[3]};
        float sz[Slot::NV];
        slot[d].values(sz);
        fetch(d);
        if constexpr (G < 128) {
            // lane q's block q (its words 0..3) -> word q of blocks 0..3: a 4 x 4 transpose over q
            auto r = __builtin_amdgcn_permlane32_swap(w4[0], w4[2], false, false);
            w4[0] = r[0]; w4[2] = r[1];
            r = __builtin_amdgcn_permlane32_swap(w4[1], w4[3], false, false);
            w4[1] = r[0]; w4[3] = r[1];
            r = __builtin_amdgcn_permlane16_swap(w4[0], w4[1], false, false);
            w4[0] = r[0]; w4[1] = r[1];
            r = __builtin_amdgcn_permlane16_swap(w4[2], w4[3], false, false);
            w4[2] = r[0]; w4[3] = r[1];
        }
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            b[2 * j] = w4[j] & 0xf0f0f0f0u;
            b[2 * j + 1] = (w4[j] << 4) & 0xf0f0f0f0u;
        }
#pragma unroll
        for (int s = 0; s < RS; ++s) {
            i32x4_t D[GS];
            const i32x4_t a0 = *(const i32x4_t *)(arow[s] + (size_t)(t * 2) * R * 64);
            const i32x4_t a1 = *(const i32x4_t *)(arow[s] + (size_t)(t * 2 + 1) * R * 64);
            const i32x4_t b0 = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]}, b1 = {(int)b[4], (int)b[5], (int)b[6], (int)b[7]};
            if constexpr (G == 128) {
                D[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b0, i32x4_t{}, 0, 0, 0);
                D[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b1, D[0], 0, 0, 0);
            } else if constexpr (G == 64) {
                D[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b0, i32x4_t{}, 0, 0, 0);
                D[1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b1, i32x4_t{}, 0, 0, 0);
            } else {
                auto half = [](const i32x4_t &v, int h) __attribute__((always_inline)) {
                    return (long)(uint32_t)v[2 * h] | ((long)v[2 * h + 1] << 32);
                };
                D[0] = __builtin_amdgcn_mfma_i32_16x16x32_i8(half(a0, 0), half(b0, 0), i32x4_t{}, 0, 0, 0);
                D[1] = __builtin_amdgcn_mfma_i32_16x16x32_i8(half(a0, 1), half(b0, 1), i32x4_t{}, 0, 0, 0);
                D[2] = __builtin_amdgcn_mfma_i32_16x16x32_i8(half(a1, 0), half(b1, 0), i32x4_t{}, 0, 0, 0);
                D[3] = __builtin_amdgcn_mfma_i32_16x16x32_i8(half(a1, 1), half(b1, 1), i32x4_t{}, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < GS; ++j) {
                const int g = (t * GS + j) * MP + 4 * s;
                const float f = __builtin_fmaf((float)D[j][0], 65536.0f, __builtin_fmaf((float)D[j][1], 256.0f, (float)D[j][2]));
                float v = f * scales[g];  // the group's product
                if constexpr (ZP) v = __builtin_fmaf(-sz[GS + j], sums[g], v);
                acc[s] = __builtin_fmaf(sz[j], v, acc[s]);
            }
        }
        if (++t < s1) return;
        // the strip is done: sums of the waves, in wave order, by wave it % W
        t = s0;
        float *r = red + (it & 1) * W * 64 * RS;
#pragma unroll
        for (int s = 0; s < RS; ++s) {
            r[(w * RS + s) * 64 + lane] = acc[s];
            acc[s] = 0.0f;
        }
        g4_barrier();
        if (w == it % W) {
            float v[RS];
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                v[s] = r[s * 64 + lane];
                for (int k = 1; k < W; ++k) v[s] += r[(k * RS + s) * 64 + lane];
            }
            epi_dispatch(a.postop, a.out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < RS; ++s)
                    if (4 * s + q < a.M)
                        epi_store1_c<BF16, decltype(P_)::value, decltype(F_)::value>(a.C, a.Other, a.Bias, a.N, 4 * s + q,
                                                                                    16 * strip + c, v[s]);
            });
        }
        ++it;
        strip += gridDim.x;
    };
    static_assert(kDepth == 4, "one call a slot");
    auto more = [&](int d) __attribute__((always_inline)) {
        item(d);
        return strip < strips;  // (uniform, and alike in every wave of the workgroup)
    };
    while (more(0) && more(1) && more(2) && more(3)) {
    }
}

int g4_waves(int K) { return K / 128 < kMaxWaves ? K / 128 : kMaxWaves; }

}  // namespace

// Whether the rows' digits fit a workgroup's LDS.
bool int4_gemv_supports(int M, int K, int group, bool zero) {
    return M <= 8 && (long)K * M <= 1 << 20 && g4_lds(M, K, group, zero, g4_waves(K)).total <= kMaxLds;
}

ternocl_status int4_gemv_run(int dtype, const void *A, const uint32_t *B, const void *S, const void *Z, void *C,
                             const void *Other, const void *Bias, int M, int N, int K, int group, int postop,
                             int out_f32, hipStream_t st) {
    const G4Args a = {(const uint16_t *)A, B, (const uint16_t *)S, (const uint16_t *)Z, C, (const uint16_t *)Other, Bias,
                      M, N, K, postop, out_f32};
    const int waves = g4_waves(K), lds = g4_lds(M, K, group, Z != nullptr, waves).total;
    // (whole runs of strips over the XCDs)
    const int strips = N / 16, per = g4_two(M > 4 ? 2 : 1, group, Z != nullptr) && lds <= kMaxLds / 2 ? 2 : 1;
    const int grid = std::min((strips + 63) / 64 * 64, 256 * per);
    hipError_t e = hipSuccess;
    auto go = [&](auto bf, auto rs, auto g, auto z) {
        auto *k = k_int4_gemv<decltype(bf)::value, decltype(rs)::value, decltype(g)::value, decltype(z)::value>;
        hipLaunchKernelGGL(k, dim3(grid), dim3(64 * waves), lds, st, a);
        e = hipGetLastError();
    };
    auto zero = [&](auto bf, auto rs, auto g) {
        if (Z) go(bf, rs, g, std::true_type{});
        else go(bf, rs, g, std::false_type{});
    };
    auto grp = [&](auto bf, auto rs) {
        if (group == 32) zero(bf, rs, std::integral_constant<int, 32>{});
        else if (group == 64) zero(bf, rs, std::integral_constant<int, 64>{});
        else zero(bf, rs, std::integral_constant<int, 128>{});
    };
    auto rows = [&](auto bf) {
        if (M <= 4) grp(bf, std::integral_constant<int, 1>{});
        else grp(bf, std::integral_constant<int, 2>{});
    };
    if (dtype == TERNOCL_BF16) rows(std::true_type{});
    else rows(std::false_type{});
    return launch_status(e);
}

}  // namespace tcl
