// int4_gemm_tile.hip -- GEMM of hundreds of rows and more on 4-bit weights with group
// scales for gfx950 (ternocl_int4_gemm): the same sums as int4_gemm_kw.hip on 128 x 256
// tiles whose eight waves share the activations in LDS.
//
// A wave's 64 x 64 part: each decoded fragment feeds two row blocks and each activation
// fragment two column blocks, with group sums (part) and the tile's (acc) in 128 registers;
// two buffers of 64 rows of K and one barrier a unit; the activations two units ahead in
// registers.  M = 1024 K = 4096 N = 14336 fp16, groups of 128: 141 to 149 us a call, by box, 807 to
// 853 TFLOP/s, about 70% of a large matrix product's; its 448 tiles on 256 CUs leave 12% idle, and of a
// wave's time VALU (decode, group sums) is 31%, waits for loads and barriers 30%, for issue 32%, MFMAs
// busy 22%.  Groups of 32 at bf16 or with zero points: per 64-row unit of a wave 256 FMAs join group
// sums and offsets, 64 operations decode, for 24 MFMAs, a third of them the offsets'; VALU 34%, the two
// waits 30% and 31%, MFMAs 14% of a wave's time, with one wave a SIMD (M = 200 K = N = 5120: 45 us, 233
// TFLOP/s).
#include "gemm_kw.hpp"
#include "int4_decode.hpp"

#include <algorithm>

namespace tcl {
namespace {

constexpr int kMB = 2, kCB = 2;  // a wave: 64 rows x 64 columns
// WM x WN waves
template <int WM_, int WN_> struct TileCfg {
    static constexpr int WM = WM_, WN = WN_, THREADS = 64 * WM * WN;
    static constexpr int BM = 64 * WM, BN = 64 * WN;
    static constexpr int A_BYTES = BM * 128;                       // a 64-k unit of the rows
    static constexpr int LOADS = A_BYTES / (16 * THREADS);         // 16-byte chunks a lane
    static_assert(LOADS * 16 * THREADS == A_BYTES, "whole loads");
};

struct I4TileArgs {
    const uint16_t *A;
    const uint32_t *B;
    const uint16_t *S, *Z;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K, postop, out_f32, ksn;
    float *part;     // ksn > 1: [ksn][M][N] slice sums
    uint64_t *cnt;   // ... and the tiles' arrival counters
};

// LDS writes are done and every wave is here; global loads in flight stay so.
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <class Cfg, bool BF16, int G, bool ZP> __global__ void __launch_bounds__(Cfg::THREADS) k_int4_gemm_tile(const I4TileArgs a) {
    constexpr int MB = kMB, CB = kCB, GU = G < 64 ? 2 : 1;
    constexpr bool OFF = BF16 || ZP;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][Cfg::A_BYTES];
    const int mt = (a.M + Cfg::BM - 1) / Cfg::BM, nt = (a.N + Cfg::BN - 1) / Cfg::BN;
    int tm, tn, sl;
    {  // XCD x takes a contiguous range of the slices' tiles, column strip by column strip
        const int per = (mt * nt * a.ksn + 7) / 8;
        int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        if (t >= mt * nt * a.ksn) return;  // whole workgroup: padding
        sl = t / (mt * nt);
        t -= sl * (mt * nt);
        tn = t / mt;
        tm = t - tn * mt;
    }
    const int m0 = tm * Cfg::BM, n0 = tn * Cfg::BN, mrows = min(Cfg::BM, a.M - m0);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, q = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % Cfg::WM, wn = wave / Cfg::WM;
    const int units = a.K / 64, u0 = 2 * (int)((long)(units / 2) * sl / a.ksn), u1 = 2 * (int)((long)(units / 2) * (sl + 1) / a.ksn);
    // A: chunk tid + THREADS i of the unit: row / 8, position / 8 swizzled by the row
    const uint16_t *ap[Cfg::LOADS];
    uint32_t ad[Cfg::LOADS];
#pragma unroll
    for (int i = 0; i < Cfg::LOADS; ++i) {
        const int ch = tid + Cfg::THREADS * i, r = ch >> 3, j = ch & 7;
        ap[i] = a.A + (size_t)(m0 + min(r, mrows - 1)) * a.K + 8 * j;
        ad[i] = (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4));
    }
    u32x4_t av[Cfg::LOADS];
    auto a_load = [&](int u) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < Cfg::LOADS; ++i) av[i] = *(const u32x4_t *)(ap[i] + 64 * (size_t)min(u, units - 1));
    };
    auto a_store = [&](int p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < Cfg::LOADS; ++i) *(u32x4_t *)(lds[p] + ad[i]) = av[i];
    };
    uint32_t ar[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = G < 64 ? 4 * (i >> 1) + 2 * q + (i & 1) : 4 * q + i;
        ar[i] = (uint32_t)((64 * wm + c) * 128 + ((j ^ (c & 7)) << 4));
    }
    I4Src<CB, 2, G, ZP, false> bs;
    bs.B = a.B;
    bs.S = a.S;
    bs.Z = a.Z;
    bs.N = a.N;
    bs.units = units;
    bs.q = q;
    bs.col = (uint32_t)min(n0 + 64 * wn + CB * c, a.N - CB);
    const I4Const k4 = i4_const<BF16, OFF>();
    const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
    const uint32_t ones[4] = {one, one, one, one};
    f32x16_t acc[MB][CB], part[MB][CB], sums[OFF ? MB : 1];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[mb][cb] = f32x16_t{};
    auto unit = [&](int u, int s) __attribute__((always_inline)) {
        // (every wave has read unit u - 1's buffer, which unit u + 1 is stored to)
        tile_barrier();
        u32x4_t af[2][MB];
        auto a_frag = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) af[i & 1][mb] = *(const u32x4_t *)(lds[s] + ar[i] + 4096 * mb);
        };
        a_frag(0);
        a_store(s ^ 1);
        a_load(u + 2);
        uint32_t w[CB][4];
        typename KwVec<CB>::S sr[GU], zr[GU];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[cb][i] = bs.w[s][cb][i];
#pragma unroll
        for (int g = 0; g < GU; ++g) {
            sr[g] = bs.sr[s][g];
            if constexpr (ZP) zr[g] = bs.zr[s][g];
        }
        bs.load(u + 2, s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < 3) a_frag(i + 1);
            const bool first = G == 128 ? i == 0 && s == 0 : G == 64 ? i == 0 : (i & 1) == 0;
            const bool last = G == 128 ? i == 3 && s == 1 : G == 64 ? i == 3 : (i & 1) == 1;
            if constexpr (OFF)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) sums[mb] = kw_mfma<BF16>(af[i & 1][mb], ones, first ? f32x16_t{} : sums[mb]);
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                uint32_t b[4];
                i4_decode<BF16, OFF>(w[cb][i], k4, b);
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) part[mb][cb] = kw_mfma<BF16>(af[i & 1][mb], b, first ? f32x16_t{} : part[mb][cb]);
            }
            if (last)
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    const int g = G < 64 ? i >> 1 : 0;
                    const float sc = i4_scale<CB, BF16>(sr[g], cb);
                    float of = -24.0f;
                    if constexpr (ZP) of -= i4_scale<CB, BF16>(zr[g], cb);
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            float v = part[mb][cb][r];
                            if constexpr (OFF) v = __builtin_fmaf(sums[mb][r], of, v);
                            acc[mb][cb][r] = __builtin_fmaf(v, sc, acc[mb][cb][r]);
                        }
                }
        }
    };
    a_load(u0);
    bs.load(u0, 0);
    a_store(0);
    a_load(u0 + 1);
    bs.load(u0 + 1, 1);
    for (int u = u0; u < u1; u += 2) {  // (whole 128-row steps)
        unit(u, 0);
        unit(u + 1, 1);
    }
    const int n = n0 + 64 * wn + CB * c;
    // this lane's outputs (m, n), (m, n + 1): element r of row block mb
    auto row_of = [&](int mb, int r) __attribute__((always_inline)) { return 64 * wm + 32 * mb + 8 * (r >> 2) + 4 * q + (r & 3); };
    if (a.ksn > 1) {  // (uniform) as kw_finish: the last of the tile's slices adds them in order
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = row_of(mb, r);
                if (m >= mrows || n >= a.N) continue;
                const uint64_t x = (uint64_t)__float_as_uint(acc[mb][0][r]) | ((uint64_t)__float_as_uint(acc[mb][1][r]) << 32);
                __hip_atomic_store((uint64_t *)(a.part + ((size_t)sl * a.M + m0 + m) * a.N + n), x, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();  // every wave's sums are stored
        uint32_t *flag = (uint32_t *)lds[0];
        if (wave == 0) {
            const bool last = kw_arrive(a.cnt + 2 * ((size_t)tm * nt + tn), a.ksn, lane);
            if (lane == 0) *flag = last;
        }
        __syncthreads();
        if (!*flag) return;  // (uniform)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
            for (int s = 0; s < a.ksn; ++s) {
                uint64_t x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    x[r] = __hip_atomic_load((const uint64_t *)(a.part + ((size_t)s * a.M + m0 + min(row_of(mb, r), mrows - 1)) * a.N +
                                                                min(n, a.N - CB)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float lo = __uint_as_float((uint32_t)x[r]), hi = __uint_as_float((uint32_t)(x[r] >> 32));
                    acc[mb][0][r] = s ? acc[mb][0][r] + lo : lo;
                    acc[mb][1][r] = s ? acc[mb][1][r] + hi : hi;
                }
            }
        }
    }
    epi_dispatch(a.postop, a.out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
        constexpr int P = decltype(P_)::value;
        constexpr bool F32 = decltype(F_)::value;
        if (n >= a.N) return;
        float bias[CB] = {0.0f, 0.0f};
        if constexpr (postop_needs_bias(P))
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
                bias[cb] = F32 ? ((const float *)a.Bias)[n + cb] : dt2f<BF16>(((const uint16_t *)a.Bias)[n + cb]);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
            // a row block's Other values all in flight (one after the other: 164 against 149 us at M =
            // 1024 K = 4096 N = 14336, silu(acc) * other)
            uint32_t o[16] = {};
            if constexpr (postop_needs_other(P))
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    o[r] = *(const uint32_t *)(a.Other + (size_t)(m0 + min(row_of(mb, r), mrows - 1)) * a.N + n);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = row_of(mb, r);
                const float x = epi_apply_c<P>(acc[mb][0][r], dt2f<BF16>(o[r] & 0xffffu), bias[0]);
                const float y = epi_apply_c<P>(acc[mb][1][r], dt2f<BF16>(o[r] >> 16), bias[1]);
                if (m >= mrows) continue;
                const size_t i = (size_t)(m0 + m) * a.N + n;
                if constexpr (F32) *(float2 *)((float *)a.C + i) = make_float2(x, y);
                else *(uint32_t *)((uint16_t *)a.C + i) = f2dt<BF16>(x) | (f2dt<BF16>(y) << 16);
            }
        }
    });
}

template <class Cfg, bool BF16, int G, bool ZP> hipError_t tile_launch(const I4TileArgs &a, hipStream_t st) {
    const int mt = (a.M + Cfg::BM - 1) / Cfg::BM, nt = (a.N + Cfg::BN - 1) / Cfg::BN;
    hipLaunchKernelGGL((k_int4_gemm_tile<Cfg, BF16, G, ZP>), dim3(8 * ((mt * nt * a.ksn + 7) / 8)), dim3(Cfg::THREADS), 0, st, a);
    return hipGetLastError();
}
template <class Cfg> hipError_t tile_pick(const I4TileArgs &a, bool bf, int group, hipStream_t st) {
    auto z = [&](auto b, auto g) {
        return a.Z ? tile_launch<Cfg, decltype(b)::value, decltype(g)::value, true>(a, st)
                   : tile_launch<Cfg, decltype(b)::value, decltype(g)::value, false>(a, st);
    };
    auto g = [&](auto b) {
        return group == 32   ? z(b, std::integral_constant<int, 32>{})
               : group == 64 ? z(b, std::integral_constant<int, 64>{})
                             : z(b, std::integral_constant<int, 128>{});
    };
    return bf ? g(std::true_type{}) : g(std::false_type{});
}

}  // namespace

// ksn K slices (> 1: their sums in part, the tiles' arrival counters at cnt); operands
// 16-byte aligned.
ternocl_status int4_gemm_tile_run(int dtype, const void *A, const uint32_t *B, const void *S, const void *Z, void *C,
                                  const void *Other, const void *Bias, int M, int N, int K, int group, int postop,
                                  int out_f32, int ksn, float *part, uint64_t *cnt, hipStream_t st) {
    const I4TileArgs a = {(const uint16_t *)A, B, (const uint16_t *)S, (const uint16_t *)Z, C, (const uint16_t *)Other, Bias,
                          M, N, K, postop, out_f32, ksn, part, cnt};
    return launch_status(tile_pick<TileCfg<2, 4>>(a, dtype == TERNOCL_BF16, group, st));
}

}  // namespace tcl
