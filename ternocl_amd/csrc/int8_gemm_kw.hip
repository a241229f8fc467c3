// int8_gemm_kw.hip -- products of 8-bit integers for few rows (ternocl_int8_gemm): a
// workgroup's waves split K, each streaming its part of the weights and the activations
// straight into matrix-core fragments.
#include "int8_epi.hpp"

namespace tcl {
hipError_t int8_tile_run(int tile, int dtype, const I8Args &a, hipStream_t st);  // int8_gemm_tile.hip
namespace {

// R MB rows x R CB columns, R = 16 or 32 (the matrix instruction), WK waves over K, PF units
// of 128 rows of K of weights in flight.  AD: 0 for activations loaded as fragments, else the
// units of them in flight on their way through a wave's own LDS.
template <int R_, int MB_, int CB_, int WK_, int PF_, int AD_> struct I8Kw {
    static constexpr int R = R_, MB = MB_, CB = CB_, WK = WK_, PF = PF_, AD = AD_;
    static constexpr int THREADS = 64 * WK, BM = R * MB, BN = R * CB;
    static constexpr int S = R / 8;            // matrix instructions (16-byte loads) a unit and block
    static constexpr int Q = R == 16 ? 1 : 4;  // 4-column quads of a lane's outputs of a block
    static constexpr int AL = BM / 8;          // 16-byte loads of a unit's rows
    static constexpr int ITEMS = MB * CB * Q * 64, SUMS = WK * ITEMS * 16, ABUF = AD ? WK * 2 * BM * 128 : 0;
    static constexpr int LDS = SUMS > ABUF ? SUMS : ABUF;
    static_assert(AD == 0 || (PF % AD == 0 && PF % 2 == 0), "slots by the unrolled walk");
};

// Workgroup -> tile: XCD x (workgroups x, x + 8, ...) takes a contiguous range of them, the
// row tiles of a column strip (and slice) next to each other, so that its weights come into
// one L2 once.
__device__ __forceinline__ bool i8_kw_tile_of(int id, int mt, int nt, int ksn, int &tm, int &tn, int &sl) {
    const int total = mt * nt * ksn, per = (total + 7) / 8;
    int t = (id & 7) * per + (id >> 3);
    if (t >= total) return false;
    tm = t % mt;
    t /= mt;
    sl = t % ksn;
    tn = t / ksn;
    return true;
}

template <int R> struct I8Acc;
template <> struct I8Acc<16> { typedef i32x4_t T; };
template <> struct I8Acc<32> { typedef i32x16_t T; };

template <class T, bool BF16> __global__ void __launch_bounds__(T::THREADS) k_int8_gemm_kw(const I8Args a) {
    constexpr int R = T::R, MB = T::MB, CB = T::CB, PF = T::PF, S = T::S, Q = T::Q, AD = T::AD, AL = T::AL;
    typedef typename I8Acc<R>::T Acc;
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_lds[];
    const int mt = (a.M + T::BM - 1) / T::BM, nt = (a.N + T::BN - 1) / T::BN;
    int tm, tn, sl;
    if (!i8_kw_tile_of(blockIdx.x, mt, nt, a.ksn, tm, tn, sl)) return;  // (whole workgroup)
    const int m0 = tm * T::BM, n0 = tn * T::BN, mrows = min(T::BM, a.M - m0);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & (R - 1), g = lane / R;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int units = a.K / 128, s0 = (int)((long)units * sl / a.ksn), s1 = (int)((long)units * (sl + 1) / a.ksn);
    const int u0 = s0 + (s1 - s0) * wave / T::WK, u1 = s0 + (s1 - s0) * (wave + 1) / T::WK;
    // instruction s of a unit: lane (c, g) holds rows (128 / S) s + 16 g .. + 15 of K of its
    // row and column
    const int8_t *Ab = a.A + (size_t)m0 * a.K;
    uint32_t va[AD ? AL : MB], vb[CB], ar[S];
    if constexpr (AD) {  // 8 rows of 128 bytes a load
#pragma unroll
        for (int i = 0; i < AL; ++i) va[i] = (uint32_t)min(8 * i + (lane >> 3), mrows - 1) * (uint32_t)a.K + 16u * (lane & 7);
#pragma unroll
        for (int s = 0; s < S; ++s) ar[s] = (uint32_t)(c * 128 + (((8 / S * s + g) ^ (c & 7)) << 4));
    } else {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) va[mb] = (uint32_t)min(R * mb + c, mrows - 1) * (uint32_t)a.K + 16u * g;
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) vb[cb] = ((uint32_t)g * (uint32_t)a.N + (uint32_t)min(n0 + R * cb + c, a.N - 1)) * 16u;
    const size_t bunit = (size_t)a.N * 128, bstep = bunit / S;
    i32x4_t bf[PF][S][CB], af[AD ? 1 : PF][S][MB], av[AD ? AD : 1][AL];
    uint8_t *ab = i8_lds + wave * 2 * T::BM * 128, *aw = ab + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
    // (past the end: read again, not multiplied)
    auto b_load = [&](int u, int p) __attribute__((always_inline)) {
        const int uc = min(u, u1 - 1);
        const int8_t *pb = a.B + bunit * (size_t)uc;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) bf[p][s][cb] = __builtin_nontemporal_load((const i32x4_t *)(pb + s * bstep + vb[cb]));
        if constexpr (!AD) {
            const int8_t *pa = Ab + 128 * (size_t)uc;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) af[p][s][mb] = *(const i32x4_t *)(pa + s * (128 / S) + va[mb]);
        }
    };
    auto a_load = [&](int u, int p) __attribute__((always_inline)) {
        const int8_t *pa = Ab + 128 * (size_t)min(u, u1 - 1);
#pragma unroll
        for (int i = 0; i < AL; ++i) av[p][i] = *(const i32x4_t *)(pa + va[i]);
    };
    auto a_store = [&](int p, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AL; ++i) *(i32x4_t *)(aw + buf * T::BM * 128 + 1024 * i) = av[p][i];
    };
    Acc acc[MB][CB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[mb][cb] = Acc{};
    // unit u in slot p: its rows lie in LDS buffer p % 2
    auto unit = [&](int u, int p, bool more) __attribute__((always_inline)) {
        if constexpr (AD) {
            a_store((p + 1) % AD, (p + 1) & 1);  // unit u + 1
            a_load(u + 1 + AD, (p + 1) % AD);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            i32x4_t f[MB];
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) f[mb] = AD ? *(const i32x4_t *)(ab + (p & 1) * T::BM * 128 + ar[s] + R * 128 * mb) : af[AD ? 0 : p][s][mb];
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) {  // (columns as the matrix' rows: a lane gets four adjacent ones)
                    if constexpr (R == 16)
                        acc[mb][cb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[p][s][cb], f[mb], acc[mb][cb], 0, 0, 0);
                    else
                        acc[mb][cb] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[p][s][cb], f[mb], acc[mb][cb], 0, 0, 0);
                }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) b_load(u + PF, p);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (u0 < u1) {
        if constexpr (AD) {
#pragma unroll
            for (int p = 0; p < AD; ++p) a_load(u0 + p, p);
        }
#pragma unroll
        for (int p = 0; p < PF; ++p) b_load(u0 + p, p);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (AD) {
            a_store(0, 0);
            a_load(u0 + AD, 0);
        }
        int u = u0;
        for (; u + PF <= u1; u += PF)
#pragma unroll
            for (int p = 0; p < PF; ++p) unit(u + p, p, true);
#pragma unroll
        for (int p = 0; p < PF - 1; ++p) {
            if (u + p >= u1) break;
            unit(u + p, p, false);
        }
    }
    // the waves' sums
    if constexpr (AD) __syncthreads();  // (they take the place of the rows)
    i32x4_t *red = (i32x4_t *)i8_lds;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int j = 0; j < Q; ++j)
                red[wave * T::ITEMS + ((mb * CB + cb) * Q + j) * 64 + lane] =
                    i32x4_t{acc[mb][cb][4 * j], acc[mb][cb][4 * j + 1], acc[mb][cb][4 * j + 2], acc[mb][cb][4 * j + 3]};
    __syncthreads();
    auto place = [&](int i, int &m, int &n) __attribute__((always_inline)) {
        const int l = i & 63, b = i >> 6, j = b % Q, cb = b / Q % CB, mb = b / Q / CB;
        m = R * mb + (l & (R - 1));
        n = n0 + R * cb + 8 * j + 4 * (l / R);
    };
    for (int i = tid; i < T::ITEMS; i += T::THREADS) {
        int m, n;
        place(i, m, n);
        if (m >= mrows || n >= a.N) continue;
        i32x4_t s = red[i];
#pragma unroll
        for (int w = 1; w < T::WK; ++w) s += red[w * T::ITEMS + i];
        if (a.ksn > 1) i8_part_store(a.part + ((size_t)sl * a.M + m0 + m) * a.N + n, s);
        else i8_store4<BF16>(a, m0 + m, n, s);
    }
    if (a.ksn == 1) return;
    // the last of the tile's slices adds them
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    uint32_t *flag = (uint32_t *)i8_lds;
    if (wave == 0) {
        const bool last = kw_arrive(a.cnt + 2 * ((size_t)tm * nt + tn), a.ksn, lane);
        if (lane == 0) *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
    for (int i = tid; i < T::ITEMS; i += T::THREADS) {
        int m, n;
        place(i, m, n);
        if (m >= mrows || n >= a.N) continue;
        const int *p = a.part + (size_t)(m0 + m) * a.N + n;
        i32x4_t s = i8_part_load(p);
        for (int k = 1; k < a.ksn; ++k) s += i8_part_load(p + (size_t)k * a.M * a.N);
        i8_store4<BF16>(a, m0 + m, n, s);
    }
}

template <class T> hipError_t i8_kw_launch(int dtype, const I8Args &a, hipStream_t st) {
    const long tiles = (long)((a.M + T::BM - 1) / T::BM) * ((a.N + T::BN - 1) / T::BN) * a.ksn;
    auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3((unsigned)(8 * ((tiles + 7) / 8))), dim3(T::THREADS), T::LDS, st, a); };
    if (dtype == TERNOCL_BF16) go(k_int8_gemm_kw<T, true>);
    else go(k_int8_gemm_kw<T, false>);
    return hipGetLastError();
}

// ---- host side: the choice of tile and K slices ------------------------------------

struct I8Choice {
    int bm, bn;
    bool tile;  // int8_gemm_tile.hip's, by its number
    int num;
};
constexpr I8Choice kI8[] = {{16, 16, false, 0}, {16, 32, false, 1}, {16, 64, false, 2}, {32, 64, true, 5}, {64, 64, true, 4},
                            {64, 128, true, 3}, {64, 256, true, 2}, {128, 256, true, 1}, {128, 512, true, 0}};

struct I8Plan {
    int choice, ks;
};

I8Plan i8_plan(int M, int N, int K, size_t ws_bytes) {
    auto tiles = [&](int i) { return (long)((M + kI8[i].bm - 1) / kI8[i].bm) * ((N + kI8[i].bn - 1) / kI8[i].bn); };
    int c = M <= 16 ? 0 : 3;
    const int last = M <= 16 ? 2 : 8;
    while (c < last && tiles(c + 1) >= 200) ++c;
    int ks = 1;
    while (ks < 8 && tiles(c) * ks * 2 <= 512 && K / ks >= 4096 && kWsHeader + (size_t)ks * 2 * M * N * 4 <= ws_bytes) ks *= 2;
    return {c, ks};
}

}  // namespace

// Workspace of a call's K split (0: none).
size_t int8_gemm_ws_need(int M, int N, int K) {
    const int ks = i8_plan(M, N, K, ~(size_t)0).ks;
    return ks == 1 ? 0 : kWsHeader + (size_t)ks * M * N * 4;
}

// (operands 16-byte aligned)
ternocl_status int8_gemm_run(int dtype, const int8_t *A, const float *SA, const int8_t *B, const float *SB, void *C,
                             const void *Other, const void *Bias, int M, int N, int K, int postop, int out_f32, void *ws,
                             size_t ws_bytes, hipStream_t st) {
    const I8Plan p = i8_plan(M, N, K, ws && ((uintptr_t)ws & 15) == 0 ? ws_bytes : 0);
    const I8Args a = {A, SA, B, SB, C, (const uint16_t *)Other, Bias, M, N, K, postop, out_f32, p.ks,
                      p.ks > 1 ? (int *)((uint8_t *)ws + kWsHeader) : nullptr, p.ks > 1 ? (uint64_t *)ws : nullptr};
    const I8Choice &c = kI8[p.choice];
    if (c.tile) return launch_status(int8_tile_run(c.num, dtype, a, st));
    const bool few = M <= 8;
    switch (c.num) {
    case 0: return launch_status(few ? i8_kw_launch<I8Kw<16, 1, 1, 4, 4, 0>>(dtype, a, st) : i8_kw_launch<I8Kw<16, 1, 1, 4, 2, 2>>(dtype, a, st));
    case 1: return launch_status(few ? i8_kw_launch<I8Kw<16, 1, 2, 4, 2, 0>>(dtype, a, st) : i8_kw_launch<I8Kw<16, 1, 2, 4, 2, 2>>(dtype, a, st));
    default: return launch_status(few ? i8_kw_launch<I8Kw<16, 1, 4, 4, 1, 0>>(dtype, a, st) : i8_kw_launch<I8Kw<16, 1, 4, 4, 2, 2>>(dtype, a, st));
    }
}

}  // namespace tcl
