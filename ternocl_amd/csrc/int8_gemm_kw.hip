// int8_gemm_kw.hip -- products of 8-bit integers with a scale for each token and channel
// (ternocl_int8_gemm) for up to some tens of rows on gfx950, and the choice between the engines:
//
//   C[m,n] = ct(epi((sum_k A[m,k] B[k,n]) SB[n] SA[m])),  exact 32-bit sums
//
// Few rows are bound by the weights' stream (K N bytes; at 24 rows 48 operations a byte, at 5 to 6
// TB/s an eighth of the rate that a large product reaches).  So nothing stands between memory and
// the matrix cores: 16 rows of a column lie together ([K/16][N][16]), so that a 16-byte load a lane is an operand
// of v_mfma_i32_16x16x64_i8 (four runs of 256 bytes, wider strips longer ones), with no LDS, no
// barrier and no instruction on the way.
//   * A workgroup's waves split K and each streams its own part of a strip of columns, several
//     units of 64 or 128 rows in flight; their sums meet once, in LDS.  Sums are whole numbers:
//     the same bits whatever the split.
//   * Columns are the instruction's rows: a lane ends with four adjacent outputs of a row, and
//     loads what their epilogue reads before the walk.
//   * Activations of up to 8 rows may be loaded as fragments (lanes past the last row read its line
//     again); of more, where a fragment load would touch a cache line a row, they go in whole lines
//     through the wave's own LDS: 48 x 5120 x 5120 15.2 -> 11.4 us.
// Captured, bf16, by card, weights used just before and in the last-level cache where they fit / weights
// from HBM, as a model's next token finds them: 1 x 4096 x 4096 (16.8 MB) 4.4 to 5.2 us / 5.5, 24 x 14336 x
// 4096 (58.7 MB, residual) 11.2 to 12.3 / 17.8, 4 x 4096 x 151680 (621 MB, fp32 out) 104 to 116: 5.3 to 5.9
// TB/s.  Both the choice of tile and the cache policy below are fitted to the former.
#include "int8_epi.hpp"

#include <algorithm>
#include <cmath>

namespace tcl {
hipError_t int8_tile_run(int tile, int dtype, const I8Args &a, hipStream_t st);  // int8_gemm_tile.hip
namespace {

// 16 MB rows x 16 CB columns, WK waves over K, PF units of U rows of K of weights in flight.
// AD: 0 for activations loaded as fragments, else the units of them in flight on their way
// through a wave's own LDS.
template <int MB_, int CB_, int WK_, int PF_, int AD_, int U_ = 128> struct I8Kw {
    static constexpr int R = 16, MB = MB_, CB = CB_, WK = WK_, PF = PF_, AD = AD_, U = U_;
    static constexpr int THREADS = 64 * WK, BM = R * MB, BN = R * CB;
    static constexpr int S = U / 64;   // matrix instructions (16-byte loads) a unit and block
    static constexpr int AL = BM / 8;  // 16-byte loads of a unit's rows
    static constexpr int ITEMS = MB * CB * 64, SUMS = WK * ITEMS * 16, ABUF = AD ? WK * 2 * BM * 128 : 0;
    static constexpr int LDS = SUMS > ABUF ? SUMS : ABUF;
    static_assert(AD == 0 || (PF % AD == 0 && PF % 2 == 0 && U == 128), "slots by the unrolled walk");
    static_assert(ITEMS <= THREADS, "four outputs a thread at most");
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

// NT: weights loaded past the last-level cache.
template <class T, bool BF16, bool NT> __global__ void __launch_bounds__(T::THREADS) k_int8_gemm_kw(const I8Args a) {
    constexpr int R = T::R, MB = T::MB, CB = T::CB, PF = T::PF, S = T::S, AD = T::AD, AL = T::AL;
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_lds[];
    const int mt = (a.M + T::BM - 1) / T::BM, nt = (a.N + T::BN - 1) / T::BN;
    int tm, tn, sl;
    if (!i8_kw_tile_of(blockIdx.x, mt, nt, a.ksn, tm, tn, sl)) return;  // (whole workgroup)
    const int m0 = tm * T::BM, n0 = tn * T::BN, mrows = min(T::BM, a.M - m0);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & (R - 1), g = lane / R;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int units = a.K / T::U, s0 = (int)((long)units * sl / a.ksn), s1 = (int)((long)units * (sl + 1) / a.ksn);
    const int u0 = s0 + (s1 - s0) * wave / T::WK, u1 = s0 + (s1 - s0) * (wave + 1) / T::WK;
    // instruction s of a unit: lane (c, g) holds rows (U / S) s + 16 g .. + 15 of K of its row
    // and column
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
    const size_t bunit = (size_t)a.N * T::U, bstep = bunit / S;
    i32x4_t bf[PF][S][CB], af[AD ? 1 : PF][S][MB], av[AD ? AD : 1][AL];
    uint8_t *ab = i8_lds + wave * 2 * T::BM * 128, *aw = ab + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
    // (past the end: read again, not multiplied)
    auto b_load = [&](int u, int p) __attribute__((always_inline)) {
        const int uc = min(u, u1 - 1);
        const int8_t *pb = a.B + bunit * (size_t)uc;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const i32x4_t *w = (const i32x4_t *)(pb + s * bstep + vb[cb]);
                bf[p][s][cb] = NT ? __builtin_nontemporal_load(w) : *w;
            }
        if constexpr (!AD) {
            const int8_t *pa = Ab + T::U * (size_t)uc;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) af[p][s][mb] = *(const i32x4_t *)(pa + s * (T::U / S) + va[mb]);
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
    // this thread's outputs (m, n .. n + 3); what their epilogue reads is on its way while the
    // products run
    const int il = tid & 63, ib = tid >> 6, m = m0 + R * (ib / CB) + (il & (R - 1)), n = n0 + R * (ib % CB) + 4 * (il / R);
    const bool mine = tid < T::ITEMS && m < m0 + mrows && n < a.N;
    I8Col col;
    I8Row row;
    if (mine) {
        col = i8_col(a, n);
        row = i8_row(a, m, n);
    }
    i32x4_t acc[MB][CB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[mb][cb] = i32x4_t{};
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
                for (int mb = 0; mb < MB; ++mb)  // (columns as the matrix' rows: a lane gets four adjacent ones)
                    acc[mb][cb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[p][s][cb], f[mb], acc[mb][cb], 0, 0, 0);
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
            red[wave * T::ITEMS + (mb * CB + cb) * 64 + lane] = acc[mb][cb];
    __syncthreads();
    if (a.ksn > 1) {
        if (mine) {
            i32x4_t s = red[tid];
#pragma unroll
            for (int w = 1; w < T::WK; ++w) s += red[w * T::ITEMS + tid];
            i8_part_store(a.part + ((size_t)sl * a.M + m) * a.N + n, s);
        }
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
    }
    if (!mine) return;
    i32x4_t s;
    if (a.ksn > 1) {
        const int *p = a.part + (size_t)m * a.N + n;
        s = i8_part_load(p);
        for (int k = 1; k < a.ksn; ++k) s += i8_part_load(p + (size_t)k * a.M * a.N);
    } else {
        s = red[tid];
#pragma unroll
        for (int w = 1; w < T::WK; ++w) s += red[w * T::ITEMS + tid];
    }
    epi_dispatch(a.postop, a.out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
        i8_out<BF16, decltype(P_)::value, decltype(F_)::value>(a, m, n, s, col, row);
    });
}

// Weights of more than 100 MB, which the 256 MB cache cannot keep beside others, go past it: 1 x
// 5120 x 34816 33.9 -> 31.8 us, 4 x 4096 x 151680 112 -> 104; smaller ones that are still there
// from their last use are read faster: 24 x 14336 x 4096 without a residual 15.7 -> 12.3 (from HBM
// 15.3 past it and 15.4).
template <class T> hipError_t i8_kw_launch(int dtype, const I8Args &a, hipStream_t st) {
    const long tiles = (long)((a.M + T::BM - 1) / T::BM) * ((a.N + T::BN - 1) / T::BN) * a.ksn;
    const bool nt = (long)a.K * a.N > 100000000;
    auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3((unsigned)(8 * ((tiles + 7) / 8))), dim3(T::THREADS), T::LDS, st, a); };
    if (dtype == TERNOCL_BF16) nt ? go(k_int8_gemm_kw<T, true, true>) : go(k_int8_gemm_kw<T, true, false>);
    else nt ? go(k_int8_gemm_kw<T, false, true>) : go(k_int8_gemm_kw<T, false, false>);
    return hipGetLastError();
}

// ---- host side: the choice of tile and K slices ------------------------------------

// A launch's time in us, by tile.  With w = tiles x slices / 256 workgroups a CU (part of them in
// whole rounds), s = stages of 128 rows of K a slice and 10^6 weights and outputs:
//   walk    = (s + edge) (one + two min(w - 1, 1) + more (w - 2)) for w above 1 and 2, `one`
//             times 1 + far where the weights come from HBM and not the last-level cache, and
//             times 1 + rows (M - 1) / 8 for activations loaded as fragments
//   memory  = weights / in + 2 outputs / out
//   time    = base + (walk^4 + memory^4)^(1/4), with slices + arrive + each slices + sums slices
//             outputs
// Fitted (logarithms, least squares, one fit a tile) to 220000 graph-timed calls on three sets of
// operands (weights up to some 85 MB: from the last-level cache), 11630 shapes of M = 1..4096, K =
// 256..14336, N = 64..151680: rms 4 to 9%.  21 tiles were timed and these 14 kept: the choice is
// 1.1% behind the fastest of them on average and 1.4% behind the fastest of all (95 of 100 within 8%,
// the worst 41%).  With weights from HBM 9 to 64 rows take 20 to 45% longer than they were timed
// at, and another tile may be ahead (32 x 4096 x 14336: 17.5 us, 32 x 64 tiles 14.8).  The second
// tile's `out` is what the fit left: no call of up to 8 rows is bound by its outputs.
// Narrow tiles fill the chip; wide ones read the activations, low ones the weights fewer times.
enum I8Kind { kFew, kRows, kTile };  // activations as fragments (M <= 8), through a wave's LDS, int8_gemm_tile.hip
struct I8Choice {
    int bm, bn, wk;  // rows, columns, waves (kTile: groups of them) over K
    I8Kind kind;
    int num;
    struct {
        double base, one, two, more, in, whole, arrive, sums, each, edge, out, far, rows;
    } t;
};
constexpr I8Choice kI8[] = {
    {16, 16, 4, kFew, 0, {2.87, 0.0272, 0.0549, 0.0614, 6.74, 1, 0.483, 8.4, 0.303, 3.77, 0.222, 1.62, 0.99}},
    {16, 32, 4, kFew, 1, {2.99, 0.0443, 0.0996, 0.12, 6.99, 1, 0.545, 4.68, 0.303, 1.36, 1.17e+07, 1.07, 0.533}},
    {16, 16, 4, kRows, 2, {2.94, 0.0397, 0.0303, 0.0727, 6.56, 0.685, 0.478, 6.13, 0.32, 1.82, 0.916, 2.18, 0}},
    {16, 32, 4, kRows, 3, {3.07, 0.0511, 0.089, 0.143, 6.81, 0.674, 0.594, 4.26, 0.31, 0.795, 2.86, 1.81, 0}},
    {16, 64, 4, kRows, 4, {3.4, 0.0847, 0.191, 0.294, 6.81, 0.754, 0.793, 3.41, 0.313, 0.573, 2.56, 1.14, 0}},
    {32, 32, 4, kRows, 5, {3.4, 0.0692, 0.12, 0.173, 7.32, 0.77, 0.659, 4.84, 0.318, 0.489, 1.13, 0.916, 0}},
    {32, 64, 4, kTile, 0, {3.19, 0.113, 0.149, 0.151, 6.06, 0.91, 0.585, 2.58, 0.348, 6.78, 0.856, 0.867, 0}},
    {32, 128, 1, kTile, 1, {3.13, 0.228, 0.234, 0.245, 6.48, 0.748, 0.337, 1.79, 1.11, 1.74, 2.38, 0.729, 0}},
    {32, 128, 2, kTile, 2, {3.18, 0.187, 0.241, 0.244, 6.19, 0.858, 0.632, 2.07, 0.622, 3.95, 1.34, 0.971, 0}},
    {64, 128, 1, kTile, 3, {3.43, 0.328, 0.337, 0.334, 6.41, 0.739, 0, 1.53, 2.01, 3.12, 2.85, 0.283, 0}},
    {64, 128, 2, kTile, 4, {2.75, 0.261, 0.43, 0.365, 6.27, 0.733, 0.226, 2.2, 1.09, 8.37, 1.16, 0.437, 0}},
    {64, 256, 1, kTile, 5, {2.87, 0.377, 0.738, 0.616, 6.49, 0.735, 0.182, 2.61, 1.95, 5.53, 1.78, 0.718, 0}},
    {128, 256, 1, kTile, 6, {4.9, 0.782, 0.999, 0.969, 6.84, 0.719, 0, 1.47, 7.36, 3.76, 2.44, 0.144, 0}},
    {128, 512, 1, kTile, 7, {3.69, 1.14, 2.39, 1.72, 5.27, 0.462, 0, 2, 7.38, 4.53, 2.34, 0.178, 0}}
};

struct I8Plan {
    int choice, ks;
};

I8Plan i8_plan(int M, int N, int K, size_t ws_bytes) {
    I8Plan best = {-1, 1};
    double least = 1e30;
    const double kn = 1e-6 * K * N, mn = 1e-6 * M * N, hbm = 1.0 / (1.0 + std::exp((85.0 - kn) / 10.0));
    for (int i = 0; i < (int)(sizeof(kI8) / sizeof(kI8[0])); ++i) {
        const I8Choice &c = kI8[i];
        // (past those rows the fragments' loads, past 48 a tile's many row blocks are far behind; up to
        // 16 rows a tile of 32 only where K is short)
        if ((c.kind == kFew && M > 8) || (c.kind == kRows && M > (c.bm == 16 ? 48 : 96)) || (c.kind == kTile && M <= 16 && K > 1024) ||
            (c.bm > 32 && c.bm >= 2 * M))
            continue;
        const long tiles = (((long)M + c.bm - 1) / c.bm) * (((long)N + c.bn - 1) / c.bn);
        if (tiles > 8000000) continue;  // (a launch's threads: 32 bits)
        for (int ks = 1; ks <= 8; ++ks) {
            if (ks > 1 && (kWsHeader + (size_t)ks * M * N * 4 > ws_bytes || K / 128 < 4 * ks || tiles * ks > 640 || tiles > 256)) break;
            const double w = tiles * ks / 256.0, r = c.t.whole * std::ceil(w) + (1.0 - c.t.whole) * w;
            double one = c.t.one * (1.0 + c.t.far * hbm) * (1.0 + c.t.rows * (M - 1) / 8.0);
            if (r > 1.0) one += c.t.two * std::min(r - 1.0, 1.0);
            if (r > 2.0) one += c.t.more * (r - 2.0);
            const double walk = ((K / 128 + ks - 1) / ks + c.t.edge) * one, mem = kn / c.t.in + 2.0 * mn / c.t.out;
            double us = c.t.base + std::sqrt(std::sqrt(walk * walk * walk * walk + mem * mem * mem * mem));
            if (ks > 1) us += c.t.arrive + c.t.each * ks + c.t.sums * ks * mn;
            if (us < least) {
                least = us;
                best = {i, ks};
            }
        }
    }
    return best;
}

}  // namespace

// Workspace of a call's K split (0: none).
size_t int8_gemm_ws_need(int M, int N, int K) {
    const int ks = i8_plan(M, N, K, ~(size_t)0).ks;
    return ks == 1 ? 0 : kWsHeader + (size_t)ks * M * N * 4;
}

// The tile of a call on aligned operands, for ternocl_kw_tile_of.
bool int8_gemm_tile(int M, int N, int K, size_t ws_bytes, ternocl_kw_tile &t) {
    const I8Plan p = i8_plan(M, N, K, ws_bytes);
    if (p.choice < 0) return false;
    const I8Choice &c = kI8[p.choice];
    t = {c.bm, c.bn, c.wk, p.ks, c.kind != kFew};
    return true;
}

// (operands 16-byte aligned)
ternocl_status int8_gemm_run(int dtype, const int8_t *A, const float *SA, const int8_t *B, const float *SB, void *C,
                             const void *Other, const void *Bias, int M, int N, int K, int postop, int out_f32, void *ws,
                             size_t ws_bytes, hipStream_t st) {
    const I8Plan p = i8_plan(M, N, K, ws && ((uintptr_t)ws & 15) == 0 ? ws_bytes : 0);
    if (p.choice < 0) {
        set_error("M x N needs more tiles than a launch holds");
        return TERNOCL_ERR_UNSUPPORTED_SHAPE;
    }
    const I8Args a = {A, SA, B, SB, C, (const uint16_t *)Other, Bias, M, N, K, postop, out_f32, p.ks,
                      p.ks > 1 ? (int *)((uint8_t *)ws + kWsHeader) : nullptr, p.ks > 1 ? (uint64_t *)ws : nullptr};
    const I8Choice &c = kI8[p.choice];
    if (c.kind == kTile) return launch_status(int8_tile_run(c.num, dtype, a, st));
    switch (c.num) {
    case 0: return launch_status(i8_kw_launch<I8Kw<1, 1, 4, 4, 0>>(dtype, a, st));
    case 1: return launch_status(i8_kw_launch<I8Kw<1, 2, 4, 4, 0, 64>>(dtype, a, st));
    case 2: return launch_status(i8_kw_launch<I8Kw<1, 1, 4, 2, 2>>(dtype, a, st));
    case 3: return launch_status(i8_kw_launch<I8Kw<1, 2, 4, 2, 2>>(dtype, a, st));
    case 4: return launch_status(i8_kw_launch<I8Kw<1, 4, 4, 2, 2>>(dtype, a, st));
    default: return launch_status(i8_kw_launch<I8Kw<2, 2, 4, 2, 2>>(dtype, a, st));
    }
}

}  // namespace tcl
