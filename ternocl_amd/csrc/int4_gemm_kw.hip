// int4_gemm_kw.hip -- GEMM of 9 to some hundreds of rows on 4-bit weights with group
// scales for gfx950 (ternocl_int4_gemm), K split over the waves of a workgroup as in
// gemm_kw.hpp:
//
//   C[m,n] = ct(epi(sum_g S[g,n] (sum_{k in g} A[m,k] q[k,n] - Z[g,n] sum_{k in g} A[m,k])))
//
// Codes go to the matrix cores as small integers of the activations' type, so that the
// products are exact and nothing is rounded but fp32 sums; a scale group's sums are
// kept apart (part) and join the tile's by one FMA with S per output.
//   * fp16 without zero points: a nibble under the exponent of 1024 (or, in the upper half of
//     a byte, 16 times it), less 1032 (a sixteenth, less 72): q itself, nine operations a
//     word of 8 codes.
//   * bf16 has no packed arithmetic here, and zero points need the activations' sums anyway:
//     a nibble in the upper mantissa bits under the exponent of 16 reads q + 24, eight
//     operations a word.  24 + Z times the group's sum of activations is taken off: that sum
//     for a lane's rows comes out of a matrix instruction against ones, once per row block for
//     all columns.
//   * A lane's B fragments are word i of block q of a 64-row unit (16 bytes a column and
//     unit); in groups of 32 rows both halves of a fragment must lie in one block: words
//     2 q and 2 q + 1 of each.
//
// Why K over the waves: a wave decodes its own weights once and needs no barrier, and few rows
// give too few tiles for a wave each.  M = 24 K = 14336 N = 4096 bf16 (30 MB, 6.0 us of a
// large copy): 15.4 us a call, of which the walk's stream is 8.5, its first loads, the waves'
// and the slices' meeting the rest.  The more columns' activations a row block reads through
// L2, the more the walk waits for them (M = 100 K = N = 5120 fp16, 64 x 64 tiles: VALU 35% of a
// wave's time, waits for loads 29%, for issue 19%, MFMAs busy 23%); int4_gemm_tile.hip takes over
// where i4_plan puts it ahead.
#include "gemm_kw.hpp"
#include "int4_decode.hpp"

#include <algorithm>

namespace tcl {
// (int4_gemm_tile.hip)
ternocl_status int4_gemm_tile_run(int dtype, const void *A, const uint32_t *B, const void *S, const void *Z, void *C,
                                  const void *Other, const void *Bias, int M, int N, int K, int group, int postop,
                                  int out_f32, int ksn, float *part, uint64_t *cnt, hipStream_t st);
namespace {

// The K walk of one wave, units [u0, u1) of its 32 MB rows into acc: kw_walk's way of
// the activations.  With G = 128, u0 and u1 are even.
template <class Cfg, bool BF16, int G, bool ZP>
__device__ __forceinline__ void i4_walk(uint8_t *abuf, const uint16_t *A, const uint32_t va[4 * Cfg::MB], int u0, int u1,
                                        int units, I4Src<Cfg::CB, Cfg::PF, G, ZP> &bs, f32x16_t acc[Cfg::MB][Cfg::CB]) {
    constexpr int MB = Cfg::MB, CB = Cfg::CB, PF = Cfg::PF;
    constexpr bool OFF = BF16 || ZP;  // something times the groups' activation sums is taken off
    const int lane = threadIdx.x & 63, c = lane & 31, q = lane >> 5;
    u32x4_t av[4 * MB];
    auto a_load = [&](int u) __attribute__((always_inline)) {
        const uint16_t *p = A + 64 * (size_t)min(u, units - 1);
#pragma unroll
        for (int i = 0; i < 4 * MB; ++i) av[i] = *(const u32x4_t *)(p + va[i]);
    };
    // chunk j of row r at position j ^ (r % 8) of its 128 bytes; k-step i of lane (c, q)
    // reads row c's chunk of word i of its B fragments
    uint8_t *aw = abuf + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
    uint32_t ar[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = G < 64 ? 4 * (i >> 1) + 2 * q + (i & 1) : 4 * q + i;
        ar[i] = (uint32_t)(c * 128 + ((j ^ (c & 7)) << 4));
    }
    const I4Const k4 = i4_const<BF16, OFF>();
    const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
    const uint32_t ones[4] = {one, one, one, one};
    auto a_store = [&](int p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4 * MB; ++i) *(u32x4_t *)(aw + p * (MB * 4096) + 1024 * i) = av[i];
    };
    u32x4_t af[2][MB];
    auto a_frag = [&](int p, int i, u32x4_t f[MB]) __attribute__((always_inline)) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) f[mb] = *(const u32x4_t *)(abuf + p * (MB * 4096) + ar[i] + 4096 * mb);
    };
    f32x16_t part[MB][CB], sums[OFF ? MB : 1];
    auto unit = [&](int u, int s, bool more) __attribute__((always_inline)) {
        const int p = s & 1;
        uint32_t w[CB][4];
        float sc[I4Src<CB, PF, G, ZP>::GU][CB], of[I4Src<CB, PF, G, ZP>::GU][CB];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[cb][i] = bs.w[s][cb][i];
#pragma unroll
            for (int g = 0; g < I4Src<CB, PF, G, ZP>::GU; ++g) {
                sc[g][cb] = i4_scale<CB, BF16>(bs.sr[s][g], cb);
                if constexpr (OFF) {
                    float z = 24.0f;
                    if constexpr (ZP) z += i4_scale<CB, BF16>(bs.zr[s][g], cb);
                    of[g][cb] = -z;
                }
            }
        }
        if (more) bs.load(u + PF, s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i == 2) {
                __builtin_amdgcn_sched_barrier(0);
                a_store(p ^ 1);
                a_load(u + 2);
                __builtin_amdgcn_sched_barrier(0);
            }
            a_frag(i < 3 ? p : p ^ 1, (i + 1) & 3, af[(i + 1) & 1]);
            const bool first = G == 128 ? i == 0 && p == 0 : G == 64 ? i == 0 : (i & 1) == 0;
            const bool last = G == 128 ? i == 3 && p == 1 : G == 64 ? i == 3 : (i & 1) == 1;
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
                for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int g = G < 64 ? i >> 1 : 0;
                            float v = part[mb][cb][r];
                            if constexpr (OFF) v = __builtin_fmaf(sums[mb][r], of[g][cb], v);
                            acc[mb][cb][r] = __builtin_fmaf(v, sc[g][cb], acc[mb][cb][r]);
                        }
        }
    };
    if (u0 < u1) {
        a_load(u0);
#pragma unroll
        for (int s = 0; s < PF; ++s) bs.load(u0 + s, s);
        __builtin_amdgcn_sched_barrier(0);
        a_store(0);
        a_load(u0 + 1);
        __builtin_amdgcn_sched_barrier(0);
        a_frag(0, 0, af[0]);
        int u = u0;
        for (; u + PF - 1 < u1; u += PF)
#pragma unroll
            for (int s = 0; s < PF; ++s) unit(u + s, s, true);
#pragma unroll
        for (int s = 0; s < PF - 1; ++s) {
            if (u + s >= u1) break;
            unit(u + s, s, false);
        }
    }
}

struct I4GemmArgs {
    const uint16_t *A;
    const uint32_t *B;
    const uint16_t *S, *Z;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K, postop, out_f32, ksn;
    float *part;
    uint64_t *cnt;
};

// ksn > 1: workgroup (tile, slice sl) runs the units of its K slice (kw_finish).
template <class Cfg, bool BF16, int G, bool ZP> __global__ void __launch_bounds__(Cfg::THREADS) k_int4_gemm_kw(const I4GemmArgs a) {
    constexpr int MB = Cfg::MB, CB = Cfg::CB, WK = Cfg::WK;
    extern __shared__ __attribute__((aligned(16))) uint8_t kw_lds[];
    const int mt = (a.M + Cfg::BM - 1) / Cfg::BM, nt = (a.N + Cfg::BN - 1) / Cfg::BN, ksn = a.ksn;
    int tms, tn;
    if (!xcd_tile_ashare(blockIdx.x, mt * ksn, nt, tms, tn)) return;  // whole workgroup: padding
    const int tm = __builtin_amdgcn_readfirstlane(tms / ksn), sl = __builtin_amdgcn_readfirstlane(tms - tm * ksn);
    const int m0 = tm * Cfg::BM, n0 = tn * Cfg::BN;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kw = wave / Cfg::WM, wm = wave % Cfg::WM;
    const int c = lane & 31, q = lane >> 5;
    // this wave's units: a contiguous part of the slice's, in whole 128-row steps
    const int units = a.K / 64, steps = a.K / 128;
    const int s0 = (int)((long)steps * sl / ksn), s1 = (int)((long)steps * (sl + 1) / ksn);
    const int u0 = 2 * (s0 + (s1 - s0) * kw / WK), u1 = 2 * (s0 + (s1 - s0) * (kw + 1) / WK);
    const int mrows = min(Cfg::BM, a.M - m0);
    // A: chunk lane + 64 i of the unit -> row i * 8 + lane / 8, 16-byte chunk lane % 8
    // (rows past the tile's re-read its last row: their outputs are not stored)
    uint32_t va[4 * MB];
#pragma unroll
    for (int i = 0; i < 4 * MB; ++i)
        va[i] = (uint32_t)min(32 * MB * wm + (lane >> 3) + 8 * i, mrows - 1) * (uint32_t)a.K + 8u * (lane & 7);
    I4Src<CB, Cfg::PF, G, ZP> bs;
    bs.B = a.B;
    bs.S = a.S;
    bs.Z = a.Z;
    bs.N = a.N;
    bs.units = units;
    bs.q = q;
    bs.col = (uint32_t)min(n0 + CB * c, a.N - CB);
    f32x16_t acc[MB][CB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[mb][cb] = f32x16_t{};
    i4_walk<Cfg, BF16, G, ZP>(kw_lds + wave * (MB * 8192), a.A + (size_t)m0 * a.K, va, u0, u1, units, bs, acc);
    kw_finish<Cfg, BF16>(acc, kw_lds, a.C, a.Other, a.Bias, a.M, a.N, m0, mrows, n0, a.postop, a.out_f32, ksn, sl, a.part,
                         ksn > 1 ? a.cnt + 2 * ((size_t)tm * nt + tn) : nullptr);
}

template <class Cfg, bool BF16, int G, bool ZP> hipError_t i4_launch(const I4GemmArgs &a, hipStream_t st) {
    const int mt = (a.M + Cfg::BM - 1) / Cfg::BM, nt = (a.N + Cfg::BN - 1) / Cfg::BN;
    hipLaunchKernelGGL((k_int4_gemm_kw<Cfg, BF16, G, ZP>), dim3(xcd_ashare_grid(mt * a.ksn, nt)), dim3(Cfg::THREADS),
                       Cfg::LDS_BYTES, st, a);
    return hipGetLastError();
}
template <class Cfg> hipError_t i4_pick(const I4GemmArgs &a, bool bf, int group, hipStream_t st) {
    auto z = [&](auto b, auto g) {
        return a.Z ? i4_launch<Cfg, decltype(b)::value, decltype(g)::value, true>(a, st)
                   : i4_launch<Cfg, decltype(b)::value, decltype(g)::value, false>(a, st);
    };
    auto g = [&](auto b) {
        return group == 32   ? z(b, std::integral_constant<int, 32>{})
               : group == 64 ? z(b, std::integral_constant<int, 64>{})
                             : z(b, std::integral_constant<int, 128>{});
    };
    return bf ? g(std::true_type{}) : g(std::false_type{});
}

// ---- host side: the choice of tile and K slices ------------------------------------

// A launch's time in us by tile: base, and per round of 256 workgroups slope for each 1024
// rows of K; for fp16 without zero points / others, groups of 64 and 128 / of 32.  A K
// split costs 1.2 us and split for each 10^6 of its slices' sums.  Fitted (logarithms, least
// squares, one fit a class) to 3700 graph-timed calls, M = 9..2048, N = 1024..34816, K =
// 1024..28672: rms 15% for K over the waves, 8% for the 128 x 256 tiles; the tile chosen by
// it is 1.4% behind the fastest of all on average (24% at most).  Wider tiles read the
// activations fewer times; narrower ones fill the chip.  64 x 256, 64 x 128 and 128 x 128
// tiles with shared activations would gain 0.2% more.
struct I4Tile {
    int bm, bn;
    double base[4], slope[4], split;
};
constexpr I4Tile kI4Tiles[] = {{32, 32, {4.2, 4.4, 4.55, 4.7}, {1.77, 1.83, 1.93, 2.12}, 12.4},
                               {32, 64, {4.6, 4.8, 5.0, 5.2}, {2.54, 2.62, 2.67, 2.95}, 9.2},
                               {64, 64, {5.3, 5.8, 6.0, 6.2}, {3.6, 4.3, 5.0, 6.2}, 5.5},
                               {128, 256, {9.2, 9.6, 10.3, 10.45}, {13.95, 18.1, 18.7, 24.6}, 2.05}};
constexpr int kI4TileCount = sizeof(kI4Tiles) / sizeof(kI4Tiles[0]);
constexpr int kI4Shared = 3;  // the tile of int4_gemm_tile.hip

struct I4Plan {
    int tile, ks;  // ks: K slices (> 1 needs the workspace)
    double us;
};

// The cheapest tile and slice count with ws_bytes of workspace.  off: bf16 or zero points.
I4Plan i4_plan(int M, int N, int K, int group, bool off, size_t ws_bytes) {
    I4Plan best = {-1, 1, 1e30};
    const int cls = (group == 32 ? 2 : 0) + (off ? 1 : 0);
    for (int i = 0; i < kI4TileCount; ++i) {
        const I4Tile &t = kI4Tiles[i];
        if (t.bm > 32 && t.bm >= 2 * M) continue;  // half the tile's rows idle: a lower one does it
        const long tiles = (long)((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
        if (tiles > 8000000) continue;  // (a launch's threads: 32 bits)
        for (int ks = 1; ks <= 8; ++ks) {
            if (ks > 1 && (kWsHeader + (size_t)ks * M * N * 4 > ws_bytes || K / ks < 512 || tiles * ks > 1024 ||
                           tiles * 16 > (long)kWsHeader))
                break;
            const double rounds = (double)((tiles * ks + 255) / 256);
            double us = t.base[cls] + t.slope[cls] * rounds * K / (1024.0 * ks);
            if (ks > 1) us += 1.2 + t.split * 1e-6 * ks * M * N;
            if (us < best.us - 1e-9) best = {i, ks, us};
        }
    }
    return best;
}

hipError_t i4_run_tile(int tile, const I4GemmArgs &a, bool bf, int group, hipStream_t st) {
    switch (tile) {
    case 0: return i4_pick<KwCfg<1, 1, 1, 8, 4>>(a, bf, group, st);
    case 1: return i4_pick<KwCfg<1, 2, 1, 8, 2>>(a, bf, group, st);
    default: return i4_pick<KwCfg<2, 2, 1, 4, 2>>(a, bf, group, st);
    }
}

}  // namespace

// Workspace of a call's K split (0: none), the larger of what it takes by type.
size_t int4_gemm_ws_need(int M, int N, int K, int group) {
    int ks = 1;
    for (int off = 0; off < 2; ++off) ks = std::max(ks, i4_plan(M, N, K, group, off, ~(size_t)0).ks);
    return ks == 1 ? 0 : kWsHeader + (size_t)ks * M * N * 4;
}

// (operands 16-byte aligned; 128 K below 2^31)
ternocl_status int4_gemm_run(int dtype, const void *A, const uint32_t *B, const void *S, const void *Z, void *C,
                             const void *Other, const void *Bias, int M, int N, int K, int group, int postop, int out_f32,
                             void *ws, size_t ws_bytes, hipStream_t st) {
    const bool bf = dtype == TERNOCL_BF16;
    const I4Plan p = i4_plan(M, N, K, group, bf || Z, ws && ((uintptr_t)ws & 15) == 0 ? ws_bytes : 0);
    if (p.tile < 0) {
        set_error("M x N needs more tiles than a launch holds");
        return TERNOCL_ERR_UNSUPPORTED_SHAPE;
    }
    float *part = p.ks > 1 ? (float *)((uint8_t *)ws + kWsHeader) : nullptr;
    uint64_t *cnt = p.ks > 1 ? (uint64_t *)ws : nullptr;
    if (p.tile == kI4Shared)
        return int4_gemm_tile_run(dtype, A, B, S, Z, C, Other, Bias, M, N, K, group, postop, out_f32, p.ks, part, cnt, st);
    const I4GemmArgs a = {(const uint16_t *)A, B, (const uint16_t *)S, (const uint16_t *)Z, C, (const uint16_t *)Other, Bias,
                          M, N, K, postop, out_f32, p.ks, part, cnt};
    return launch_status(i4_run_tile(p.tile, a, bf, group, st));
}

}  // namespace tcl
