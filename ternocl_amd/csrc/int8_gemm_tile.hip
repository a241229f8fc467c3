// int8_gemm_tile.hip -- products of 8-bit integers with a scale for each token and channel
// (ternocl_int8_gemm) for tens to thousands of rows on gfx950's int8 matrix cores:
//
//   C[m,n] = ct(epi((sum_k A[m,k] B[k,n]) SB[n] SA[m])),  exact 32-bit sums
//
// A tile's waves share its rows of A through LDS, chunk j of a row at j ^ (row % 8) (j ^ (row / 2 % 8),
// which spreads 16 rows over all banks, runs the same), and take the weights, each its own columns,
// straight into fragments ([K/16][N][16]: 16 bytes a lane).  A stage is 128 rows of K: two LDS buffers, the next
// stage stored in the middle of the current one, one barrier; one to four more stages of A are on
// their way in registers (4096 x 5120 x 34816: one 720 us, two 698) and four or eight steps of
// weights.
//   * 128 x 512, eight waves side by side of 128 x 64: for each stage 2048 cycles of matrix
//     instructions a SIMD, 1152 of LDS and 1280 of L1 a CU.  256 x 256 as four waves of 128 x 128
//     840 us where this took 782, as eight waves 787.  4096 x 5120 x 34816 takes 642 to 697 us by
//     card (2.1 to 2.3 10^15 operations a second; the library's int8 product 730, its 8192^3 one 2.13
//     10^15), bound by power: the same instructions on operands of zeros take 520 us at 2.21 GHz
//     with the matrix cores busy 57% of the SIMDs' time, on normal ones 650 us at 1.5 to 1.75 GHz, busy
//     61 to 62%, timed in turn.
//   * Small tiles of tens to hundreds of rows are as long as their stages' latency (loads, LDS,
//     barrier: some 0.4 us): groups of waves split K, each with its own buffers, and add their sums
//     through LDS once (128 x 4096 x 4096 11.3 -> 8.4 us; what the epilogue reads loaded during the
//     walk 8.1).
//   * The epilogue: 32 rows of a wave's sums through LDS, so that 8 CB lanes have a row's adjacent
//     columns; the switch of its kind once a wave and the rows' loads together (4096 x 5120 x 34816 670
//     -> 642 us, 1024 x 4096 x 14336 with silu(acc) * other 92 -> 64).
#include "int8_epi.hpp"

namespace tcl {
namespace {

// A tile of WM x WN waves, each with 32 MB rows x 32 CB columns, and WK such groups of waves
// over K.  AD: stages of activations in flight (registers), PF: 32-row steps of weights in
// flight.
template <int MB_, int CB_, int WM_, int WN_, int WK_, int AD_, int PF_> struct I8Tile {
    static constexpr int MB = MB_, CB = CB_, WM = WM_, WN = WN_, WK = WK_, AD = AD_, PF = PF_, G = WM * WN;
    static constexpr int U = AD > PF / 4 ? AD : PF / 4;  // stages a turn of the walk
    static_assert(PF % 4 == 0 && U % AD == 0 && U % (PF / 4) == 0, "slots by the unrolled walk");
    static constexpr int GT = 64 * G, THREADS = GT * WK, BM = 32 * MB * WM, BN = 32 * CB * WN;
    static constexpr int AP = BM * 8 / GT;  // 16-byte chunks of A a thread and stage of 128 rows of K
    static_assert(AP * GT == BM * 8, "whole chunks");
    static constexpr int STAGE = BM * 128, ROWS = WK * 2 * STAGE;  // two buffers a group
    static constexpr int PITCH = 32 * CB + 4, SUMS = WK * G * 32 * PITCH * 4;  // a wave's 32 rows of sums
    static constexpr int LDS = ROWS > SUMS ? ROWS : SUMS;
    static_assert(LDS <= 160 * 1024, "a CU");
};

// Workgroup -> tile: XCD x (workgroups x, x + 8, ...) takes a contiguous range of `total` parts
// (`parts` a tile, from tile `first` on) in panels of up to `rows` row tiles (1024 rows),
// columns after columns, so that its 32 resident tiles of 128 x 512 are about 8 x 4 and share
// their rows and columns in its L2, and up to 1024 rows fetch the weights once.
__device__ __forceinline__ bool i8_tile_of(int id, int first, int total, int mt, int nt, int rows, int parts, int &tm, int &tn, int &part) {
    const int per = (total + 7) / 8;
    int t = (id & 7) * per + (id >> 3);
    if (t >= total || (id >> 3) >= per) return false;
    part = t % parts;
    t = first + t / parts;
    const int panel = t / (rows * nt), r = t - panel * rows * nt, pm = min(rows, mt - rows * panel);
    tn = r / pm;
    tm = rows * panel + (r - tn * pm);
    return true;
}

// The tile of rows m0 and columns n0 on, slice sl; cnt: its counter.
template <class T, bool BF16> __device__ __forceinline__ void i8_tile(const I8Args &a, uint8_t *i8_lds, int m0, int n0, int sl, uint64_t *cnt) {
    constexpr int MB = T::MB, CB = T::CB, AP = T::AP, PF = T::PF, AD = T::AD;
    const int mrows = min(T::BM, a.M - m0);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave / T::G, gw = wave % T::G, wm = gw / T::WN, wn = gw % T::WN;
    // this group's part of the slice's stages of 128 rows of K; all groups walk as many (`turns`)
    const int stages = a.K / 128, s0 = (int)((long)stages * sl / a.ksn), s1 = (int)((long)stages * (sl + 1) / a.ksn);
    const int t0 = s0 + (s1 - s0) * kg / T::WK, t1 = s0 + (s1 - s0) * (kg + 1) / T::WK, turns = (s1 - s0 + T::WK - 1) / T::WK;
    // A: chunk tid % 8 of rows tid / 8 + i GT / 8 (rows past the last read it again), to
    // position chunk ^ (row % 8) of the row's 128 bytes
    const int ar = (tid % T::GT) >> 3, ac = tid & 7;
    const int8_t *Ab = a.A + (size_t)m0 * a.K;
    uint32_t va[AP];
#pragma unroll
    for (int i = 0; i < AP; ++i) va[i] = (uint32_t)min(ar + i * (T::GT / 8), mrows - 1) * (uint32_t)a.K + 16u * ac;
    uint8_t *rows = i8_lds + kg * 2 * T::STAGE, *aw = rows + ar * 128 + ((ac ^ (ar & 7)) << 4);
    i32x4_t av[AD][AP];
    auto a_load = [&](int t, int p) __attribute__((always_inline)) {
        const int8_t *pa = Ab + 128 * (size_t)min(t, stages - 1);
#pragma unroll
        for (int i = 0; i < AP; ++i) av[p][i] = *(const i32x4_t *)(pa + va[i]);
    };
    auto a_store = [&](int p, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AP; ++i) *(i32x4_t *)(aw + buf * T::STAGE + i * (T::GT / 8) * 128) = av[p][i];
    };
    // step s of a stage: lane (c, h) holds rows 32 s + 16 h .. + 15 of K of its column and row
    uint32_t aro[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) aro[s] = (uint32_t)((wm * 32 * MB + c) * 128 + (((2 * s + h) ^ (c & 7)) << 4));
    i32x4_t af[2][MB];
    auto a_frag = [&](int buf, int s, i32x4_t f[MB]) __attribute__((always_inline)) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) f[mb] = *(const i32x4_t *)(rows + buf * T::STAGE + aro[s] + 4096 * mb);
    };
    const int nb = n0 + wn * 32 * CB;
    uint32_t vb[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) vb[cb] = ((uint32_t)h * (uint32_t)a.N + (uint32_t)min(nb + 32 * cb + c, a.N - 1)) * 16u;
    const size_t bstep = (size_t)a.N * 32;  // bytes of a step of 32 rows of K
    i32x4_t bf[PF][CB];
    auto b_load = [&](int step, int slot) __attribute__((always_inline)) {
        const int8_t *p = a.B + bstep * (size_t)min(step, 4 * stages - 1);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) bf[slot][cb] = *(const i32x4_t *)(p + vb[cb]);
    };
    // the epilogue takes 32 rows of a wave's sums at a time through LDS, so that a row's columns lie
    // on adjacent lanes; the groups' waves share the addition
    constexpr int LPR = 8 * CB, RPI = 64 / LPR, NI = 32 / RPI / T::WK;  // lanes a row, rows a pass, passes a wave
    static_assert(NI * RPI * T::WK == 32, "whole passes");
    int *red = (int *)i8_lds + gw * 32 * T::PITCH;
    const int rr = RPI * kg + lane / LPR, rc = 4 * (lane % LPR), n = nb + rc, nc = min(n, a.N - 4);
    // (few outputs a lane: what the epilogue reads is on its way while the products run)
    constexpr bool EARLY = MB == 1 && NI <= 2;
    I8Col col;
    I8Row row[NI];
    if (EARLY && a.ksn == 1) {
        col = i8_col(a, nc);
#pragma unroll
        for (int i = 0; i < NI; ++i) row[i] = i8_row(a, m0 + min(32 * wm + rr + RPI * T::WK * i, mrows - 1), nc);
    }
    i32x16_t acc[MB][CB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[mb][cb] = i32x16_t{};
    // stage t: slots by its place p in a turn, LDS buffer `buf`
    auto stage = [&](int t, int p, int buf) __attribute__((always_inline)) {
        const int next = buf ^ 1;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int slot = (4 * p + s) % PF;
            if (s == 2) {  // the next stage's rows, then the one barrier of a stage
                a_store((p + 1) % AD, next);
                a_load(t + 1 + AD, (p + 1) % AD);
            }
            if (s < 3) a_frag(buf, s + 1, af[(s + 1) & 1]);
            if (s == 3) {
                __syncthreads();
                a_frag(next, 0, af[0]);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (T::WK == 1 || t < t1)  // (uniform; a group may have a stage less)
#pragma unroll
                for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)  // (columns as the matrix' rows: a lane gets four adjacent ones)
                        acc[mb][cb] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[slot][cb], af[s & 1][mb], acc[mb][cb], 0, 0, 0);
            b_load(4 * t + s + PF, slot);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int p = 0; p < AD; ++p) a_load(t0 + p, p);
#pragma unroll
    for (int s = 0; s < PF; ++s) b_load(4 * t0 + s, s);
    __builtin_amdgcn_sched_barrier(0);
    a_store(0, 0);
    a_load(t0 + AD, 0);
    __syncthreads();
    a_frag(0, 0, af[0]);
    int buf = 0, i = 0;
    for (; i + T::U <= turns; i += T::U)
#pragma unroll
        for (int p = 0; p < T::U; ++p) {
            stage(t0 + i + p, p, buf);
            buf ^= 1;
        }
#pragma unroll
    for (int p = 0; p < T::U - 1; ++p) {
        if (i + p >= turns) break;
        stage(t0 + i + p, p, buf);
        buf ^= 1;
    }
    __syncthreads();
    auto blocks = [&](auto emit) __attribute__((always_inline)) {  // emit(first row, its NI sums, RPI WK rows apart)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *(i32x4_t *)(red + kg * T::G * 32 * T::PITCH + c * T::PITCH + 32 * cb + 8 * j + 4 * h) =
                        i32x4_t{acc[mb][cb][4 * j], acc[mb][cb][4 * j + 1], acc[mb][cb][4 * j + 2], acc[mb][cb][4 * j + 3]};
            if constexpr (T::WK > 1) {
                __syncthreads();
            } else {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            i32x4_t s[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int *p = red + (rr + RPI * T::WK * i) * T::PITCH + rc;
                s[i] = *(const i32x4_t *)p;
#pragma unroll
                for (int k = 1; k < T::WK; ++k) s[i] += *(const i32x4_t *)(p + k * T::G * 32 * T::PITCH);
            }
            emit((wm * MB + mb) * 32 + rr, s);
            if constexpr (T::WK > 1) {
                if (mb < MB - 1) __syncthreads();
            } else {
                __builtin_amdgcn_wave_barrier();
            }
        }
    };
    if (a.ksn == 1) {
        if constexpr (!EARLY) col = i8_col(a, nc);
        epi_dispatch(a.postop, a.out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
            blocks([&](int m, const i32x4_t *s) __attribute__((always_inline)) {
                if constexpr (!EARLY)
#pragma unroll
                    for (int i = 0; i < NI; ++i) row[i] = i8_row(a, m0 + min(m + RPI * T::WK * i, mrows - 1), nc);
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    if (m + RPI * T::WK * i < mrows && n < a.N)
                        i8_out<BF16, decltype(P_)::value, decltype(F_)::value>(a, m0 + m + RPI * T::WK * i, n, s[i], col, row[i]);
            });
        });
        return;
    }
    blocks([&](int m, const i32x4_t *s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (m + RPI * T::WK * i < mrows && n < a.N) i8_part_store(a.part + ((size_t)sl * a.M + m0 + m + RPI * T::WK * i) * a.N + n, s[i]);
    });
    // the last of the tile's slices adds them
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    uint32_t *flag = (uint32_t *)i8_lds;
    if (wave == 0) {
        const bool last = kw_arrive(cnt, a.ksn, lane);
        if (lane == 0) *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
    epi_dispatch(a.postop, a.out_f32, [&](auto P_, auto F_) __attribute__((always_inline)) {
        for (int i = tid; i < mrows * (T::BN / 4); i += T::THREADS) {
            const int m = m0 + i / (T::BN / 4), nn = n0 + 4 * (i % (T::BN / 4));
            if (nn >= a.N) continue;
            const I8Col cl = i8_col(a, nn);
            const I8Row rw = i8_row(a, m, nn);
            const int *p = a.part + (size_t)m * a.N + nn;
            i32x4_t s = i8_part_load(p);
            for (int k = 1; k < a.ksn; ++k) s += i8_part_load(p + (size_t)k * a.M * a.N);
            i8_out<BF16, decltype(P_)::value, decltype(F_)::value>(a, m, nn, s, cl, rw);
        }
    });
}

template <class T, bool BF16> __global__ void __launch_bounds__(T::THREADS) k_int8_gemm_tile(const I8Args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_lds[];
    const int mt = (a.M + T::BM - 1) / T::BM, nt = (a.N + T::BN - 1) / T::BN;
    int tm, tn, sl;
    if (!i8_tile_of(blockIdx.x, 0, mt * nt * a.ksn, mt, nt, 1024 / T::BM, a.ksn, tm, tn, sl)) return;  // (whole workgroup)
    i8_tile<T, BF16>(a, i8_lds, tm * T::BM, tn * T::BN, sl, a.ksn > 1 ? a.cnt + 2 * ((size_t)tm * nt + tn) : nullptr);
}

// The first `full` tiles as T's (a multiple of 256, a workgroup a CU), those of the last partial
// round as two of H's each, half as wide: 4096 x 5120 x 34816 (8.5 rounds) 702 -> 670 us.
template <class T, class H, bool BF16> __global__ void __launch_bounds__(T::THREADS) k_int8_gemm_tail(const I8Args a, int full) {
    static_assert(H::BM == T::BM && 2 * H::BN == T::BN && H::THREADS == T::THREADS, "halves");
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_lds[];
    const int mt = (a.M + T::BM - 1) / T::BM, nt = (a.N + T::BN - 1) / T::BN;
    int tm, tn, sl, id = blockIdx.x;
    if (id < full) {
        if (i8_tile_of(id, 0, full, mt, nt, 1024 / T::BM, 1, tm, tn, sl)) i8_tile<T, BF16>(a, i8_lds, tm * T::BM, tn * T::BN, 0, nullptr);
    } else if (i8_tile_of(id - full, full, 2 * (mt * nt - full), mt, nt, 1024 / T::BM, 2, tm, tn, sl)) {
        const int n0 = tn * T::BN + sl * H::BN;
        if (n0 < a.N) i8_tile<H, BF16>(a, i8_lds, tm * T::BM, n0, 0, nullptr);
    }
}

template <class T> hipError_t i8_tile_launch(int dtype, const I8Args &a, hipStream_t st) {
    const long tiles = (long)((a.M + T::BM - 1) / T::BM) * ((a.N + T::BN - 1) / T::BN) * a.ksn;
    const dim3 g((unsigned)(8 * ((tiles + 7) / 8)));
    auto go = [&](auto k) { hipLaunchKernelGGL(k, g, dim3(T::THREADS), T::LDS, st, a); };
    if (dtype == TERNOCL_BF16) go(k_int8_gemm_tile<T, true>);
    else go(k_int8_gemm_tile<T, false>);
    return hipGetLastError();
}

// 128 x 512 tiles, the last partial round of up to 128 as halves.
hipError_t i8_wide_launch(int dtype, const I8Args &a, hipStream_t st) {
    typedef I8Tile<4, 2, 1, 8, 1, 2, 4> T;
    typedef I8Tile<4, 1, 1, 8, 1, 2, 4> H;
    const long tiles = (long)((a.M + T::BM - 1) / T::BM) * ((a.N + T::BN - 1) / T::BN);
    const int rem = (int)(tiles % 256);
    if (a.ksn > 1 || tiles < 256 || rem == 0 || rem > 128) return i8_tile_launch<T>(dtype, a, st);
    const int full = (int)(tiles - rem);
    const dim3 g((unsigned)(full + 8 * ((2 * rem + 7) / 8)));
    constexpr int lds = T::LDS > H::LDS ? T::LDS : H::LDS;
    auto go = [&](auto k) { hipLaunchKernelGGL(k, g, dim3(T::THREADS), lds, st, a, full); };
    if (dtype == TERNOCL_BF16) go(k_int8_gemm_tail<T, H, true>);
    else go(k_int8_gemm_tail<T, H, false>);
    return hipGetLastError();
}

}  // namespace

hipError_t int8_tile_run(int tile, int dtype, const I8Args &a, hipStream_t st) {
    switch (tile) {
    case 0: return i8_tile_launch<I8Tile<1, 1, 1, 2, 4, 2, 8>>(dtype, a, st);
    case 1: return i8_tile_launch<I8Tile<1, 1, 1, 4, 1, 2, 8>>(dtype, a, st);
    case 2: return i8_tile_launch<I8Tile<1, 1, 1, 4, 2, 2, 8>>(dtype, a, st);
    case 3: return i8_tile_launch<I8Tile<2, 1, 1, 4, 1, 2, 8>>(dtype, a, st);
    case 4: return i8_tile_launch<I8Tile<2, 1, 1, 4, 2, 4, 8>>(dtype, a, st);
    case 5: return i8_tile_launch<I8Tile<2, 1, 1, 8, 1, 4, 8>>(dtype, a, st);
    case 6: return i8_tile_launch<I8Tile<4, 2, 1, 4, 1, 1, 4>>(dtype, a, st);
    default: return i8_wide_launch(dtype, a, st);
    }
}

}  // namespace tcl
