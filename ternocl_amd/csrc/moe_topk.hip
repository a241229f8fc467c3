// moe_topk.hip -- routing to experts: the ids and weights that the MoE layers take,
// from the router's logits (ternocl_moe_topk).
//
//   s = softmax(l) or 1 / (1 + e^-l), v = s + bias; the topk_group groups with the
//   largest sums of their group_best largest v stay; ids = the topk largest v, RW = s
//   of those (renormalised), times scale.
//
// L lanes take a token (64 / L tokens a wave), lane i of them holding experts i, i + L, ...
// With L = 16 (up to 16 choices, 15 with a bias) the values that can be among the topk go to
// a list that is ranked at once; with L = 64 topk rounds pick the largest value (a maximum
// over the lanes), the lowest index that has it (a minimum over those), and drop it, at
// three times the instructions (T = 1 E = 64, 8 choices 4.0 against 3.1 us, T = 4000 E =
// 128 7.0 against 4.3).
//   * Without a bias the logits themselves order the experts -- softmax and the sigmoid
//     rise with them, and in exact arithmetic only equal logits give equal scores -- so the
//     rounds compare fp32 logits, exactly.
//   * With a bias (and for the sums of two that value a group) v is computed in fp32.
//     Where two picks in a row are closer than its error (tk_margin) tells apart, the picks
//     up to the next wider gap are ranked by their 64-bit values; where there is none before
//     the list's end, where groups kept and dropped may be the other way round (TkGroup), or a
//     value is NaN or +inf, the token is done again with 64-bit values (tk_exact, the whole
//     wave).  Of N(0, 1.5) logits over 256 experts,
//     sigmoid scores, about 1 token in 2000 has close picks, 1 in 16000 close groups.
//
// What bounds it: launch and latency for few tokens (T = 1 E = 128 3.2 us, T = 2048 E = 64 4.0
// us).  For many, the latency of a wave's dependent steps: T = 16384 E = 256 fp32, 8 of 4 of 8
// groups with a bias, 12.4 us, 15 to 17.7 where some token takes 64 bits; a wave's time is 18% VALU,
// 48% waits for loads and LDS, 23% waits for issue, and the SIMDs' VALU is busy 28% of it.  Without
// either, bf16: 7.2 us (17%, 58%, 18%).
#include "common.hpp"

#include <algorithm>

namespace tcl {
namespace {

typedef unsigned long long u64;

// Keys: larger value, larger key; -0 as +0, -inf 0, NaN all ones.
__device__ __forceinline__ u64 tk_key(double v) {
    const u64 b = (u64)__double_as_longlong(v + 0.0);
    if (v != v) return ~0ull;
    if (b == 0xfff0000000000000ull) return 0ull;
    return b ^ ((u64)((long long)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double tk_value(u64 k) {  // of a key that is neither 0 nor a NaN's
    return __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
}

template <int M> __device__ __forceinline__ uint32_t tk_xor(uint32_t v, int lane) {
    return __float_as_uint(lane_xor<M>(__uint_as_float(v), lane));
}
template <int M> __device__ __forceinline__ u64 tk_xor(u64 v, int lane) {
    return (u64)tk_xor<M>((uint32_t)v, lane) | ((u64)tk_xor<M>((uint32_t)(v >> 32), lane) << 32);
}
template <class K> __device__ __forceinline__ K tk_max(K v, int lane) {
    v = max(v, tk_xor<1>(v, lane));
    v = max(v, tk_xor<2>(v, lane));
    v = max(v, tk_xor<4>(v, lane));
    v = max(v, tk_xor<8>(v, lane));
    v = max(v, tk_xor<16>(v, lane));
    return max(v, tk_xor<32>(v, lane));
}
struct TkArgs {
    const void *logits;
    const float *bias;
    int *ids;
    void *RW;
    long ld;
    int ltype, T, E, topk, wtype, score, n_group, topk_group, group_best, renorm;
    float scale;
};

constexpr int kTkWaves = 4;

// Twice the error of an fp32 value v of a choice: two values further apart are in order.
// A sigmoid: its argument's two roundings (times s (1 - s) |l|, below 0.23), the
// exponential's and the reciprocal's last places, below 2^-22 together.  A softmax term:
// 37 additions of its row's sum at most, each term's argument (E |l - max| <= ln 512) and
// last place, below 56 x 2^-24 < 2^-18 of the row's largest.  The bias's addition: 2^-24 |v|.
// s: twice the scores' part, kSigmoidError or 2^-17 of the largest term.
constexpr float kSigmoidError = 0x1p-21f;
__device__ __forceinline__ float tk_margin(float v, float s) { return s + 0x1p-22f * fabsf(v); }

// A value's bits as an integer in the order of the values (-0 as +0), kNone for -inf; and
// back.  (Integer comparisons: fmaxf quiets its operands first, twice the instructions.)
constexpr int kNone = -0x7fffffff - 1;
__device__ __forceinline__ int tk_int(float v) {
    const int b = __float_as_int(v + 0.0f);
    return v == -__builtin_inff() ? kNone : b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float tk_float(int k) {
    return k == kNone ? -__builtin_inff() : __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}

// A group's value, and the error of that: its scores' (err, tk_margin's s) and, of its one or
// two additions of a bias and of their sum, 2^-24 each of the terms, which may be far larger
// than the sum (1.25 times that: of the error's own roundings).  b2: kNone where one value counts.
struct TkGroup {
    int value;
    float error;
};
__device__ __forceinline__ TkGroup tk_group(int b1, int b2, float err) {
    const float x = tk_float(b1), y = b2 == kNone ? 0.0f : tk_float(b2);
    // (of two values above -inf the sum is no -inf, no empty group's value, in 64 bits)
    constexpr int kLowest = (int)0x80800000u;  // tk_int(-FLT_MAX)
    return {max(tk_int(x + y), min(b2, kLowest)), __builtin_fmaf(fabsf(y), 0x1.4p-23f, __builtin_fmaf(fabsf(x), 0x1.4p-23f, err))};
}
// Whether a group may be on the other side of mid, a value between the least kept and the
// largest dropped one: where none is, exactly those kept are the largest.
__device__ __forceinline__ bool tk_group_close(int value, float error, float mid) {
    return value != kNone && !(fabsf(tk_float(value) - mid) > error);
}

// Sum, maximum, minimum over the L lanes of a token
template <int L, class V, class Op> __device__ __forceinline__ V tk_lanes(V v, int lane, Op op) {
    auto x = [&](auto m) __attribute__((always_inline)) {
        if constexpr (std::is_same_v<V, int>) v = op(v, __float_as_int(lane_xor<decltype(m)::value>(__int_as_float(v), lane)));
        else v = op(v, lane_xor<decltype(m)::value>(v, lane));
    };
    x(std::integral_constant<int, 1>{});
    x(std::integral_constant<int, 2>{});
    x(std::integral_constant<int, 4>{});
    x(std::integral_constant<int, 8>{});
    if constexpr (L == 64) {
        x(std::integral_constant<int, 16>{});
        x(std::integral_constant<int, 32>{});
    }
    return v;
}
__device__ __forceinline__ float tk_fmax2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float tk_add2(float a, float b) { return a + b; }
__device__ __forceinline__ int tk_imax2(int a, int b) { return max(a, b); }
__device__ __forceinline__ int tk_imin2(int a, int b) { return min(a, b); }
template <int L> __device__ __forceinline__ double tk_dsum(double v) {
#pragma unroll
    for (int d = 1; d < L; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ float tk_logit(const TkArgs &a, int t, int e) {
    const size_t i = (size_t)t * a.ld + e;
    if (a.ltype == TERNOCL_FP32) return ((const float *)a.logits)[i];
    const uint32_t h = ((const uint16_t *)a.logits)[i];
    return a.ltype == TERNOCL_BF16 ? dt2f<true>(h) : dt2f<false>(h);
}
// The softmax sum of token t in 64 bits, relative to its largest logit mx: L lanes, the logits
// read again (the double exponentials of 32 experts a lane would hold it at 2 waves a SIMD)
template <int L> __device__ __forceinline__ double tk_total(const TkArgs &a, int t, int sub, float mx) {
    double p = 0.0;
#pragma unroll 4
    for (int e = sub; e < a.E; e += L) {
        const float y = tk_logit(a, t, e);
        p += y == -__builtin_inff() ? 0.0 : exp((double)y - (double)mx);
    }
    return tk_dsum<L>(p);
}
// Logits e0, e0 + step, ... of token t (-inf past the last expert), all loads in flight
template <int n> __device__ __forceinline__ void tk_logits(const TkArgs &a, int t, int e0, int step, float l[n]) {
    const size_t row = (size_t)t * a.ld;
    if (a.ltype == TERNOCL_FP32) {
#pragma unroll
        for (int j = 0; j < n; ++j) l[j] = ((const float *)a.logits)[row + min(e0 + j * step, a.E - 1)];
    } else {
        uint16_t h[n];
#pragma unroll
        for (int j = 0; j < n; ++j) h[j] = ((const uint16_t *)a.logits)[row + min(e0 + j * step, a.E - 1)];
        if (a.ltype == TERNOCL_BF16) {
#pragma unroll
            for (int j = 0; j < n; ++j) l[j] = dt2f<true>(h[j]);
        } else {
#pragma unroll
            for (int j = 0; j < n; ++j) l[j] = dt2f<false>(h[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < n; ++j) l[j] = e0 + j * step < a.E ? l[j] : -__builtin_inff();
}

// n values of 2 or 4 bytes each that lie together, in loads of 16 bytes or all of them (p
// aligned to that)
template <int bytes, int n> __device__ __forceinline__ void tk_load(const void *p, uint32_t o[n]) {
    constexpr int total = bytes * n, step = total < 16 ? total : 16;
    uint32_t w[(total + 3) / 4];
#pragma unroll
    for (int i = 0; i < total / step; ++i) {
        const uint8_t *q = (const uint8_t *)p + 16 * i;
        if constexpr (step == 16) {
            const uint4 v = *(const uint4 *)q;
            __builtin_memcpy(w + 4 * i, &v, 16);
        } else if constexpr (step == 8) {
            const uint2 v = *(const uint2 *)q;
            __builtin_memcpy(w, &v, 8);
        } else if constexpr (step == 4) {
            w[0] = *(const uint32_t *)q;
        } else {
            w[0] = *(const uint16_t *)q;
        }
    }
#pragma unroll
    for (int j = 0; j < n; ++j) o[j] = bytes == 4 ? w[j] : (w[j / 2] >> (16 * (j & 1))) & 0xffffu;
}
// Logits e0 .. e0 + n - 1 of token t (all of them experts, or none: -inf)
template <int n> __device__ __forceinline__ void tk_logits_together(const TkArgs &a, int t, int e0, float l[n]) {
    const size_t i = (size_t)t * a.ld + (e0 < a.E ? e0 : 0);
    uint32_t w[n];
    if (a.ltype == TERNOCL_FP32) {
        tk_load<4, n>((const float *)a.logits + i, w);
#pragma unroll
        for (int j = 0; j < n; ++j) l[j] = __uint_as_float(w[j]);
    } else {
        tk_load<2, n>((const uint16_t *)a.logits + i, w);
        if (a.ltype == TERNOCL_BF16) {
#pragma unroll
            for (int j = 0; j < n; ++j) l[j] = dt2f<true>(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < n; ++j) l[j] = dt2f<false>(w[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < n; ++j) l[j] = e0 < a.E ? l[j] : -__builtin_inff();
}

// The outputs of slot r of token t: expert id (-1: none) with logit l.  mx, total: the
// row's largest logit and its softmax sum; L lanes hold the token's slots.
template <int L>
__device__ __forceinline__ void tk_write(const TkArgs &a, int t, int r, int id, float l, float mx, double total, bool on) {
    const bool live = r < a.topk && id >= 0;
    double wt;
    if (a.score == 0) wt = exp((double)l - (double)mx) / total;
    else wt = 1.0 / (1.0 + exp(-(double)l));
    if (!live) wt = 0.0;
    if (a.renorm) {
        const double sum = tk_dsum<L>(wt);
        wt = sum == 0.0 ? 0.0 : wt / sum;
    }
    wt *= (double)a.scale;
    if (!on || r >= a.topk) return;
    const size_t o = (size_t)t * a.topk + r;
    a.ids[o] = id;
    const float f = live ? (float)wt : 0.0f;
    if (a.wtype == TERNOCL_FP32) ((float *)a.RW)[o] = f;
    else ((uint16_t *)a.RW)[o] = (uint16_t)(a.wtype == TERNOCL_BF16 ? f2dt<true>(f) : f2dt<false>(f));
}

// Token t by a whole wave, compared by 64-bit keys in the order of the values (0: never
// chosen, all ones: NaN).  gkey: the wave's LDS, 64 VX keys.
template <int VX> __device__ __forceinline__ void tk_exact(const TkArgs &a, int t, int lane, u64 *gkey) {
    const bool grouped = a.topk_group < a.n_group;
    const int e0 = VX * lane;
    float l[VX];
    double s[VX], p = 0.0;
    tk_logits<VX>(a, t, e0, 1, l);
    float mx = l[0];  // (NaN passed over: it reaches the sum)
#pragma unroll
    for (int j = 1; j < VX; ++j) mx = fmaxf(mx, l[j]);
    mx = tk_lanes<64>(mx, lane, tk_fmax2);
#pragma unroll
    for (int j = 0; j < VX; ++j) {
        if (a.score == 0) s[j] = l[j] == -__builtin_inff() ? 0.0 : exp((double)l[j] - (double)mx);
        else s[j] = 1.0 / (1.0 + exp(-(double)l[j]));
        p += s[j];
    }
    const double total = a.score == 0 ? tk_dsum<64>(p) : 1.0;
    u64 key[VX];
#pragma unroll
    for (int j = 0; j < VX; ++j) {
        s[j] = s[j] / total;
        const double v = a.bias ? s[j] + (double)a.bias[min(e0 + j, a.E - 1)] : (double)l[j];
        key[j] = l[j] == -__builtin_inff() ? 0 : tk_key(v);
    }
    if (grouped) {
        // a group's value as a key of its own (0: none to choose), lane g for group g
        const int per = a.E / a.n_group;
#pragma unroll
        for (int j = 0; j < VX; ++j) gkey[e0 + j] = a.group_best == 2 && !a.bias ? (key[j] ? tk_key(s[j]) : 0) : key[j];
        __builtin_amdgcn_wave_barrier();  // (the wave's own LDS, in order)
        u64 k1 = 0, k2 = 0;
        if (lane < a.n_group)
#pragma unroll 8
            for (int i = 0; i < per; ++i) {
                const u64 k = gkey[lane * per + i];
                k2 = max(k2, min(k, k1));
                k1 = max(k1, k);
            }
        u64 gv = k1;
        if (a.group_best == 2 && k1 != 0 && k1 != ~0ull && k2 != 0) gv = tk_key(tk_value(k1) + tk_value(k2));
        // kept: fewer than topk_group groups come before it
        int before = 0;
        for (int g = 0; g < a.n_group; ++g) {
            const u64 ov = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)gv, g) |
                           ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(gv >> 32), g) << 32);
            before += ov > gv || (ov == gv && g < lane);
        }
        const u64 kept = __ballot(before < a.topk_group);
#pragma unroll
        for (int j = 0; j < VX; ++j)
            if (!((kept >> (min(e0 + j, a.E - 1) / per)) & 1)) key[j] = 0;
    }
    int id = -1;
    float lv = 0.0f;
    for (int r = 0; r < a.topk; ++r) {
        u64 best = key[0];
#pragma unroll
        for (int j = 1; j < VX; ++j) best = max(best, key[j]);
        const u64 m = tk_max(best, lane);
        if (m == 0) break;  // (uniform)
        const int from = __builtin_ctzll(__ballot(best == m));
        int at = 0;
        float x = 0.0f;
#pragma unroll
        for (int j = VX - 1; j >= 0; --j)
            if (key[j] == m) {
                at = j;
                x = l[j];
            }
        at = lane == from ? at : -1;
#pragma unroll
        for (int j = 0; j < VX; ++j)
            if (at == j) key[j] = 0;
        const int e = __builtin_amdgcn_readlane(e0 + at, from);
        x = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), from));
        if (lane == r) {
            id = e;
            lv = x;
        }
    }
    tk_write<64>(a, t, lane, id, lv, mx, total, true);
}

// GROUPED: 0 no choice of groups; 1 any groups; 2 groups of whole lanes, a power of two of
// them: lane i holds experts i VPL .. + VPL - 1 then.  Many tokens of 257 experts and more are
// four waves a SIMD only in 128 registers (up to 216 without the bound: that call 33.4 -> 23.6
// us, E = 512 10 choices without a bias 14.0 -> 11.5).
template <int L, int VPL, int GROUPED> __global__ void __launch_bounds__(64 * kTkWaves, L == 16 && VPL == 32 ? 4 : 1) k_moe_topk(const TkArgs a) {
    constexpr int TPW = 64 / L, VX = VPL * L / 64 > 0 ? VPL * L / 64 : 1;
    // a wave's values [tokens][L VPL] while groups are valued; its tokens' lists [32] and
    // picks in order [16]; tk_exact's keys
    __shared__ __attribute__((aligned(16))) u64 space[kTkWaves][std::max({(TPW * L * VPL + 1) / 2, 64 * VX, L == 16 ? 192 : 0})];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = lane % L, tok = lane / L;
    const int t0 = (blockIdx.x * kTkWaves + w) * TPW, t = t0 + tok;
    if (t0 >= a.T) return;  // (whole wave; no barrier follows)
    const bool on = t < a.T;
    const int tc = min(t, a.T - 1);
    const float ninf = -__builtin_inff();
    float l[VPL], bias[VPL];
    auto load_bias = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) bias[j] = a.bias[min(sub + L * j, a.E - 1)];
    };
    int v[VPL];  // what experts are chosen by (tk_int)
    constexpr int E0 = GROUPED == 2 ? VPL : 1, ES = GROUPED == 2 ? 1 : L;  // lane i's experts E0 i + ES j
    if constexpr (GROUPED == 2) {
        tk_logits_together<VPL>(a, tc, E0 * sub, l);
        if (a.bias) {
            uint32_t w[VPL];
            tk_load<4, VPL>(a.bias + (E0 * sub < a.E ? E0 * sub : 0), w);
#pragma unroll
            for (int j = 0; j < VPL; ++j) bias[j] = __uint_as_float(w[j]);
        }
    } else {
        tk_logits<VPL>(a, tc, sub, L, l);
        if (VPL < 32 && a.bias) load_bias();
    }
    bool odd = false;  // this token needs 64 bits
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        odd |= !(l[j] < __builtin_inff());
        v[j] = tk_int(l[j]);
    }
    float mx = ninf;
    double total = 1.0;
    const bool two = GROUPED != 0 && a.group_best == 2;
    if (a.score == 0) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) mx = fmaxf(mx, l[j]);
        mx = tk_lanes<L>(mx, lane, tk_fmax2);
    }
    if (a.score == 0 && !a.renorm) {
        // The weights' denominator: in 64 bits for fp32 weights, in 32 bits for 16-bit ones, where its
        // error (tk_margin's count: 2^-18 of the sum) is 1/64 of an fp16's rounding, 1/512 of a bf16's.
        // (64 bits for all: T = 16384 E = 256 8.3 -> 14.6 us, T = 2048 E = 64 3.6 -> 4.6; 64 bits only where
        // the 32-bit sum leaves a rounding open 12.1 and 4.7)
        if (a.wtype == TERNOCL_FP32) {
            total = tk_total<L>(a, tc, sub, mx);
        } else {
            float p = 0.0f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) p += l[j] == ninf ? 0.0f : __builtin_amdgcn_exp2f((l[j] - mx) * 1.44269504088896341f);
            total = (double)tk_lanes<L>(p, lane, tk_add2);
        }
    }
    float s[VPL];  // the scores, where choices are made by them
    float err = kSigmoidError;  // (tk_margin)
    if (a.bias || two) {
        float p = 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if (a.score == 0) s[j] = l[j] == ninf ? 0.0f : __builtin_amdgcn_exp2f((l[j] - mx) * 1.44269504088896341f);
            else s[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -1.44269504088896341f));
            p += s[j];
        }
        if (a.score == 0) {
            const float r = 1.0f / tk_lanes<L>(p, lane, tk_add2);
#pragma unroll
            for (int j = 0; j < VPL; ++j) s[j] *= r;
            err = 0x1p-17f * r;
        }
        if (a.bias) {
            if constexpr (VPL >= 32 && GROUPED != 2) {  // (registers)
                __builtin_amdgcn_sched_barrier(0);
                load_bias();
            }
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const float x = s[j] + bias[j];
                v[j] = l[j] == ninf ? kNone : tk_int(x);
                odd |= !(x < __builtin_inff());
            }
        }
    }
    if constexpr (GROUPED == 2) {
        // a group's largest two: a lane's own, then over its lanes
        const int lpg = a.E / a.n_group / VPL, g = sub / lpg;
        int b1 = kNone, b2 = kNone;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int y = two && !a.bias ? (v[j] == kNone ? kNone : tk_int(s[j])) : v[j];
            b2 = max(b2, min(y, b1));
            b1 = max(b1, y);
        }
        auto merge = [&](auto m) __attribute__((always_inline)) {
            if (lpg <= decltype(m)::value) return;  // (uniform)
            const int o1 = __float_as_int(lane_xor<decltype(m)::value>(__int_as_float(b1), lane));
            const int o2 = __float_as_int(lane_xor<decltype(m)::value>(__int_as_float(b2), lane));
            b2 = max(min(b1, o1), max(b2, o2));
            b1 = max(b1, o1);
        };
        merge(std::integral_constant<int, 1>{});
        merge(std::integral_constant<int, 2>{});
        merge(std::integral_constant<int, 4>{});
        merge(std::integral_constant<int, 8>{});
        if constexpr (L == 64) {
            merge(std::integral_constant<int, 16>{});
            merge(std::integral_constant<int, 32>{});
        }
        const TkGroup gr = tk_group(b1, two ? b2 : kNone, err);
        const int gv = gr.value;
        // kept: fewer than topk_group groups come before it
        int *val = (int *)space[w] + tok * L;
        val[g] = gv;  // (by each of its lanes)
        __builtin_amdgcn_wave_barrier();  // (the wave's own LDS, in order)
        int before = 0;
        for (int i = 0; i < a.n_group; i += 4) {
            const int4 o = *(const int4 *)(val + i);
            before += o.x > gv || (o.x == gv && i < g);
            before += i + 1 < a.n_group && (o.y > gv || (o.y == gv && i + 1 < g));
            before += i + 2 < a.n_group && (o.z > gv || (o.z == gv && i + 2 < g));
            before += i + 3 < a.n_group && (o.w > gv || (o.w == gv && i + 3 < g));
        }
        const bool keep = before < a.topk_group, real = g < a.n_group;
        if (a.bias || two) {
            const float lo = tk_float(tk_lanes<L>(real && keep ? gv : 0x7fffffff, lane, tk_imin2));
            const float hi = tk_float(tk_lanes<L>(real && !keep ? gv : kNone, lane, tk_imax2));
            odd |= real && tk_group_close(gv, gr.error, 0.5f * lo + 0.5f * hi);
        }
#pragma unroll
        for (int j = 0; j < VPL; ++j) v[j] = keep ? v[j] : kNone;
        if constexpr (L == 16) {
            // dealt to the lanes as without groups: kept ones fill a few lanes otherwise
            int *deal = (int *)space[w] + tok * L * VPL;
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < VPL; j += 4) *(int4 *)(deal + VPL * sub + j) = make_int4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < VPL; ++j) v[j] = deal[sub + L * j];
        }
    }
    if constexpr (GROUPED == 1) {
        const int per = a.E / a.n_group;
        int *val = (int *)space[w] + tok * L * VPL;
#pragma unroll
        for (int j = 0; j < VPL; ++j) val[sub + L * j] = two && !a.bias ? (v[j] == kNone ? kNone : tk_int(s[j])) : v[j];
        __builtin_amdgcn_wave_barrier();  // (the wave's own LDS, in order)
        // lane g + part 2^sh values part `part` of group g (of groups g, g + L, ... where they are
        // more than the lanes): the largest one or two of every parts-th member, from another
        // one on in each group and token, for the banks.  (T = 16384, one of two groups of 196,
        // 4 choices: a lane a group 43.6, this 33.4 us)
        constexpr int GPL = 64 / L;
        int gv[GPL];
        TkGroup gr[GPL];
        const int sh = min(32 - __builtin_clz(a.n_group - 1), L == 64 ? 6 : 4), parts = L >> sh;  // (n_group > 1)
        const int g0 = sub & ((1 << sh) - 1), part = sub >> sh, members = (per - part + parts - 1) / parts;
#pragma unroll
        for (int k = 0; k < GPL; ++k) {
            const int g = g0 + L * k;
            int b1 = kNone, b2 = kNone;
            if (L * k < a.n_group) {  // (uniform)
                const int *x = val + min(g, a.n_group - 1) * per;
                const int begin = min(part, per - 1);
                int i = begin + parts * max(min(g + tok, members - 1), 0);
                for (int n = 0; n * parts < per; n += 4) {
                    int o[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        o[u] = x[i];
                        i = i + parts < per ? i + parts : begin;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int y = n + u < members ? o[u] : kNone;
                        b2 = max(b2, min(y, b1));
                        b1 = max(b1, y);
                    }
                }
            }
            auto merge = [&](auto m) __attribute__((always_inline)) {
                if (decltype(m)::value < 1 << sh) return;  // (uniform)
                const int o1 = __float_as_int(lane_xor<decltype(m)::value>(__int_as_float(b1), lane));
                const int o2 = __float_as_int(lane_xor<decltype(m)::value>(__int_as_float(b2), lane));
                b2 = max(min(b1, o1), max(b2, o2));
                b1 = max(b1, o1);
            };
            if (k == 0) {  // (further groups: parts is 1)
                merge(std::integral_constant<int, 2>{});
                merge(std::integral_constant<int, 4>{});
                merge(std::integral_constant<int, 8>{});
                if constexpr (L == 64) {
                    merge(std::integral_constant<int, 16>{});
                    merge(std::integral_constant<int, 32>{});
                }
            }
            gr[k] = {kNone, 0.0f};
            if (k == 0 || L * k < a.n_group) gr[k] = tk_group(b1, two ? b2 : kNone, err);  // (past the last group: that again)
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < GPL; ++k)
            if (part == 0 && g0 + L * k < a.n_group) val[g0 + L * k] = gr[k].value;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < GPL; ++k) gv[k] = sub + L * k < a.n_group ? val[sub + L * k] : kNone;
        // kept: fewer than topk_group groups come before it
        int before[GPL] = {};
#pragma unroll 4
        for (int g = 0; g < a.n_group; ++g) {
            const int o = val[g];
#pragma unroll
            for (int k = 0; k < GPL; ++k) before[k] += o > gv[k] || (o == gv[k] && g < sub + L * k);
        }
        u64 kept = 0;
        int low = 0x7fffffff, high = kNone;  // the least kept, the largest dropped
#pragma unroll
        for (int k = 0; k < GPL; ++k) {
            const bool keep = before[k] < a.topk_group && sub + L * k < a.n_group;
            const u64 b = __ballot(keep);
            kept |= L == 64 ? b : ((b >> (L * tok)) & ((1ull << (L & 63)) - 1)) << (L * k);
            if (keep) low = min(low, gv[k]);
            else high = max(high, gv[k]);
        }
        if (a.bias || two) {
            const float lo = tk_float(tk_lanes<L>(low, lane, tk_imin2)), hi = tk_float(tk_lanes<L>(high, lane, tk_imax2));
#pragma unroll
            for (int k = 0; k < GPL; ++k)
                if (k == 0 || L * k < a.n_group) odd |= tk_group_close(gr[k].value, gr[k].error, 0.5f * lo + 0.5f * hi);
        }
        // (experts past E: none anyway)
        const float inv = 1.0f / (float)per;  // (e + 1/2) / per, e < 512: 2^-10 or more from a whole number
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (!((kept >> ((int)__builtin_fmaf((float)sub, inv, ((float)(L * j) + 0.5f) * inv) & 63)) & 1)) v[j] = kNone;
    }
    bool close = false;  // picks to be put in order by their 64-bit values (alike in a token's lanes)
    int id = -1, pick = kNone;  // lane r: the r-th largest value's expert, and the value
    if constexpr (L == 16) {
        // The need-th largest of the 16 lanes' maxima is a bound that at least need values
        // reach (15 or so of 256 for need = 10): those go to a list, whose 64-bit keys (value,
        // lowest index) are ranked each against all.  Where more than kList reach it (for need =
        // 14 every second time, for 16 nearly always), the need-th largest of the lanes' two
        // largest is the bound; still more (equal values): tk_exact.
        constexpr int kList = 32;
        const int need = min(a.topk + (a.bias ? 2 : 0), L);
        int best = v[0];
#pragma unroll
        for (int j = 1; j < VPL; ++j) best = max(best, v[j]);
        int above = 0;
        auto turns = [](auto &&turn) __attribute__((always_inline)) {  // (row_ror i)
            turn(std::integral_constant<int, 0x121>{}), turn(std::integral_constant<int, 0x122>{});
            turn(std::integral_constant<int, 0x123>{}), turn(std::integral_constant<int, 0x124>{});
            turn(std::integral_constant<int, 0x125>{}), turn(std::integral_constant<int, 0x126>{});
            turn(std::integral_constant<int, 0x127>{}), turn(std::integral_constant<int, 0x128>{});
            turn(std::integral_constant<int, 0x129>{}), turn(std::integral_constant<int, 0x12a>{});
            turn(std::integral_constant<int, 0x12b>{}), turn(std::integral_constant<int, 0x12c>{});
            turn(std::integral_constant<int, 0x12d>{}), turn(std::integral_constant<int, 0x12e>{});
            turn(std::integral_constant<int, 0x12f>{});
        };
        turns([&](auto i) __attribute__((always_inline)) {
            above += __builtin_amdgcn_mov_dpp(best, decltype(i)::value, 0xf, 0xf, true) > best;
        });
        int bound = max(tk_lanes<L>(above < need ? best : 0x7fffffff, lane, tk_imin2), kNone + 1);
        int place, total_n;
        auto places = [&]() __attribute__((always_inline)) {
            int count = 0;
#pragma unroll
            for (int j = 0; j < VPL; ++j) count += v[j] >= bound;
            // places in the list: the counts of the lanes before (row_shr 1, 2, 4, 8: 0 comes in)
            place = count;
            place += __builtin_amdgcn_update_dpp(0, place, 0x111, 0xf, 0xf, true);
            place += __builtin_amdgcn_update_dpp(0, place, 0x112, 0xf, 0xf, true);
            place += __builtin_amdgcn_update_dpp(0, place, 0x114, 0xf, 0xf, true);
            place += __builtin_amdgcn_update_dpp(0, place, 0x118, 0xf, 0xf, true);
            total_n = tk_lanes<L>(place, lane, tk_imax2);  // (the last lane's)
            place -= count;
        };
        places();
        if (__ballot(total_n > kList)) {  // (uniform)
            int b1 = kNone, b2 = kNone, n1 = 0;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                b2 = max(b2, min(v[j], b1));
                b1 = max(b1, v[j]);
            }
            int n2 = b1 > b2;
            turns([&](auto i) __attribute__((always_inline)) {
                const int o1 = __builtin_amdgcn_mov_dpp(b1, decltype(i)::value, 0xf, 0xf, true);
                const int o2 = __builtin_amdgcn_mov_dpp(b2, decltype(i)::value, 0xf, 0xf, true);
                n1 += (o1 > b1) + (o2 > b1);
                n2 += (o1 > b2) + (o2 > b2);
            });
            const int low = min(n1 < need ? b1 : 0x7fffffff, n2 < need ? b2 : 0x7fffffff);
            bound = max(tk_lanes<L>(low, lane, tk_imin2), kNone + 1);
            places();
        }
        odd |= total_n > kList;
        u64 *list = space[w] + tok * kList, *order = space[w] + TPW * kList + tok * L;
        __builtin_amdgcn_wave_barrier();  // (the wave's own LDS, in order)
        list[sub] = list[sub + L] = order[sub] = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (v[j] >= bound) {
                if (place < kList) list[place] = ((u64)((uint32_t)v[j] ^ 0x80000000u) << 32) | (uint32_t)~(sub + L * j);
                ++place;
            }
        __builtin_amdgcn_wave_barrier();
        const u64 k0 = list[sub], k1 = list[sub + L];
        int r0 = 0, r1 = 0;
        for (int i = 0; i < kList; i += 2) {
            if (__ballot(i < total_n) == 0) break;  // (uniform)
            const ulonglong2 o = *(const ulonglong2 *)(list + i);
            r0 += (o.x > k0) + (o.y > k0);
            r1 += (o.x > k1) + (o.y > k1);
        }
        if (k0 && r0 < L) order[r0] = k0;
        if (k1 && r1 < L) order[r1] = k1;
        __builtin_amdgcn_wave_barrier();
        const u64 k = order[sub];
        int last = a.topk - 1;  // the last pick
        if (a.bias) {
            // a pick too close to the next one (the 16th: not known)
            const u64 next = order[min(sub + 1, L - 1)];
            const float x = tk_float((int)((uint32_t)(k >> 32) ^ 0x80000000u)), y = tk_float((int)((uint32_t)(next >> 32) ^ 0x80000000u));
            const bool amb = k != 0 && (sub == L - 1 ? total_n > L : next != 0 && !(x - y > tk_margin(x, err)));
            const uint32_t near = (uint32_t)(__ballot(amb) >> (L * tok)) & 0xffffu;
            last = __builtin_ctz(~near & ~((1u << (a.topk - 1)) - 1));  // (16: none of them is apart)
            // (close ones up to the list's end: those below the bound may be close too, and larger in 64 bits)
            odd |= last >= L || (last == total_n - 1 && bound > kNone + 1);
            close = (near & ((1u << min(last, L - 1)) - 1)) != 0;
        }
        if (k && sub <= last) {
            id = (int)~(uint32_t)k;
            pick = (int)((uint32_t)(k >> 32) ^ 0x80000000u);
        }
    } else {
        // topk rounds: the largest value, of equal ones the lowest index.  With a bias they go on
        // until a pick is apart from the next value.
        float last = __builtin_inff();
        bool settled = false;  // (alike in a token's lanes)
        for (int r = 0; a.bias || r < a.topk; ++r) {
            int best = v[0];
#pragma unroll
            for (int j = 1; j < VPL; ++j) best = max(best, v[j]);
            const int m = tk_lanes<L>(best, lane, tk_imax2);
            if (a.bias) {
                const float x = tk_float(m);
                const bool apart = m == kNone || last - x > tk_margin(last, err);
                settled |= r >= a.topk && apart;
                if (r >= a.topk && __ballot(!settled) == 0) break;  // (uniform)
                if (r == L) {  // more close values than lanes
                    odd |= !settled;
                    break;
                }
                close |= !settled && r > 0 && !apart;
                last = x;
            } else if (__ballot(m != kNone) == 0) {
                break;  // (uniform)
            }
            int e = 1 << 20;
#pragma unroll
            for (int j = VPL - 1; j >= 0; --j) e = v[j] == m ? E0 * sub + ES * j : e;
            e = tk_lanes<L>(e, lane, tk_imin2);
            const int at = e - E0 * sub;
#pragma unroll
            for (int j = 0; j < VPL; ++j) v[j] = at == ES * j ? kNone : v[j];
            if (sub == r && m != kNone && !settled) {
                id = e;
                pick = m;
            }
        }
    }
    float lv = tk_float(pick);
    if (a.bias) lv = id >= 0 ? tk_logit(a, tc, id) : 0.0f;
    int slot = sub;
    if (__ballot(close && !odd && on)) {  // (uniform)
        double x = 0.0;
        if (a.score == 0) {
            x = exp((double)lv - (double)mx) / tk_total<L>(a, tc, sub, mx);
        } else {
            x = 1.0 / (1.0 + exp(-(double)lv));
        }
        x += (double)a.bias[max(id, 0)];
        int rank = 0;
        for (int r = 0; r < L; ++r) {
            const double o = __shfl(x, L * tok + r, 64);
            const int oe = __shfl(id, L * tok + r, 64);
            if (__ballot(oe >= 0) == 0) break;  // (uniform: no token has a pick r)
            rank += oe >= 0 && (o > x || (o == x && oe < id));
        }
        if (close && id >= 0) slot = rank;
    }
    const u64 redo = __ballot(odd && on);
    const u64 own = L == 64 ? ~0ull : ((1ull << (L & 63)) - 1) << (L * tok);
    tk_write<L>(a, t, slot, id, lv, mx, total, on && !(redo & own));
    if (redo)
        for (int k = 0; k < TPW; ++k) {
            const u64 mask = L == 64 ? ~0ull : ((1ull << (L & 63)) - 1) << (L * k);
            if (redo & mask) tk_exact<VX>(a, t0 + k, lane, space[w]);
        }
}

template <int L, int VPL> void tk_launch(const TkArgs &a, hipStream_t st) {
    const int per = kTkWaves * 64 / L;
    const dim3 g((a.T + per - 1) / per), b(64 * kTkWaves);
    const size_t es = a.ltype == TERNOCL_FP32 ? 4 : 2, part = std::min<size_t>(16, VPL * es);
    const int members = a.E / a.n_group, lpg = members / VPL;
    const bool lanes = members % VPL == 0 && (lpg & (lpg - 1)) == 0 && (uintptr_t)a.logits % part == 0 &&
                       a.ld * es % part == 0 && (uintptr_t)a.bias % std::min(16, VPL * 4) == 0;
    if (a.topk_group == a.n_group) hipLaunchKernelGGL((k_moe_topk<L, VPL, 0>), g, b, 0, st, a);
    else if (lanes) hipLaunchKernelGGL((k_moe_topk<L, VPL, 2>), g, b, 0, st, a);
    else hipLaunchKernelGGL((k_moe_topk<L, VPL, 1>), g, b, 0, st, a);
}

}  // namespace

ternocl_status moe_topk_run(int ltype, const void *logits, long ld, const float *bias, int *ids, int wtype, void *RW, int T,
                            int E, int topk, int score, int n_group, int topk_group, int group_best, int renorm,
                            float scale, hipStream_t st) {
    const TkArgs a = {logits, bias, ids, RW, ld, ltype, T, E, topk, wtype, score, n_group, topk_group, group_best, renorm, scale};
    if (topk + (bias ? 1 : 0) <= 16) {  // (16 lanes hold the picks, with a bias the next one too)
        if (E <= 64) tk_launch<16, 4>(a, st);
        else if (E <= 128) tk_launch<16, 8>(a, st);
        else if (E <= 256) tk_launch<16, 16>(a, st);
        else tk_launch<16, 32>(a, st);
    } else {
        if (E <= 64) tk_launch<64, 1>(a, st);
        else if (E <= 128) tk_launch<64, 2>(a, st);
        else if (E <= 256) tk_launch<64, 4>(a, st);
        else tk_launch<64, 8>(a, st);
    }
    return check_launch();
}

}  // namespace tcl
