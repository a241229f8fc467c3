// moe_topk.hip -- routing to experts: the ids and weights that the MoE layers take,
// from the router's logits (ternocl_moe_topk).
//
//   s = softmax(l) or 1 / (1 + e^-l), v = s + bias; the topk_group groups with the
//   largest sums of their group_best largest v stay; ids = the topk largest v, RW = s
//   of those (renormalised), times scale.
//
// One wave per token, lane i holding the VPL experts from VPL i on, so that of equal
// values the lowest lane's lowest expert is the lowest index.  What is compared are
// unsigned keys in the order of the values (0: never chosen, all ones: NaN):
//   * without a bias the logits themselves order the experts -- softmax and the sigmoid
//     rise with them, and in exact arithmetic only equal logits give equal scores --
//     so a key is the 32 bits of the fp32 logit;
//   * with a bias v is computed in fp64 (fp32 scores would tie or swap values closer
//     than 2^-24 that differ), a key is its 64 bits.
#include "common.hpp"

namespace tcl {
namespace {

typedef unsigned long long u64;

template <int LT> __device__ __forceinline__ float tk_load(const void *p, size_t i) {
    if constexpr (LT == TERNOCL_FP32) return ((const float *)p)[i];
    else return dt2f<LT == TERNOCL_BF16>(((const uint16_t *)p)[i]);
}

// Keys: larger value, larger key; -0 as +0, -inf 0, NaN all ones.
__device__ __forceinline__ uint32_t tk_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return ~0u;
    if (b == 0xff800000u) return 0u;
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
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
__device__ __forceinline__ float tk_fmax(float v, int lane) {
    v = fmaxf(v, lane_xor<1>(v, lane));
    v = fmaxf(v, lane_xor<2>(v, lane));
    v = fmaxf(v, lane_xor<4>(v, lane));
    v = fmaxf(v, lane_xor<8>(v, lane));
    v = fmaxf(v, lane_xor<16>(v, lane));
    return fmaxf(v, lane_xor<32>(v, lane));
}
__device__ __forceinline__ double tk_sum(double v) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}

struct TkArgs {
    const void *logits;
    const float *bias;
    int *ids;
    void *RW;
    long ld;
    int T, E, topk, wtype, score, n_group, topk_group, group_best, renorm;
    float scale;
};

constexpr int kTkWaves = 4;

// WIDE: 64-bit keys of v (a bias); else the logits' own.  GROUPED: a choice of groups.
template <int LT, int VPL, bool WIDE, bool GROUPED>
__global__ void __launch_bounds__(64 * kTkWaves) k_moe_topk(const TkArgs a) {
    typedef std::conditional_t<WIDE, u64, uint32_t> Key;
    __shared__ u64 gkey[GROUPED ? kTkWaves : 1][GROUPED ? 64 * VPL : 1];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kTkWaves + w;
    if (t >= a.T) return;  // (whole wave; no barrier follows)
    const int e0 = VPL * lane;
    float l[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const float x = tk_load<LT>(a.logits, (size_t)t * a.ld + min(e0 + j, a.E - 1));
        l[j] = e0 + j < a.E ? x : -__builtin_inff();
    }
    // softmax: the row's largest logit (NaN passed over: it reaches the sum below)
    float mx = l[0];
#pragma unroll
    for (int j = 1; j < VPL; ++j) mx = fmaxf(mx, l[j]);
    mx = tk_fmax(mx, lane);
    double total = 1.0;
    const bool need_scores = WIDE || (GROUPED && a.group_best == 2);
    double s[VPL];
    if (a.score == 0 && (need_scores || !a.renorm)) {
        double p = 0.0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            s[j] = l[j] == -__builtin_inff() ? 0.0 : exp((double)l[j] - (double)mx);
            p += s[j];
        }
        total = tk_sum(p);
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = s[j] / total;
    } else if (need_scores) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = 1.0 / (1.0 + exp(-(double)l[j]));
    }
    Key key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        if constexpr (WIDE) {
            const double v = s[j] + (double)a.bias[min(e0 + j, a.E - 1)];
            key[j] = l[j] == -__builtin_inff() ? 0 : tk_key(v);
        } else {
            key[j] = tk_key(l[j]);
        }
    }
    if constexpr (GROUPED) {
        // a group's value as a key of its own (0: none to choose), lane g for group g
        const int per = a.E / a.n_group;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if constexpr (WIDE) gkey[w][e0 + j] = key[j];
            else gkey[w][e0 + j] = a.group_best == 2 ? (key[j] ? tk_key(s[j]) : 0) : (u64)key[j];
        }
        __builtin_amdgcn_wave_barrier();  // (the wave's own LDS, in order)
        u64 k1 = 0, k2 = 0;
        if (lane < a.n_group)
            for (int i = 0; i < per; ++i) {
                const u64 k = gkey[w][lane * per + i];
                k2 = max(k2, min(k, k1));
                k1 = max(k1, k);
            }
        u64 gv = k1;
        if (a.group_best == 2 && k1 != 0 && k1 != ~0ull && k2 != 0) gv = tk_key(tk_value(k1) + tk_value(k2));
        // kept: fewer than topk_group groups come before it
        int before = 0;
        for (int g = 0; g < a.n_group; ++g) {
            const u64 o = (u64)__builtin_amdgcn_readlane((int)(uint32_t)gv, g) & 0xffffffffull;
            const u64 ov = o | ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(gv >> 32), g) << 32);
            before += ov > gv || (ov == gv && g < lane);
        }
        const u64 kept = __ballot(before < a.topk_group);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (!((kept >> (min(e0 + j, a.E - 1) / per)) & 1)) key[j] = 0;
    }
    // topk rounds: the largest key, of equal ones the lowest lane's lowest
    int id = -1;       // lane r: round r's expert
    float lv = 0.0f;   // ... and its logit
    for (int r = 0; r < a.topk; ++r) {
        Key best = key[0];
#pragma unroll
        for (int j = 1; j < VPL; ++j) best = max(best, key[j]);
        const Key m = tk_max(best, lane);
        if (m == 0) break;  // (uniform)
        const int from = __builtin_ctzll(__ballot(best == m));
        int e = 0;
        float x = 0.0f;
#pragma unroll
        for (int j = VPL - 1; j >= 0; --j)
            if (key[j] == m) {
                e = e0 + j;
                x = l[j];
            }
        bool taken = false;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (lane == from && !taken && key[j] == m) {
                key[j] = 0;
                taken = true;
            }
        e = __builtin_amdgcn_readlane(e, from);
        x = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), from));
        if (lane == r) {
            id = e;
            lv = x;
        }
    }
    // the weights, one lane each, in fp64 (a lane's work for the whole wave: one exp)
    const bool live = lane < a.topk && id >= 0;
    double wt;
    if (a.score == 0) wt = exp((double)lv - (double)mx) / total;
    else wt = 1.0 / (1.0 + exp(-(double)lv));
    if (!live) wt = 0.0;
    if (a.renorm) {
        const double sum = tk_sum(wt);
        wt = sum == 0.0 ? 0.0 : wt / sum;
    }
    wt *= (double)a.scale;
    if (lane < a.topk) {
        const size_t o = (size_t)t * a.topk + lane;
        a.ids[o] = id;
        const float f = live ? (float)wt : 0.0f;
        if (a.wtype == TERNOCL_FP32) ((float *)a.RW)[o] = f;
        else ((uint16_t *)a.RW)[o] = (uint16_t)(a.wtype == TERNOCL_BF16 ? f2dt<true>(f) : f2dt<false>(f));
    }
}

template <int LT, int VPL> void tk_launch(const TkArgs &a, hipStream_t st) {
    const dim3 g((a.T + kTkWaves - 1) / kTkWaves), b(64 * kTkWaves);
    const bool grouped = a.topk_group < a.n_group;
    if (a.bias) {
        if (grouped) hipLaunchKernelGGL((k_moe_topk<LT, VPL, true, true>), g, b, 0, st, a);
        else hipLaunchKernelGGL((k_moe_topk<LT, VPL, true, false>), g, b, 0, st, a);
    } else {
        if (grouped) hipLaunchKernelGGL((k_moe_topk<LT, VPL, false, true>), g, b, 0, st, a);
        else hipLaunchKernelGGL((k_moe_topk<LT, VPL, false, false>), g, b, 0, st, a);
    }
}

template <int LT> void tk_vpl(const TkArgs &a, hipStream_t st) {
    if (a.E <= 64) tk_launch<LT, 1>(a, st);
    else if (a.E <= 128) tk_launch<LT, 2>(a, st);
    else if (a.E <= 256) tk_launch<LT, 4>(a, st);
    else tk_launch<LT, 8>(a, st);
}

}  // namespace

ternocl_status moe_topk_run(int ltype, const void *logits, long ld, const float *bias, int *ids, int wtype, void *RW, int T,
                            int E, int topk, int score, int n_group, int topk_group, int group_best, int renorm,
                            float scale, hipStream_t st) {
    const TkArgs a = {logits, bias, ids, RW, ld, T, E, topk, wtype, score, n_group, topk_group, group_best, renorm, scale};
    if (ltype == TERNOCL_FP32) tk_vpl<TERNOCL_FP32>(a, st);
    else if (ltype == TERNOCL_BF16) tk_vpl<TERNOCL_BF16>(a, st);
    else tk_vpl<TERNOCL_FP16>(a, st);
    return check_launch();
}

}  // namespace tcl
