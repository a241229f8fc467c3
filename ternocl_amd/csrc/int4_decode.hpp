// int4_decode.hpp -- 4-bit weights (ternocl_int4_gemm's layout) as the B operands of the
// matrix-core GEMMs: the codes' decode and a lane's loads of words and scales.
#pragma once

#include "gemm_kw.hpp"

namespace tcl {
namespace {

// A word's 8 codes as B fragment dwords (rows 2 d, 2 d + 1 in dword d): with OFF q + 24, a
// nibble in the upper mantissa bits under the exponent of 16; without (fp16 alone has the
// packed arithmetic for it) q.
struct I4Const {
    uint32_t lo, hi, xlo, xhi;
};
template <bool BF16, bool OFF> __device__ __forceinline__ I4Const i4_const() {
    static_assert(OFF || !BF16);
    I4Const k = BF16  ? I4Const{0x00780078u, 0u, 0x41c041c0u, 0u}
                : OFF ? I4Const{0x03c003c0u, 0u, 0x4e004e00u, 0u}
                      : I4Const{0x000f000fu, 0x00f000f0u, 0x64086408u, 0x64806480u};
    asm("" : "+s"(k.lo));
    asm("" : "+s"(k.xlo));
    if constexpr (!OFF) {
        asm("" : "+s"(k.hi));
        asm("" : "+s"(k.xhi));
    }
    return k;
}
template <bool BF16, bool OFF> __device__ __forceinline__ void i4_decode(uint32_t x, const I4Const &k, uint32_t b[4]) {
    if constexpr (BF16) {
        b[0] = ((x << 3) & k.lo) ^ k.xlo;
        b[1] = ((x >> 1) & k.lo) ^ k.xlo;
        b[2] = ((x >> 5) & k.lo) ^ k.xlo;
        b[3] = ((x >> 9) & k.lo) ^ k.xlo;
    } else if constexpr (OFF) {
        b[0] = ((x << 6) & k.lo) ^ k.xlo;
        b[1] = ((x << 2) & k.lo) ^ k.xlo;
        b[2] = ((x >> 2) & k.lo) ^ k.xlo;
        b[3] = ((x >> 6) & k.lo) ^ k.xlo;
    } else {
        const uint32_t y = x >> 8;
        const uint32_t p[4] = {(x & k.lo) ^ k.xlo, (x & k.hi) ^ k.xhi, (y & k.lo) ^ k.xlo, (y & k.hi) ^ k.xhi};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            half2_t h;
            __builtin_memcpy(&h, &p[d], 4);
            if (d & 1) h = h * half2_t{(_Float16)0.0625f, (_Float16)0.0625f} - half2_t{(_Float16)72.0f, (_Float16)72.0f};
            else h = h - half2_t{(_Float16)1032.0f, (_Float16)1032.0f};
            __builtin_memcpy(&b[d], &h, 4);
        }
    }
}

// The walk's B source: CB adjacent columns' words of a unit and the scales (zeros) of its
// groups.
template <int CB, int PF, int G, bool ZP, bool NT = true> struct I4Src {
    static constexpr int GU = G < 64 ? 2 : 1;  // groups of a unit
    typedef typename KwVec<CB>::S SV;
    const uint32_t *B;
    const uint16_t *S, *Z;
    int N, units, q;
    uint32_t col;
    uint32_t w[PF][CB][4];
    SV sr[PF][GU], zr[PF][ZP ? GU : 1];
    template <class V> static __device__ __forceinline__ V ld(const V *p) {
        if constexpr (NT) return __builtin_nontemporal_load(p);
        else return *p;
    }
    __device__ __forceinline__ void load(int u, int s) {
        const int uc = min(u, units - 1);
        if constexpr (G < 64) {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const u32x2_t t = ld((const u32x2_t *)(B + ((size_t)(2 * uc + b) * N + col + cb) * 4 + 2 * q));
                    w[s][cb][2 * b] = t[0];
                    w[s][cb][2 * b + 1] = t[1];
                }
        } else {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const u32x4_t t = ld((const u32x4_t *)(B + ((size_t)(2 * uc + q) * N + col + cb) * 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) w[s][cb][i] = t[i];
            }
        }
#pragma unroll
        for (int g = 0; g < GU; ++g) {
            const size_t o = (size_t)(G < 64 ? 2 * uc + g : uc * 64 / G) * N + col;
            sr[s][g] = *(const SV *)(S + o);
            if constexpr (ZP) zr[s][g] = *(const SV *)(Z + o);
        }
    }
};

// Half `cb` of a vector of CB DT values
template <int CB, bool BF16> __device__ __forceinline__ float i4_scale(const typename KwVec<CB>::S &v, int cb) {
    uint32_t sw[(CB + 1) / 2] = {};
    __builtin_memcpy(sw, &v, sizeof(v));
    return dt2f<BF16>((sw[cb >> 1] >> (16 * (cb & 1))) & 0xffffu);
}

}  // namespace
}  // namespace tcl
