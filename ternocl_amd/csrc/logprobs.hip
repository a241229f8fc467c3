// logprobs.hip -- log probabilities of given tokens, entropy and top alternatives of
// rows of logits (ternocl_logprobs), in one pass over them.
//
//   d = scale * (l - max), r = sum e^d over all entries but one of the largest
//   ln p = d - log1p(r),   H = log1p(r) - (sum d e^d) / (1 + r)
//
// (the largest entry's own term, 1, is left out of r: a peaked row's r may be far
// below 2^-24, and 1 + r would lose it).
//
// The stream: a workgroup's 256 threads take 16-byte vectors in turn, kU of them in
// flight per thread; a wave keeps one running maximum for its lanes, raised at most
// once per batch of kU vectors (r and t = sum d e^d, in base 2, are scaled then).  What
// bounds it is HBM; a few rows are spread over workgroups, and the last of a row's to
// arrive (a counter in the workspace, whatever it held) joins their sums.
//
// The alternatives: every thread also keeps the largest of each run of its vectors (a
// "piece").  The topn-th largest of the 256 threads' maxima is a bound that at least topn
// entries reach, and only pieces whose maximum reaches it hold any: those are read again,
// their entries at or above the bound (about topn of them where values are spread)
// collected in LDS and ranked by (logit, lowest index).  Where more than kFlags pieces or
// kCap entries reach it (many equal logits), a radix selection over the whole row first
// finds the exact topn-th (value, index) key.
//
// V = 151680, 20 alternatives: 512 rows fp32 61.6 us, 5.0 TB/s (a large copy's rate), bf16
// 46.1 us (a row a workgroup, two waves a SIMD, too few to put VALU beside loads: 39% of a wave's
// time each, the SIMDs' VALU busy 54% of it); one row 10.2 us (latency: the stream, the arrival, the
// alternatives, and the code's fetch).  On counters that were not left at zero the split rows
// take 18 to 21 us more (kw_arrive counts its up to 32 arrivals by exchanges).
#include "common.hpp"

namespace tcl {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256, kWaves = 4;
constexpr int kU = 4;      // vectors in flight per thread
constexpr int kPieces = 32;  // runs of batches per thread, chunks of a row at most
constexpr int kPairs = kPieces / 2;
constexpr int kCap = 512;  // candidates ranked in LDS

template <int LT> struct LpVec {
    static constexpr int NV = LT == TERNOCL_FP32 ? 4 : 8;  // entries of 16 bytes
    static constexpr int ES = LT == TERNOCL_FP32 ? 4 : 2;
};

template <int LT> __device__ __forceinline__ void lp_unpack(const uint4 &v, float x[LpVec<LT>::NV]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (LT == TERNOCL_FP32) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[2 * i] = dt2f<LT == TERNOCL_BF16>(w[i] & 0xffffu);
            x[2 * i + 1] = dt2f<LT == TERNOCL_BF16>(w[i] >> 16);
        }
    }
}
template <int LT> __device__ __forceinline__ float lp_load1(const void *row, int i) {
    if constexpr (LT == TERNOCL_FP32) return ((const float *)row)[i];
    else return dt2f<LT == TERNOCL_BF16>(((const uint16_t *)row)[i]);
}

// A row: `head` entries before its first 16-byte boundary, then nvec vectors, then the
// rest.  Head and rest (at most 14 entries) are the "edge", entry e of it thread e's.
template <int LT> struct LpRow {
    const uint8_t *p;
    int V, head, nvec, edge;
    __device__ __forceinline__ LpRow(const void *logits, long ld, int m, int V_) : V(V_) {
        constexpr int NV = LpVec<LT>::NV, ES = LpVec<LT>::ES;
        p = (const uint8_t *)logits + (size_t)m * ld * ES;
        head = min(V, (int)((16 - ((uintptr_t)p & 15)) & 15) / ES);
        nvec = (V - head) / NV;
        edge = V - NV * nvec;
    }
    __device__ __forceinline__ int edge_index(int e) const { return e < head ? e : e + LpVec<LT>::NV * nvec; }
    __device__ __forceinline__ uint4 vec(int i) const {
        return *(const uint4 *)(p + (size_t)head * LpVec<LT>::ES + 16 * (size_t)i);
    }
};

__device__ __forceinline__ float lp_wave_max(float v, int lane) {
    v = fmaxf(v, lane_xor<1>(v, lane));
    v = fmaxf(v, lane_xor<2>(v, lane));
    v = fmaxf(v, lane_xor<4>(v, lane));
    v = fmaxf(v, lane_xor<8>(v, lane));
    v = fmaxf(v, lane_xor<16>(v, lane));
    return fmaxf(v, lane_xor<32>(v, lane));
}
__device__ __forceinline__ float lp_wave_sum(float v, int lane) {
    v += lane_xor<1>(v, lane);
    v += lane_xor<2>(v, lane);
    v += lane_xor<4>(v, lane);
    v += lane_xor<8>(v, lane);
    v += lane_xor<16>(v, lane);
    return v + lane_xor<32>(v, lane);
}

// Sums of a set of entries: largest m (-inf: none above -inf), r and t as above, t in
// base 2 (sum of e2 2^e2, e2 = d log2 e).  A NaN anywhere makes r NaN.
struct LpSum {
    float m, r, t;
};
// a and b together; c = scale * log2 e.
__device__ __forceinline__ LpSum lp_join(LpSum a, LpSum b, float c) {
    if (b.m > a.m) {
        const LpSum x = a;
        a = b;
        b = x;
    }
    LpSum o = a;
    if (b.m == -__builtin_inff()) {  // nothing in b (or a NaN in its r)
        o.r += b.r;
        return o;
    }
    const float d = (b.m - a.m) * c, f = __builtin_amdgcn_exp2f(d);
    o.r += f * (1.0f + b.r);
    if (f > 0.0f) o.t += f * (b.t + d * (1.0f + b.r));
    return o;
}

// One entry's terms: (2^e2, e2 2^e2).  (No -inf times 0; a NaN stays one in r.)
__device__ __forceinline__ void lp_term(float x, float m, float c, float &r, float &t) {
    const float d = (x - m) * c, e = __builtin_amdgcn_exp2f(d);
    r += e;
    t = __builtin_fmaf(fmaxf(d, -1000.0f), e, t);
}

// A wave's running sums: m uniform, r and t a lane's part of the sums relative to m.
struct LpState {
    float m, r, t;
    __device__ __forceinline__ void init() {
        m = -__builtin_inff();
        r = t = 0.0f;
    }
    // n entries of each lane (padding: -inf) whose lane maximum is tm
    template <int n> __device__ __forceinline__ void add(float (&x)[n], float tm, float c, int lane) {
        const float wm = __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(lp_wave_max(tm, lane))));
        if (wm > m) {  // (uniform) a new maximum
            if (m != -__builtin_inff()) {
                // the lanes' sums so far, and the old maximum's own term in lane 0
                const float d = (m - wm) * c, f = __builtin_amdgcn_exp2f(d);
                const float old = r + (lane == 0 ? 1.0f : 0.0f);
                t = f > 0.0f ? f * (t + d * old) : 0.0f;
                r = f * old;
            }
            m = wm;
            bool done = lane != __builtin_ctzll(__ballot(tm == wm));  // one of its entries is left out
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const bool hit = !done && x[i] == wm;
                x[i] = hit ? -__builtin_inff() : x[i];
                done |= hit;
            }
        }
        if (m == -__builtin_inff()) {  // only -inf so far (or NaN: its r must show it)
#pragma unroll
            for (int i = 0; i < n; ++i) r += x[i] != x[i] ? x[i] : 0.0f;
            return;
        }
#pragma unroll
        for (int i = 0; i < n; ++i) lp_term(x[i], m, c, r, t);
    }
};

// Streams vectors [v0, v1) of a row (and, with edge, its edge entries) through this
// workgroup; put(p, x): the largest entry of this thread's piece p (bpp batches of 256 kU
// vectors; the edge belongs to piece 0).  Leaves each wave's sums in LDS, wsum[wave]
// (a barrier follows before they are read).
template <int LT, bool TOP, class Put>
__device__ __forceinline__ void lp_stream(const LpRow<LT> &row, int v0, int v1, bool edge, int bpp, float c, LpSum *wsum,
                                          Put &&put) {
    constexpr int NV = LpVec<LT>::NV;
    const int tid = threadIdx.x, lane = tid & 63;
    LpState st;
    st.init();
    float piece = -__builtin_inff();
    if (edge && __builtin_amdgcn_readfirstlane(tid) < 64) {
        float x[1] = {-__builtin_inff()};
        if (tid < row.edge) x[0] = lp_load1<LT>(row.p, row.edge_index(tid));
        piece = fmaxf(x[0], -__builtin_inff());
        st.add(x, piece, c, lane);
    }
    int b = 0, p = 0;
    uint4 raw[kU], ahead[kU];
    auto fetch = [&](int v, uint4 (&o)[kU]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kU; ++u) o[u] = row.vec(min(v + u * kThreads + tid, v1 - 1));
    };
    // a batch from vector v on; part: some of its vectors are past v1
    auto batch = [&](int v, auto part) __attribute__((always_inline)) {
        float x[kU * NV];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float y[NV];
            lp_unpack<LT>(raw[u], y);
            raw[u] = ahead[u];
            const bool in = !decltype(part)::value || v + u * kThreads + tid < v1;
#pragma unroll
            for (int i = 0; i < NV; ++i) x[u * NV + i] = in ? y[i] : -__builtin_inff();
        }
        float tm = x[0];
#pragma unroll
        for (int i = 1; i < kU * NV; ++i) tm = fmaxf(tm, x[i]);
        tm = fmaxf(tm, -__builtin_inff());
        st.add(x, tm, c, lane);
        if constexpr (TOP) {
            piece = fmaxf(piece, tm);
            if (++b == bpp) {
                put(p, piece);
                piece = -__builtin_inff();
                b = 0;
                ++p;
            }
        }
    };
    if (v0 < v1) fetch(v0, raw);
    int v = v0;
    for (; v + kThreads * kU <= v1; v += kThreads * kU) {
        if (v + kThreads * kU < v1) fetch(v + kThreads * kU, ahead);
        batch(v, std::false_type{});
    }
    if (v < v1) batch(v, std::true_type{});
    if constexpr (TOP) {
        if (b || p == 0) put(p, piece);
    }
    const float r = lp_wave_sum(st.r, lane), t = lp_wave_sum(st.t, lane);
    if (lane == 0) wsum[tid >> 6] = LpSum{st.m, r, t};
}

struct LpArgs {
    const void *logits;
    long ld;
    const int *tokens;
    float *logp, *entropy;
    int *top_ids;
    float *top_logp;
    int M, V, topn;
    float scale;
    int chunks, chunk_vecs;  // of the split launch
    uint64_t *arrived;       // [M][2]: arrival counters (workspace header)
    float *sums;             // [M][chunks][3] (workspace)
    float *maxima;           // [M][chunks][256] (workspace)
};

constexpr int kFlags = 512;  // pieces read again at most
struct LpLds {
    uint32_t thread[kThreads];  // the threads' maxima, in order (lp_ord)
    u64 cand[kCap];
    uint32_t flag[kFlags];
    uint32_t hist[256];
    int count, flags, need;
    u64 key;
};
// A value's bits as an unsigned integer in the order of the values (-0 as +0).
__device__ __forceinline__ uint32_t lp_ord(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ u64 lp_key(float v, int i) { return ((u64)lp_ord(v) << 32) | (uint32_t)~i; }  // larger: before
__device__ __forceinline__ float lp_key_value(u64 k) {
    const uint32_t h = (uint32_t)(k >> 32);
    return __uint_as_float(h & 0x80000000u ? h ^ 0x80000000u : ~h);
}


// Calls f(value, index) on every entry of the row, thread by thread.
template <int LT, class F> __device__ __forceinline__ void lp_scan(const LpRow<LT> &row, F &&f) {
    constexpr int NV = LpVec<LT>::NV;
    const int tid = threadIdx.x;
    if (tid < row.edge) {
        const int i = row.edge_index(tid);
        f(lp_load1<LT>(row.p, i), i);
    }
    for (int v = tid; v < row.nvec; v += kThreads) {
        float y[NV];
        lp_unpack<LT>(row.vec(v), y);
#pragma unroll
        for (int i = 0; i < NV; ++i) f(y[i], row.head + v * NV + i);
    }
}

// scale (x - m), finite wherever that is in fp32 (halves: the difference may be past its range).
__device__ __forceinline__ float lp_scaled(float x, float m, float scale) { return (0.5f * x - 0.5f * m) * (2.0f * scale); }

// The token asked for (-1: none).
__device__ __forceinline__ int lp_token(const LpArgs &a, int m) {
    const int tok = a.tokens ? a.tokens[m] : -1;
    return tok < a.V ? tok : -1;
}

// The maxima of a row's pieces, two of one piece row in a load: thread t has pairs t + 256 i
// of [pieces][128] pairs.
struct LpMaxima {
    float x[2 * kPairs];
    template <class Get> __device__ __forceinline__ void load(int pieces, Get &&get) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const int j = threadIdx.x + kThreads * i;
            const float2 v = get(min(j, 128 * pieces - 1));
            x[2 * i] = j < 128 * pieces ? v.x : -__builtin_inff();
            x[2 * i + 1] = j < 128 * pieces ? v.y : -__builtin_inff();
        }
    }
};

// The row's outputs from its sums and its pieces' maxima, p < pieces: thread t's piece p holds
// vectors p span + t + 256 i, i < span / 256 (and, with p = 0, edge entry t).
template <int LT, bool TOP>
__device__ __forceinline__ void lp_finish(const LpArgs &a, const LpRow<LT> &row, int m, const LpSum &s,
                                          int tok, float tok_x, const LpMaxima &pm, int pieces, int span, LpLds &L) {
    constexpr int NV = LpVec<LT>::NV;
    const int tid = threadIdx.x, lane = tid & 63;
    const bool empty = s.m == -__builtin_inff() && s.r == 0.0f;
    const bool bad = !(s.r < __builtin_inff()) || s.m == __builtin_inff();
    const float l1 = log1pf(s.r), nan = __builtin_nanf("");
    if (tid == 0) {
        if (a.logp) {
            const float o = bad ? nan : empty ? -__builtin_inff() : lp_scaled(tok_x, s.m, a.scale) - l1;
            a.logp[m] = tok < 0 ? 0.0f : o;
        }
        if (a.entropy)
            a.entropy[m] = bad ? nan : empty ? 0.0f : l1 - s.t * 0.693147180559945309f / (1.0f + s.r);
    }
    if constexpr (!TOP) return;
    int *ids = a.top_ids + (size_t)m * a.topn;
    float *out = a.top_logp + (size_t)m * a.topn;
    if (bad || empty) {  // (uniform)
        if (tid < a.topn) {
            ids[tid] = -1;
            out[tid] = bad ? nan : -__builtin_inff();
        }
        return;
    }
    // the bound: of 256 threads' maxima (each of its pairs above), the topn-th largest's upper
    // 16 bits (topn entries at least reach it)
    float v = pm.x[0];
#pragma unroll
    for (int i = 1; i < 2 * kPairs; ++i) v = fmaxf(v, pm.x[i]);
    L.thread[tid] = lp_ord(v) >> 16;
    if (tid == 0) L.count = L.flags = 0;
    __syncthreads();
    uint32_t o4[4], found = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) o4[i] = L.thread[64 * i + lane];
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {  // (rolled, as below: a few rows' call is as long as its code takes to fetch)
        const uint32_t t = found | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += __builtin_popcountll(__ballot(o4[i] >= t));
        if (n >= a.topn) found = t;  // (uniform)
    }
    const uint32_t bound = found << 16;  // (of lp_ord; a row with fewer entries than topn above -inf: 0x007f << 16)
    // the pieces that hold entries at or above it
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i < 2 * kPairs; ++i) hits |= (uint32_t)(pm.x[i] > -__builtin_inff() && lp_ord(pm.x[i]) >= bound) << i;
    while (hits) {
        const int i = __builtin_ctz(hits), n = atomicAdd(&L.flags, 1);
        if (n < kFlags) L.flag[n] = (uint32_t)(2 * (tid + kThreads * (i >> 1)) + (i & 1));
        hits &= hits - 1;
    }
    __syncthreads();
    const int flags = L.flags, per = span / kThreads + 1;  // (the last: the edge)
    // those of n entries (indices i0 + their place) into the list, one addition to its count
    auto take = [&](auto &x, auto n, int i0) __attribute__((always_inline)) {
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < decltype(n)::value; ++i) mask |= (uint32_t)(x[i] > -__builtin_inff() && lp_ord(x[i]) >= bound) << i;
        if (!mask) return;
        int at = atomicAdd(&L.count, __builtin_popcount(mask));
#pragma unroll
        for (int i = 0; i < decltype(n)::value; ++i)
            if (mask >> i & 1) {
                if (at < kCap) L.cand[at] = lp_key(x[i], i0 + i);
                ++at;
            }
    };
    if (flags <= kFlags)
        for (int it = tid; it < flags * per; it += kThreads) {
            const int f = it / per, j = it - f * per, p = (int)L.flag[f] / kThreads, t = (int)L.flag[f] % kThreads;
            if (j == per - 1) {
                if (p == 0 && t < row.edge) {
                    const int i = row.edge_index(t);
                    const float x[1] = {lp_load1<LT>(row.p, i)};
                    take(x, std::integral_constant<int, 1>{}, i);
                }
            } else {
                const int w = p * span + t + kThreads * j;
                if (w < row.nvec) {
                    float y[NV];
                    lp_unpack<LT>(row.vec(w), y);
                    take(y, std::integral_constant<int, NV>{}, row.head + w * NV);
                }
            }
        }
    __syncthreads();
    int count = L.count;
    if (count > kCap || flags > kFlags) {  // (uniform)
        // the topn-th largest key, 8 bits at a time over the whole row
        u64 prefix = 0;
        int need = a.topn;
        for (int shift = 56; shift >= 0; shift -= 8) {
            __syncthreads();
            L.hist[tid] = 0;
            __syncthreads();
            lp_scan<LT>(row, [&](float x, int i) __attribute__((always_inline)) {
                const u64 k = lp_key(x, i);
                if (x > -__builtin_inff() && (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))))
                    atomicAdd(&L.hist[(k >> shift) & 255], 1u);
            });
            __syncthreads();
            if (tid == 0) {
                int b = 255, n = need;
                while (b > 0 && (int)L.hist[b] < n) n -= (int)L.hist[b--];
                L.key = prefix | ((u64)b << shift);
                L.need = n;
            }
            __syncthreads();
            prefix = L.key;
            need = L.need;
        }
        if (tid == 0) L.count = 0;
        __syncthreads();
        lp_scan<LT>(row, [&](float x, int i) __attribute__((always_inline)) {
            const u64 k = lp_key(x, i);
            if (k >= prefix && x > -__builtin_inff()) {
                const int n = atomicAdd(&L.count, 1);
                if (n < kCap) L.cand[n] = k;
            }
        });
        __syncthreads();
        count = min(L.count, kCap);
    }
    for (int c = tid; c < count; c += kThreads) {
        const u64 k = L.cand[c];
        int before = 0;
#pragma unroll 4
        for (int i = 0; i < count; ++i) before += L.cand[i] > k;
        if (before < a.topn) {
            ids[before] = (int)~(uint32_t)k;
            out[before] = lp_scaled(lp_key_value(k), s.m, a.scale) - l1;
        }
    }
    for (int i = count + tid; i < a.topn; i += kThreads) {
        ids[i] = -1;
        out[i] = -__builtin_inff();
    }
}

// A row per workgroup.  LDS: the pieces' maxima [pieces][256].
template <int LT, bool TOP> __global__ void __launch_bounds__(kThreads) k_logprobs_row(const LpArgs a, int pieces, int bpp) {
    extern __shared__ __attribute__((aligned(16))) float lp_pm[];
    __shared__ LpSum wsum[kWaves];
    __shared__ std::conditional_t<TOP, LpLds, int> L;
    const int m = blockIdx.x, tid = threadIdx.x;
    const LpRow<LT> row(a.logits, a.ld, m, a.V);
    const int tok = lp_token(a, m);  // (used only after the stream)
    const float c = a.scale * 1.44269504088896341f;
    if constexpr (TOP)
        for (int p = 1; p < pieces; ++p) lp_pm[p * kThreads + tid] = -__builtin_inff();
    lp_stream<LT, TOP>(row, 0, row.nvec, true, bpp, c, wsum, [&](int p, float x) __attribute__((always_inline)) {
        lp_pm[p * kThreads + tid] = x;
    });
    __syncthreads();
    LpSum s = wsum[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) s = lp_join(s, wsum[i], c);
    const float tok_x = lp_load1<LT>(row.p, max(tok, 0));
    LpMaxima pm;
    if constexpr (TOP) pm.load(pieces, [&](int j) __attribute__((always_inline)) { return ((const float2 *)lp_pm)[j]; });
    lp_finish<LT, TOP>(a, row, m, s, tok, tok_x, pm, pieces, bpp * kThreads * kU, reinterpret_cast<LpLds &>(L));
}

__device__ __forceinline__ void lp_put(float *p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float lp_get(const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A row over a.chunks workgroups, a chunk a piece of each thread: the one that arrives
// last has the others' sums and maxima (agent-scope stores, done before the arrival) and
// finishes the row.
template <int LT, bool TOP> __global__ void __launch_bounds__(kThreads) k_logprobs_split(const LpArgs a) {
    __shared__ LpSum wsum[kWaves];
    __shared__ std::conditional_t<TOP, LpLds, int> L;
    __shared__ int flag;
    const int m = blockIdx.y, k = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const LpRow<LT> row(a.logits, a.ld, m, a.V);
    const int tok = lp_token(a, m);  // (used only after the stream)
    const float c = a.scale * 1.44269504088896341f;
    const int v0 = min(k * a.chunk_vecs, row.nvec), v1 = min(row.nvec, v0 + a.chunk_vecs);
    float *sums = a.sums + 3 * (size_t)m * a.chunks, *maxima = a.maxima + (size_t)m * a.chunks * kThreads;
    lp_stream<LT, TOP>(row, v0, v1, k == 0, a.chunk_vecs, c, wsum, [&](int, float x) __attribute__((always_inline)) {
        lp_put(maxima + k * kThreads + tid, x);
    });
    __syncthreads();
    LpSum s = wsum[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) s = lp_join(s, wsum[i], c);
    if (tid == 0) {
        lp_put(sums + 3 * k, s.m);
        lp_put(sums + 3 * k + 1, s.r);
        lp_put(sums + 3 * k + 2, s.t);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();  // every wave's stores are done
    if (tid < 64) {
        const bool last = kw_arrive(a.arrived + 2 * (size_t)m, a.chunks, lane);
        if (lane == 0) flag = last;
    }
    __syncthreads();
    if (!flag) return;  // (uniform)
    const float tok_x = lp_load1<LT>(row.p, max(tok, 0));
    LpMaxima pm;
    if constexpr (TOP)
        pm.load(a.chunks, [&](int j) __attribute__((always_inline)) {
            const uint64_t v = __hip_atomic_load((const uint64_t *)maxima + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
        });
    s = LpSum{-__builtin_inff(), 0.0f, 0.0f};
    if (lane < a.chunks) s = LpSum{lp_get(sums + 3 * lane), lp_get(sums + 3 * lane + 1), lp_get(sums + 3 * lane + 2)};
    {  // the chunks' sums, one a lane, relative to the largest maximum (lp_join, all at once)
        const float top = lp_wave_max(s.m, lane);
        const bool one = lane == __builtin_ctzll(__ballot(s.m == top));  // (its own term left out)
        const bool none = s.m == -__builtin_inff();
        const float d = none ? 0.0f : (s.m - top) * c, f = none ? 0.0f : __builtin_amdgcn_exp2f(d), n = 1.0f + s.r;
        const float r = none || one ? s.r : f * n, t = one ? s.t : f > 0.0f ? f * (s.t + d * n) : 0.0f;
        s = LpSum{top, lp_wave_sum(r, lane), lp_wave_sum(t, lane)};
    }
    lp_finish<LT, TOP>(a, row, m, s, tok, tok_x, pm, a.chunks, a.chunk_vecs, reinterpret_cast<LpLds &>(L));
}

// Workgroups a row is spread over (nv: entries of a vector): as many as whole batches
// give, while all rows stay within about kSplit workgroups.
constexpr int kSplit = 1024;
int lp_chunks(int M, int V, int nv, int &chunk_vecs) {
    const long batch = (long)kThreads * kU;
    const long nb = V < nv ? 1 : ((long)V / nv + batch - 1) / batch;
    long c = M >= kSplit / 2 ? 1 : kSplit / M;
    if (c > nb) c = nb;
    if (c > kPieces) c = kPieces;
    const long per = (nb + c - 1) / c;
    chunk_vecs = (int)(per * batch);
    return (int)((nb + per - 1) / per);
}

}  // namespace

static size_t lp_ws(int M, int V, int topn, int nv) {
    int cv;
    const int c = lp_chunks(M, V, nv, cv);
    return c == 1 ? 0 : kWsHeader + (size_t)M * c * (12 + (topn ? 4 * kThreads : 0)) + 4;
}
size_t logprobs_ws_need(int M, int V, int topn) {  // (whichever the type)
    const size_t a = lp_ws(M, V, topn, 4), b = lp_ws(M, V, topn, 8);
    return a > b ? a : b;
}

ternocl_status logprobs_run(int ltype, const void *logits, long ld, const int *tokens, float *logp, float *entropy,
                            int *top_ids, float *top_logp, int M, int V, int topn, float scale, void *ws,
                            size_t ws_bytes, hipStream_t st) {
    LpArgs a = {logits, ld, tokens, logp, entropy, top_ids, top_logp, M, V, topn, scale, 1, 0, nullptr, nullptr, nullptr};
    const int nv = ltype == TERNOCL_FP32 ? 4 : 8;
    const size_t need = lp_ws(M, V, topn, nv);
    if (need && ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0) a.chunks = lp_chunks(M, V, nv, a.chunk_vecs);
    const bool split = a.chunks > 1;
    if (split) {
        a.arrived = (uint64_t *)ws;  // (kSplit / 2 rows of 16 bytes: within the header)
        a.sums = (float *)((uint8_t *)ws + kWsHeader);
        a.maxima = a.sums + align_up(3 * (size_t)M * a.chunks, 2);
    }
    // pieces of the unsplit launch: at most kPieces runs of batches
    const int nb = (V / nv + kThreads * kU - 1) / (kThreads * kU);
    const int bpp = nb > kPieces ? (nb + kPieces - 1) / kPieces : 1, pieces = nb > 0 ? (nb + bpp - 1) / bpp : 1;
    auto go = [&](auto lt, auto top) {
        constexpr int LT = decltype(lt)::value;
        constexpr bool TOP = decltype(top)::value;
        if (split) {
            hipLaunchKernelGGL((k_logprobs_split<LT, TOP>), dim3(a.chunks, M), dim3(kThreads), 0, st, a);
        } else {
            hipLaunchKernelGGL((k_logprobs_row<LT, TOP>), dim3(M), dim3(kThreads), TOP ? pieces * kThreads * 4 : 0, st, a,
                               pieces, bpp);
        }
    };
    auto lt = [&](auto top) {
        if (ltype == TERNOCL_FP32) go(std::integral_constant<int, TERNOCL_FP32>{}, top);
        else if (ltype == TERNOCL_BF16) go(std::integral_constant<int, TERNOCL_BF16>{}, top);
        else go(std::integral_constant<int, TERNOCL_FP16>{}, top);
    };
    if (topn) lt(std::true_type{});
    else lt(std::false_type{});
    return check_launch();
}

}  // namespace tcl
