// Dense attention whose scores may be capped, biased by distance and masked: what its kernels share.
//
//   s_ij = scale q_i . k_j      c_ij = cap tanh(s_ij / cap)  (s_ij without a cap)      x_ij = c_ij - slope_h |pos_i - j|
//   o_i = sum_j exp(x_ij - lse_i) v_j      lse_i = log sum_j exp(x_ij)      over the keys j of one run [lo_i, hi_i)
//
// Every mask there is (documents, a causal order, a prefix that all queries of a document see, keys behind a length) lets a
// query see ONE run of keys, so a mask is three numbers per query, and a tile of scores is whole, mixed or empty by four
// numbers per 64 queries.  Kernels work in units of log2: scores carry a factor log2(e), exp is ex2.
#pragma once
#include <cuda.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace lcbsa {

constexpr int kDenseCounters = 2;
constexpr int kDenseUnit = 64;              // rows of a query unit, keys of a key unit
constexpr int kDenseStats = 2 * kDenseUnit;  // floats of a query unit in the plan of the backward: -lse * log2(e) [64], -delta [64]
constexpr int kSeenPitch = kDenseUnit + 1;  // int4 of a query unit in the plan
constexpr uint32_t kBadRow = 0x7fc0dadau;    // a NaN in the place of -delta: the row's dout holds a value that is not finite
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What a query sees: keys [lo, hi); pos is its position among the keys.
struct Seen {
    int lo, hi, pos;
};

// The mask as the caller describes it.  cu_q, cu_k (both or neither): first query / key of every document of a batch entry, and the end of
// the last, docs + 1 numbers `cu_stride` apart per entry; without them the sequence is one document, with k_len[b] keys where that is given.
struct DenseMask {
    const int32_t *cu_q, *cu_k, *k_len, *prefix;
    int docs, causal;
    long long cu_stride, prefix_stride;  // per batch entry, 0: the same for all
};

struct DenseArgs {
    int dtype, B, Hq, Hk, group, D, Sq, Sk;
    View q, k, v, o, dout, dq, dk, dv;
    DenseMask mask;
    float scale, cap;
    int impl;              // LCBSA_ATTN_*
    const float* slopes;   // [Hq] or null
    float* lse;            // [B*Hq, Sq], natural log; nullable in the forward
    void* rest;            // nullable, dense [B, Hq, Sq, D] in the input type: what rounding the output left, for delta
    unsigned int* status;
    // carved out of the workspace (see dense_plan_kernel)
    int4* seen;            // [B, units, 65]: lo, hi, pos, 0 of a unit's 64 queries (those behind the last see nothing), then
                           // min lo, max hi over the queries that see a key, max lo, min hi over all of them
    int2* hulls;           // [B, key units]: first and one past the last query that can see a key of the unit (backward)
    float* stats;          // [B*Hq, units, 2, 64]: -lse * log2(e) and -rowsum(dout * out) of a unit's queries, -inf and 0 behind the last;
                           // kBadRow in the place of -delta where dout is not finite (backward)
    float* part;           // sums of dk and dv of parts of a group of heads (backward)
    int* next_item;        // items taken by the persistent kernels, zero when they start
};

__host__ __device__ __forceinline__ int dense_units(int n) { return (n + kDenseUnit - 1) / kDenseUnit; }

// Number of entries of cu[0 .. docs] that are <= x (the entries ascend).
__device__ __forceinline__ int dense_count_le(const int32_t* cu, int docs, int x) {
    int lo = 0, hi = docs + 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Whatever the bounds hold, the run lies inside [0, Sk).
__device__ __forceinline__ Seen dense_seen(const DenseMask& m, int b, int i, int Sq, int Sk) {
    int k0 = 0, k1 = Sk, q1 = Sq, d = 0;
    if (m.cu_q != nullptr) {
        const int32_t *cq = m.cu_q + b * m.cu_stride, *ck = m.cu_k + b * m.cu_stride;
        d = dense_count_le(cq, m.docs, i) - 1;
        if (d < 0 || d >= m.docs) return Seen{0, 0, 0};  // before the first document or behind the last
        k0 = min(max(__ldg(ck + d), 0), Sk);
        k1 = min(max(__ldg(ck + d + 1), k0), Sk);
        q1 = min(__ldg(cq + d + 1), Sq);
    } else if (m.k_len != nullptr) {
        k1 = min(max(__ldg(m.k_len + b), 0), Sk);
    }
    const int pos = k1 - (q1 - i);  // the last query of a document stands at its last key
    int hi = k1;
    if (m.causal) {
        const int pre = m.prefix != nullptr ? min(max(__ldg(m.prefix + b * m.prefix_stride + d), 0), Sk - k0) : 0;
        hi = min(max(max(pos + 1, k0 + pre), k0), k1);
    }
    return Seen{k0, hi, pos};
}

// A score in units of log2, as the exponent of its probability: x2 = scale log2(e) s, with a cap cap log2(e) tanh(y), y = scale s / cap.
//
//   |y| > 1/2: tanh(y) = 1 - t, t = 2 / (1 + exp(2 y)): two special functions, right at both ends (exp = inf: 1; exp = 0: -1), off by a few
//   2^-24 in between.  (The machine's own tanh is off by 2^-11, which a cap of 50 would make 2 % of a probability.)
//   |y| <= 1/2, where that difference would cost a large cap its small scores: tanh(y) = y p(y^2), p of degree 3 through the Chebyshev nodes
//   of [0, 1/4], off by 4.6 * 2^-23 of the value; with the powers of scale / cap (kept between 2^-20 and 2^20 by the entry) in its coefficients
//   x2 = s (c0 + t (c1 + t (c2 + t c3))), t = s^2: five operations of the arithmetic units, where the special functions (16 a clock and
//   SM, one per score already) would take twice as long as the rest of a tile.  Most tiles have no other scores and skip the first form.
//   At the low end of the range c3 is rounded to the grid of 2^-149, which moves x2 by 2^-150 s^7 <= 2^-17.  At the high end scale (scale / cap)^6
//   passes 2^128 for scales of 2^8 and more: there y = s scale / cap is formed first, the coefficients are those of y, and every tile takes
//   the way of the large scores.
struct ScoreShape {
    float mul;     // scale * log2(e)
    float mul_ex;  // 2 * scale / cap * log2(e)
    float cap2;    // cap * log2(e)
    float unit;    // 1, or scale / cap where the powers of that are not in the coefficients
    float c[4];    // of (unit s)
    float s_small; // scores up to this magnitude go through the polynomial
    float s_fast;  // s_small if the polynomial of s itself serves them, else -1: no score does without the factor `unit`
    float slope2;  // slope of the head * log2(e)
};
inline ScoreShape score_shape(float scale, float cap) {
    const double e = 1.4426950408889634, y = cap > 0.f ? (double)scale / cap : 0.0;
    const double p[4] = {0.9999994510270873, -0.3332628423141673, 0.13189939425594957, -0.044392738432622175};
    ScoreShape s;
    s.mul = (float)(scale * e);
    s.mul_ex = (float)(2.0 * y * e);
    s.cap2 = (float)(cap * e);
    const bool fits = std::fabs(scale * e * p[3] * y * y * y * y * y * y) < 0x1p127;  // the others are finite then, too
    s.unit = fits ? 1.f : (float)y;
    double f = fits ? scale * e : cap * e;
    for (int i = 0; i < 4; ++i, f *= fits ? y * y : 1.0) s.c[i] = (float)(f * p[i]);
    s.s_small = y != 0.0 ? (float)(0.5 / (y < 0 ? -y : y)) : 0.f;
    s.s_fast = fits ? s.s_small : -1.f;
    s.slope2 = 0.f;
    return s;
}
__device__ __forceinline__ float dense_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float dense_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two scores of at most s_fast, times the unit, -> cap log2(e) tanh(y) + c, and the same without c and with 1 - tanh(y)^2 (used by the backward)
__device__ __forceinline__ float2 capped_small_plus(const ScoreShape& f, float2 s, float2 c) {
    auto both = [](float x) { return make_float2(x, x); };
    const float2 t = __fmul2_rn(s, s);
    float2 p = __ffma2_rn(t, both(f.c[3]), both(f.c[2]));
    p = __ffma2_rn(p, t, both(f.c[1]));
    p = __ffma2_rn(p, t, both(f.c[0]));
    return __ffma2_rn(s, p, c);
}
__device__ __forceinline__ float2 capped_small(const ScoreShape& f, float2 s, float2& slack) {
    const float2 x = capped_small_plus(f, s, make_float2(0.f, 0.f));
    const float i = 1.f / f.cap2;
    const float2 t = __fmul2_rn(x, make_float2(i, i));
    slack = __ffma2_rn(t, make_float2(-t.x, -t.y), make_float2(1.f, 1.f));
    return x;
}

// Two scores of any size.  What a score comes to is a matter of the score alone, to the bit: a small one comes out as from the forms above, so a
// tile may take this way because of a score that is hidden from a row and change nothing of the row.
__device__ __forceinline__ float2 capped_large(const ScoreShape& f, float2 s, float2& t) {
    t = make_float2(2.f * dense_rcp(1.f + dense_ex2(s.x * f.mul_ex)), 2.f * dense_rcp(1.f + dense_ex2(s.y * f.mul_ex)));
    return __ffma2_rn(t, make_float2(-f.cap2, -f.cap2), make_float2(f.cap2, f.cap2));
}
__device__ __forceinline__ float2 capped_pick(const ScoreShape& f, float2 s, float2 small, float2 large) {
    return make_float2(fabsf(s.x) <= f.s_small ? small.x : large.x, fabsf(s.y) <= f.s_small ? small.y : large.y);
}
__device__ __forceinline__ float2 capped_any_plus(const ScoreShape& f, float2 s, float2 c) {
    float2 t;
    const float2 large = __fadd2_rn(capped_large(f, s, t), c);
    return capped_pick(f, s, capped_small_plus(f, __fmul2_rn(s, make_float2(f.unit, f.unit)), c), large);
}
__device__ __forceinline__ float2 capped_any(const ScoreShape& f, float2 s, float2& slack) {
    float2 t, small_slack;
    const float2 large = capped_large(f, s, t), small = capped_small(f, __fmul2_rn(s, make_float2(f.unit, f.unit)), small_slack);
    slack = capped_pick(f, s, small_slack, __fmul2_rn(t, __fadd2_rn(make_float2(2.f, 2.f), make_float2(-t.x, -t.y))));
    return capped_pick(f, s, small, large);
}

// The bias of n columns whose keys lie on one side of the query, plus a constant: plus - slope |at - j| is a line in the column's number j.
// Four chains of pairs, eight columns a step.
struct BiasLine {
    float2 c[4], step8;
};
// at <= 0: the keys are ahead; at >= n - 1: behind
__device__ __forceinline__ BiasLine bias_line(float at, float slope2, float plus) {
    const float sl = at > 0.f ? slope2 : -slope2, base = fmaf(-sl, at, plus);
    BiasLine l;
#pragma unroll
    for (int k = 0; k < 4; ++k) l.c[k] = make_float2(fmaf(sl, (float)(2 * k), base), fmaf(sl, (float)(2 * k + 1), base));
    l.step8 = make_float2(8.f * sl, 8.f * sl);
    return l;
}
// pair number k (columns 2k, 2k + 1), called once for each in ascending order
__device__ __forceinline__ float2 bias_next(BiasLine& l, int k) {
    const float2 v = l.c[k & 3];
    l.c[k & 3] = __fadd2_rn(v, l.step8);
    return v;
}

// Whether one of the eight 16-bit values of a 16-byte chunk is an infinity or a NaN (all exponent bits set).
template <typename T>
__device__ __forceinline__ bool chunk_nonfinite(const uint4& v) {
    constexpr uint32_t kExp = DType<T>::code == LCBSA_BF16 ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t kLow = DType<T>::code == LCBSA_BF16 ? 0x00800080u : 0x04000400u;
    // adding one to the exponent field of (v & kExp) carries out of it exactly when all its bits are set
    auto hot = [](uint32_t u) { return (((u & kExp) >> 1) + (kLow >> 1)) & 0x40004000u; };
    return (hot(v.x) | hot(v.y) | hot(v.z) | hot(v.w)) != 0;
}
// A warp: whether a tile of n 16-byte chunks holds one.  Every pair of values times zero is added up: 0, or NaN from the first infinity or
// NaN on; one instruction a pair (the test of the exponents takes four), so a tile of 16 KB takes some 170 instructions.
template <typename T, int n>
__device__ __forceinline__ bool tile_nonfinite(const uint4* tile, int lane) {
    using T2 = typename std::conditional<DType<T>::code == LCBSA_BF16, __nv_bfloat162, __half2>::type;
    const uint32_t z = 0u;
    const T2 zero = *reinterpret_cast<const T2*>(&z);
    T2 a0 = zero, a1 = zero, a2 = zero, a3 = zero;
#pragma unroll 8
    for (int c = lane; c < n; c += 32) {
        const uint4 v = tile[c];
        a0 = __hfma2(*reinterpret_cast<const T2*>(&v.x), zero, a0);
        a1 = __hfma2(*reinterpret_cast<const T2*>(&v.y), zero, a1);
        a2 = __hfma2(*reinterpret_cast<const T2*>(&v.z), zero, a2);
        a3 = __hfma2(*reinterpret_cast<const T2*>(&v.w), zero, a3);
    }
    const T2 a = __hadd2(__hadd2(a0, a1), __hadd2(a2, a3));
    return __any_sync(0xffffffffu, !__hbeq2(a, a));
}
template <typename T>
__device__ __forceinline__ uint32_t zero_nonfinite(uint32_t u) {
    constexpr uint32_t kExp = DType<T>::code == LCBSA_BF16 ? 0x7f80u : 0x7c00u;
    if ((u & kExp) == kExp) u &= 0xffff0000u;
    if (((u >> 16) & kExp) == kExp) u &= 0x0000ffffu;
    return u;
}

// The order of the items of a persistent kernel: waves of `wave` heads, in a wave tile by tile over its heads, so that the tiles with most work
// can come first and the last items are short.  One wave, unless what the heads stream (bytes each) does not fit the L2 together: then
// as few waves of as many heads as possible.  37 heads of 4096 tokens, 77 MB of keys and values: dQ 375 us in one wave, 336 us in waves of 10;
// 16 heads of 8192 tokens, 33 MB, causal: 343 us in one wave, 367 us in waves of 5, whose last one starts its longest items last.
inline int dense_wave(int heads, double bytes) {
    const int waves = (int)(heads * bytes / 48e6) + 1;
    return heads * bytes <= 64e6 ? heads : (heads + waves - 1) / waves;
}
__device__ __forceinline__ void dense_item(int idx, int heads, int tiles, int wave, int& bh, int& tile) {
    const int first = idx / (wave * tiles) * wave, rest = idx % (wave * tiles), n = min(wave, heads - first);
    tile = rest / n;
    bh = first + rest % n;
}

// the plan of a call (dense_plan.cu)
size_t dense_plan_bytes(const DenseArgs& a, bool backward);
void dense_plan_carve(DenseArgs& a, void* workspace, bool backward);
cudaError_t launch_dense_plan(const DenseArgs& a, cudaStream_t st);
// dense_few.cu: the entry to the forward, and the kernel for few queries; dense_tc.cu: the forward on tcgen05; dense_bwd_tc.cu: the backward
bool dense_supported(const DenseArgs& a, const char** why);
size_t dense_fwd_workspace_bytes(const DenseArgs& a);
cudaError_t launch_dense_fwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why);
bool dense_tc_supported(const DenseArgs& a);
cudaError_t launch_dense_tc(const DenseArgs& a, cudaStream_t st, const char** why);
// a tensor map over [B, H, S, D] rows in boxes of `box` rows x 64 columns (dense_tc.cu)
bool dense_rows_map(CUtensorMap* tm, int dtype, const View& v, int B, int H, int S, int D, int box, int* fold);
bool dense_bwd_supported(const DenseArgs& a, const char** why);
size_t dense_bwd_workspace_bytes(const DenseArgs& a);
cudaError_t launch_dense_bwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why);

}  // namespace lcbsa
