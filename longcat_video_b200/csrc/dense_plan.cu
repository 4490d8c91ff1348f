// The plan of a dense attention call: what its masks come to (see dense_common.cuh).
//
// What every query sees, in the order of the queries; per unit of 64 queries the union of the runs of its rows (min lo, max hi) and the
// run that all see (max lo, min hi); per unit of 64 keys the first and the last query that can see one of them, from the
// documents at its two ends.  A warp takes a query unit, a thread of the CTAs behind them a key unit.  The backward's row sums need none of it
// and ride in the same launch.  Bound by issue slots where the row sums are many: 37 heads of 2048 rows 15.6 us, 74 % of them busy, DRAM 46 % (three streams
// of 16 bytes a thread, one row per eight or sixteen lanes).
#include "dense_common.cuh"

namespace lcbsa {

namespace {

__device__ __forceinline__ void plan_cta(const DenseArgs& a, int cta, int b, int q_ctas) {
    if (cta == 0 && b == 0 && threadIdx.x < kDenseCounters) a.next_item[threadIdx.x] = 0;
    const int lane = threadIdx.x & 31, n_u = dense_units(a.Sq), n_k = dense_units(a.Sk);
    if (cta < q_ctas) {
        const int u = cta * 4 + (threadIdx.x >> 5);
        if (u >= n_u) return;
        int u_lo = 0x7fffffff, u_hi = 0, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = u * kDenseUnit + e * 32 + lane;
            Seen s{0, 0, 0};
            if (i < a.Sq) {  // rows behind the last query see nothing and count for nothing: whatever they come to is not stored
                s = dense_seen(a.mask, b, i, a.Sq, a.Sk);
                if (s.lo < s.hi) {
                    u_lo = min(u_lo, s.lo);
                    u_hi = max(u_hi, s.hi);
                    all_lo = max(all_lo, s.lo);
                    all_hi = min(all_hi, s.hi);
                } else {
                    all_hi = 0;
                }
            }
            a.seen[((long long)b * n_u + u) * kSeenPitch + e * 32 + lane] = make_int4(s.lo, s.hi, s.pos, 0);
        }
        u_lo = __reduce_min_sync(0xffffffffu, u_lo);
        u_hi = __reduce_max_sync(0xffffffffu, u_hi);
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        if (lane == 0) a.seen[((long long)b * n_u + u) * kSeenPitch + kDenseUnit] = make_int4(min(u_lo, u_hi), u_hi, all_lo, all_hi);
        return;
    }
    const int u = (cta - q_ctas) * 128 + threadIdx.x;
    if (u >= n_k) return;
    const DenseMask& m = a.mask;
    const int k_first = u * kDenseUnit, k_last = min(k_first + kDenseUnit, a.Sk) - 1;
    int d = 0, k0 = 0, k1 = a.Sk, q0 = 0, q1 = a.Sq, q_end = a.Sq;
    if (m.cu_q != nullptr) {
        const int32_t *cq = m.cu_q + b * m.cu_stride, *ck = m.cu_k + b * m.cu_stride;
        d = max(dense_count_le(ck, m.docs, k_first) - 1, 0);
        const int d1 = min(dense_count_le(ck, m.docs, k_last) - 1, m.docs - 1);
        if (d > d1) {
            a.hulls[(long long)b * n_k + u] = make_int2(0, 0);
            return;
        }
        k0 = min(max(__ldg(ck + d), 0), a.Sk);
        k1 = min(max(__ldg(ck + d + 1), k0), a.Sk);
        q0 = __ldg(cq + d);
        q1 = min(max(__ldg(cq + d + 1), 0), a.Sq);
        q_end = __ldg(cq + d1 + 1);
    } else if (m.k_len != nullptr) {
        k1 = min(max(__ldg(m.k_len + b), 0), a.Sk);
        if (k_first >= k1) q_end = 0;
    }
    if (m.causal) {
        const int pre = m.prefix != nullptr ? min(max(__ldg(m.prefix + b * m.prefix_stride + d), 0), a.Sk - k0) : 0;
        const int key = max(k_first, k0);
        if (key >= k0 + pre) q0 = max(q0, q1 - (k1 - key));
    }
    q0 = min(max(q0, 0), a.Sq);
    a.hulls[(long long)b * n_k + u] = make_int2(q0, min(max(q_end, q0), a.Sq));
}

// Backward: rowsum(dout * out) in fp32, out with what its rounding left: a half step of out moves dS by as much as rounding dS does (dq
// of a causal row of 600 keys, bf16, is off by 1.53 times its own rounding without the rest, 1.46 with it).  D / 8 lanes a row; rows
// behind the last query get a probability of zero (-lse of -inf) whatever their distance to a key counts for: their entries are not
// masked in a unit that is whole.
template <typename T, int D>
__device__ __forceinline__ void stats_cta(const DenseArgs& a, long long cta) {
    constexpr int kLanes = D / 8;
    const int sub = threadIdx.x % kLanes;
    const long long r = cta * (128 / kLanes) + threadIdx.x / kLanes;  // (b * Hq + h) * units * 64 + row of the unit: whole CTAs of them
    const int n_u = dense_units(a.Sq);
    float s = 0.f;
    bool bad = false;
    const long long bh = r / ((long long)n_u * kDenseUnit);
    const int i = (int)(r % ((long long)n_u * kDenseUnit)), b = (int)(bh / a.Hq), h = (int)(bh % a.Hq);
    if (i < a.Sq) {
        const uint4 o = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.o.data) + b * a.o.sb + h * a.o.sh + i * a.o.ss + sub * 8);
        const uint4 g = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.dout.data) + b * a.dout.sb + h * a.dout.sh + i * a.dout.ss + sub * 8);
        uint4 left = make_uint4(0u, 0u, 0u, 0u);
        if (a.rest != nullptr) left = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.rest) + (bh * a.Sq + i) * D + sub * 8);
        bad = chunk_nonfinite<T>(g);
        const T *op = reinterpret_cast<const T*>(&o), *gp = reinterpret_cast<const T*>(&g), *lp = reinterpret_cast<const T*>(&left);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(DType<T>::to_f32(op[e]) + DType<T>::to_f32(lp[e]), DType<T>::to_f32(gp[e]), s);
    }
#pragma unroll
    for (int x = kLanes / 2; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    bad = (__ballot_sync(0xffffffffu, bad) >> (threadIdx.x & 31 & ~(kLanes - 1)) & ((1u << kLanes) - 1u)) != 0u;
    if (sub == 0) {
        float* dst = a.stats + r / kDenseUnit * kDenseStats + r % kDenseUnit;
        dst[0] = i < a.Sq ? -(a.lse[bh * a.Sq + i] * kLog2e) : -INFINITY;
        dst[kDenseUnit] = bad ? __uint_as_float(kBadRow) : i < a.Sq ? -s : 0.f;
    }
}

// The plan's CTAs first (per batch entry q_ctas for the query units, then those of the key units), the backward's row sums behind them.
template <typename T, int D>
__global__ void __launch_bounds__(128) dense_plan_kernel(const __grid_constant__ DenseArgs a, int q_ctas, int entry_ctas) {
    const int planned = entry_ctas * a.B;
    if ((int)blockIdx.x < planned) plan_cta(a, blockIdx.x % entry_ctas, blockIdx.x / entry_ctas, q_ctas);
    else stats_cta<T, D>(a, (long long)blockIdx.x - planned);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t dense_plan_bytes(const DenseArgs& a, bool backward) {
    const size_t n_u = dense_units(a.Sq), n_k = dense_units(a.Sk);
    return 256 + align256(a.B * n_u * kSeenPitch * sizeof(int4)) + (backward ? align256(a.B * n_k * sizeof(int2)) : 0);
}

void dense_plan_carve(DenseArgs& a, void* workspace, bool backward) {
    const size_t n_u = dense_units(a.Sq);
    unsigned char* w = static_cast<unsigned char*>(workspace);
    a.next_item = reinterpret_cast<int*>(w);
    w += 256;
    a.seen = reinterpret_cast<int4*>(w);
    w += align256(a.B * n_u * kSeenPitch * sizeof(int4));
    a.hulls = backward ? reinterpret_cast<int2*>(w) : nullptr;
}

cudaError_t launch_dense_plan(const DenseArgs& a, cudaStream_t st) {
    const int q_ctas = (dense_units(a.Sq) + 3) / 4, entry_ctas = q_ctas + (a.hulls != nullptr ? (dense_units(a.Sk) + 127) / 128 : 0);
    const long long rows = a.hulls != nullptr ? (long long)a.B * a.Hq * dense_units(a.Sq) * kDenseUnit : 0;
    const long long ctas = (long long)entry_ctas * a.B + rows * (a.D / 8) / 128;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    if (ctas == 0) return cudaSuccess;
    if (a.dtype == LCBSA_BF16) {
        if (a.D == 128) dense_plan_kernel<__nv_bfloat16, 128><<<(unsigned)ctas, 128, 0, st>>>(a, q_ctas, entry_ctas);
        else dense_plan_kernel<__nv_bfloat16, 64><<<(unsigned)ctas, 128, 0, st>>>(a, q_ctas, entry_ctas);
    } else {
        if (a.D == 128) dense_plan_kernel<__half, 128><<<(unsigned)ctas, 128, 0, st>>>(a, q_ctas, entry_ctas);
        else dense_plan_kernel<__half, 64><<<(unsigned)ctas, 128, 0, st>>>(a, q_ctas, entry_ctas);
    }
    return cudaGetLastError();
}

}  // namespace lcbsa
