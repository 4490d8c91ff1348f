// Dense attention backward (see dense_common.cuh for the forward's formulas): dq, dk, dv from dout, the output and the lse.
//
//   delta_i = dout_i . o_i        p_ij = exp(x_ij - lse_i)        dv_j = sum_i p_ij dout_i
//   ds_ij = p_ij (dout_i . v_j - delta_i) (1 - tanh^2(s_ij / cap)) scale        dq_i = sum_j ds_ij k_j        dk_j = sum_i ds_ij q_i
//
// dk_j and dv_j also add up over the query heads that share the key head.  Two passes, so that every gradient is summed by one CTA in
// one order and nothing is added with atomics: a CTA of the first owns 64 queries and walks the keys that they see, a CTA of
// the second owns 64 keys and walks the queries that may see them, head after head.  S and dP are computed in both.
// 64 x 64 tiles on mma.sync m16n8k16, four warps of 16 rows, the streamed tiles double-buffered with cp.async; S, dP, P and dS stay in
// registers, where the accumulator layout of one product is the A operand of the next; P and dS are rounded to the input type for it.
//
// Masked places hold anything: a masked pair's P and dS are set to zero, and in tiles that only some rows see, values that are not finite
// are taken out of the operand of the second product once the first has read it (0 * inf is not 0).  A pair that is seen has its NaN from
// the first product; for dv it is the query's delta that says that dout_i is not finite.
#include "dense_common.cuh"
#include "mma_common.cuh"

namespace lcbsa {

namespace {

constexpr int kTile = kDenseUnit;
constexpr int kBwdThreads = 128;

// ------------------------------------------------------------------------------------------ the plan
//
// What every query sees, in the order of the queries; per unit of 64 queries the union of the runs of its rows (min lo, max hi) and the
// run that all see (max lo, min hi); per unit of 64 keys the first and the last query that can see one of them, from the
// documents at its two ends.  A warp takes a query unit, a thread of the CTAs behind them a key unit.
__global__ void __launch_bounds__(128) dense_plan_kernel(const __grid_constant__ DenseArgs a, int q_ctas) {
    const int b = blockIdx.y, lane = threadIdx.x & 31, n_u = dense_units(a.Sq), n_k = dense_units(a.Sk);
    if ((int)blockIdx.x < q_ctas) {
        const int u = blockIdx.x * 4 + (threadIdx.x >> 5);
        if (u >= n_u) return;
        int u_lo = 0x7fffffff, u_hi = 0, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = u * kTile + e * 32 + lane;
            Seen s{0, 0, 0};
            if (i < a.Sq) s = dense_seen(a.mask, b, i, a.Sq, a.Sk);
            a.rows[(long long)b * n_u * kTile + i] = make_int4(s.lo, s.hi, s.pos, 0);
            if (s.lo < s.hi) {
                u_lo = min(u_lo, s.lo);
                u_hi = max(u_hi, s.hi);
                all_lo = max(all_lo, s.lo);
                all_hi = min(all_hi, s.hi);
            } else {
                all_hi = 0;
            }
        }
        u_lo = __reduce_min_sync(0xffffffffu, u_lo);
        u_hi = __reduce_max_sync(0xffffffffu, u_hi);
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        if (lane == 0) a.units[(long long)b * n_u + u] = make_int4(min(u_lo, u_hi), u_hi, all_lo, all_hi);
        return;
    }
    const int u = (blockIdx.x - q_ctas) * 128 + threadIdx.x;
    if (u >= n_k) return;
    const DenseMask& m = a.mask;
    const int k_first = u * kTile, k_last = min(k_first + kTile, a.Sk) - 1;
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
        q1 = __ldg(cq + d + 1);
        q_end = __ldg(cq + d1 + 1);
    } else if (m.k_len != nullptr) {
        k1 = min(max(__ldg(m.k_len + b), 0), a.Sk);
        if (k_first >= k1) q_end = 0;
    }
    if (m.causal) {
        const int pre = m.prefix != nullptr ? min(max(__ldg(m.prefix + b * m.prefix_stride + d), 0), a.Sk) : 0;
        const int key = max(k_first, k0);
        if (key >= k0 + pre) q0 = max(q0, q1 - (k1 - key));
    }
    q0 = min(max(q0, 0), a.Sq);
    a.hulls[(long long)b * n_k + u] = make_int2(q0, min(max(q_end, q0), a.Sq));
}

// One warp per query row: rowsum(dout * out) in fp32.
template <typename T, int D>
__global__ void __launch_bounds__(256) dense_delta_kernel(const __grid_constant__ DenseArgs a) {
    constexpr int kPer = D / 32;
    const int lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= (long long)a.B * a.Hq * a.Sq) return;
    const int i = (int)(r % a.Sq), bh = (int)(r / a.Sq), b = bh / a.Hq, h = bh % a.Hq;
    const T* o = static_cast<const T*>(a.o.data) + b * a.o.sb + h * a.o.sh + i * a.o.ss + lane * kPer;
    const T* g = static_cast<const T*>(a.dout.data) + b * a.dout.sb + h * a.dout.sh + i * a.dout.ss + lane * kPer;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) s = fmaf(DType<T>::to_f32(o[e]), DType<T>::to_f32(g[e]), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (lane == 0) a.delta[r] = s;
}

// ------------------------------------------------------------------------------------------ the two passes

// 64 rows from row `first` on into a swizzled [64][D] tile; rows outside [lo, hi) are zero
template <typename T, int D>
__device__ __forceinline__ void load_rows(unsigned char* tile, const T* head, long long ss, int first, int lo, int hi, int tid) {
    constexpr int CPR = D * 2 / 16;
    const uint32_t base = mm::smem_u32(tile);
#pragma unroll
    for (int v = tid; v < kTile * CPR; v += kBwdThreads) {
        const int r = v / CPR, c = v % CPR, row = first + r;
        const bool there = row >= lo && row < hi;
        mm::cp_async16(base + r * (D * 2) + ((c ^ (r & 7)) << 4), head + (there ? (long long)row * ss : 0) + c * 8, there);
    }
}

template <typename T, int D>
__device__ __forceinline__ void store_rows(const unsigned char* tile, T* head, long long ss, int first, int hi, int tid) {
    constexpr int CPR = D * 2 / 16;
    for (int v = tid; v < kTile * CPR; v += kBwdThreads) {
        const int r = v / CPR, c = v % CPR;
        if (first + r < hi)
            *reinterpret_cast<uint4*>(head + (long long)(first + r) * ss + c * 8) =
                *reinterpret_cast<const uint4*>(tile + r * (D * 2) + ((c ^ (r & 7)) << 4));
    }
}

// All threads: values of a tile (or of two) that are not finite become zero.  Contains barriers; the tile is read by nobody before.
template <typename T, int kBytes>
__device__ __forceinline__ void scrub(unsigned char* t0, unsigned char* t1, int tid) {
    bool bad = false;
#pragma unroll 4
    for (int v = tid; v < kBytes / 16; v += kBwdThreads) {
        bad |= chunk_nonfinite<T>(reinterpret_cast<const uint4*>(t0)[v]);
        if (t1 != nullptr) bad |= chunk_nonfinite<T>(reinterpret_cast<const uint4*>(t1)[v]);
    }
    if (!__syncthreads_or(bad)) return;
    for (int v = tid; v < kBytes / 4; v += kBwdThreads) {
        uint32_t* p = reinterpret_cast<uint32_t*>(t0) + v;
        *p = zero_nonfinite<T>(*p);
        if (t1 != nullptr) {
            p = reinterpret_cast<uint32_t*>(t1) + v;
            *p = zero_nonfinite<T>(*p);
        }
    }
    __syncthreads();
}

template <int D> constexpr int bwd_smem() { return 6 * kTile * D * 2 + 2 * kTile * (16 + 8); }

template <typename T, int D, bool kCap, bool kBias>
__global__ void __launch_bounds__(kBwdThreads, 2) dense_dq_kernel(const __grid_constant__ DenseArgs a, const ScoreShape shape) {
    constexpr int kTB = kTile * D * 2;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const q_s = smem;  // later the staged dQ
    unsigned char* const do_s = q_s + kTB;
    unsigned char* const k_s = do_s + kTB;      // [2]
    unsigned char* const v_s = k_s + 2 * kTB;   // [2]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_u = dense_units(a.Sq);
    const int u = n_u - 1 - (int)(blockIdx.x % n_u);  // with a causal order the last queries have most keys: they start first
    const int bh = blockIdx.x / n_u, b = bh / a.Hq, h = bh % a.Hq, hk = h / a.group;
    const T* const qh = static_cast<const T*>(a.q.data) + b * a.q.sb + h * a.q.sh;
    const T* const doh = static_cast<const T*>(a.dout.data) + b * a.dout.sb + h * a.dout.sh;
    const T* const kh = static_cast<const T*>(a.k.data) + b * a.k.sb + hk * a.k.sh;
    const T* const vh = static_cast<const T*>(a.v.data) + b * a.v.sb + hk * a.v.sh;
    T* const dqh = static_cast<T*>(const_cast<void*>(a.dq.data)) + b * a.dq.sb + h * a.dq.sh;
    const int4 un = a.units[(long long)b * n_u + u];
    const int n_tiles = un.y > un.x ? (un.y - un.x + kTile - 1) / kTile : 0;

    load_rows<T, D>(q_s, qh, a.q.ss, u * kTile, 0, a.Sq, tid);
    load_rows<T, D>(do_s, doh, a.dout.ss, u * kTile, 0, a.Sq, tid);
    mm::cp_async_commit();
    if (n_tiles > 0) {
        load_rows<T, D>(k_s, kh, a.k.ss, un.x, un.x, un.y, tid);
        load_rows<T, D>(v_s, vh, a.v.ss, un.x, un.x, un.y, tid);
    }
    mm::cp_async_commit();
    mm::cp_async_wait<1>();
    __syncthreads();
    uint32_t qf[D / 16][4], dof[D / 16][4];
    mm::load_a_frags<D>(qf, mm::smem_u32(q_s), warp, lane);
    mm::load_a_frags<D>(dof, mm::smem_u32(do_s), warp, lane);

    int4 seen[2];
    float lse2[2], dl[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = u * kTile + warp * 16 + (lane >> 2) + 8 * e;
        seen[e] = a.rows[(long long)b * n_u * kTile + i];
        const bool there = i < a.Sq;
        lse2[e] = there ? a.lse[(long long)bh * a.Sq + i] * kLog2e : 0.f;
        dl[e] = there ? a.delta[(long long)bh * a.Sq + i] : 0.f;
    }
    ScoreShape f = shape;
    if (kBias) f.slope2 = __ldg(a.slopes + h) * kLog2e;

    float dq[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) dq[i][0] = dq[i][1] = dq[i][2] = dq[i][3] = 0.f;

    for (int it = 0; it < n_tiles; ++it) {
        const int buf = it & 1, key0 = un.x + it * kTile;
        if (it + 1 < n_tiles) {
            load_rows<T, D>(k_s + (buf ^ 1) * kTB, kh, a.k.ss, key0 + kTile, un.x, un.y, tid);
            load_rows<T, D>(v_s + (buf ^ 1) * kTB, vh, a.v.ss, key0 + kTile, un.x, un.y, tid);
        }
        mm::cp_async_commit();
        mm::cp_async_wait<1>();
        __syncthreads();
        const uint32_t kt = mm::smem_u32(k_s) + buf * kTB, vt = mm::smem_u32(v_s) + buf * kTB;
        const bool mixed = key0 < un.z || key0 + kTile > un.w;
        float s[8][4], dp[8][4];
        mm::mma_abt2<T, D>(s, dp, qf, dof, kt, vt, lane);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = key0 + nt * 8 + 2 * (lane & 3) + (e & 1), r = e >> 1;
                float t2 = 0.f;
                const float x = shaped_score<kCap, kBias>(f, s[nt][e], fabsf((float)(seen[r].z - j)), t2);
                float ds = dense_ex2(x - lse2[r]) * (dp[nt][e] - dl[r]) * a.scale;
                if (kCap) ds *= t2 * (2.f - t2);
                if (mixed && (j < seen[r].x || j >= seen[r].y)) ds = 0.f;
                dp[nt][e] = ds;
            }
        }
        if (mixed) scrub<T, kTB>(k_s + buf * kTB, nullptr, tid);
        mm::mma_xb<T, D>(dq, dp, kt, lane);  // dQ += dS K
        __syncthreads();
    }
    mm::cp_async_wait<0>();
    __syncthreads();
    mm::stage_rows<T, D>(q_s, dq, warp, lane);
    __syncthreads();
    store_rows<T, D>(q_s, dqh, a.dq.ss, u * kTile, a.Sq, tid);
}

template <typename T, int D, bool kCap, bool kBias>
__global__ void __launch_bounds__(kBwdThreads, 2) dense_dkdv_kernel(const __grid_constant__ DenseArgs a, const ScoreShape shape) {
    constexpr int kTB = kTile * D * 2;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const k_s = smem;            // later the staged dK
    unsigned char* const v_s = k_s + kTB;       // later the staged dV
    unsigned char* const q_s = v_s + kTB;       // [2]
    unsigned char* const do_s = q_s + 2 * kTB;  // [2]
    int4* const seen_s = reinterpret_cast<int4*>(do_s + 2 * kTB);           // [2][64]
    float2* const ld_s = reinterpret_cast<float2*>(seen_s + 2 * kTile);     // [2][64] lse * log2(e), delta
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_u = dense_units(a.Sq), n_k = dense_units(a.Sk);
    const int u = blockIdx.x % n_k;  // with a causal order the first keys have most queries
    const int bh = blockIdx.x / n_k, b = bh / a.Hk, hk = bh % a.Hk;
    const int key0 = u * kTile;
    const T* const kh = static_cast<const T*>(a.k.data) + b * a.k.sb + hk * a.k.sh;
    const T* const vh = static_cast<const T*>(a.v.data) + b * a.v.sb + hk * a.v.sh;
    const int2 hull = a.hulls[(long long)b * n_k + u];
    const int u_first = hull.x / kTile, u_count = hull.y > hull.x ? (hull.y - 1) / kTile - u_first + 1 : 0;
    const int4* const units = a.units + (long long)b * n_u;

    // the next (head, query unit) behind `at` of which some row sees one of the keys; at = head * u_count + unit
    const int total = u_count * a.group;
    auto next = [&](int at) {
        while (at < total) {
            const int4 un = units[u_first + at % u_count];
            if (un.x < key0 + kTile && un.y > key0 && un.x < un.y) break;
            ++at;
        }
        return at;
    };
    auto request = [&](int at, int buf) {
        const int h = hk * a.group + at / u_count, qu = u_first + at % u_count, i0 = qu * kTile;
        load_rows<T, D>(q_s + buf * kTB, static_cast<const T*>(a.q.data) + b * a.q.sb + h * a.q.sh, a.q.ss, i0, 0, a.Sq, tid);
        load_rows<T, D>(do_s + buf * kTB, static_cast<const T*>(a.dout.data) + b * a.dout.sb + h * a.dout.sh, a.dout.ss, i0, 0, a.Sq, tid);
        if (tid < kTile) {
            seen_s[buf * kTile + tid] = a.rows[(long long)b * n_u * kTile + i0 + tid];
            const long long r = ((long long)b * a.Hq + h) * a.Sq + i0 + tid;
            const bool there = i0 + tid < a.Sq;
            ld_s[buf * kTile + tid] = there ? make_float2(a.lse[r] * kLog2e, a.delta[r]) : make_float2(0.f, 0.f);
        }
    };
    load_rows<T, D>(k_s, kh, a.k.ss, key0, 0, a.Sk, tid);
    load_rows<T, D>(v_s, vh, a.v.ss, key0, 0, a.Sk, tid);
    mm::cp_async_commit();
    int at = next(0);
    if (at < total) request(at, 0);
    mm::cp_async_commit();
    mm::cp_async_wait<1>();
    __syncthreads();

    float dk[D / 8][4], dv[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
        dk[i][0] = dk[i][1] = dk[i][2] = dk[i][3] = 0.f;
        dv[i][0] = dv[i][1] = dv[i][2] = dv[i][3] = 0.f;
    }
    ScoreShape f = shape;
    for (int buf = 0; at < total; buf ^= 1) {
        const int nx = next(at + 1);
        if (nx < total) request(nx, buf ^ 1);
        mm::cp_async_commit();
        mm::cp_async_wait<1>();
        __syncthreads();
        if (kBias) f.slope2 = __ldg(a.slopes + hk * a.group + at / u_count) * kLog2e;
        const int4 un = units[u_first + at % u_count];
        const bool mixed = key0 < un.z || key0 + kTile > un.w;
        const uint32_t qt = mm::smem_u32(q_s) + buf * kTB, dot = mm::smem_u32(do_s) + buf * kTB;
        const int4* const sn = seen_s + buf * kTile;
        const float2* const ld = ld_s + buf * kTile;
        float st[8][4], dpt[8][4];
        mm::mma_abt2_sa<T, D>(st, dpt, mm::smem_u32(k_s), mm::smem_u32(v_s), qt, dot, warp, lane);
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = nt * 8 + 2 * (lane & 3) + (e & 1), j = key0 + warp * 16 + (lane >> 2) + 8 * (e >> 1);
                const int4 se = sn[col];
                const float2 l = ld[col];
                float t2 = 0.f;
                const float x = shaped_score<kCap, kBias>(f, st[nt][e], fabsf((float)(se.z - j)), t2);
                float p = dense_ex2(x - l.x);
                float ds = p * (dpt[nt][e] - l.y) * a.scale;
                if (kCap) ds *= t2 * (2.f - t2);
                if (mixed) {
                    if (!isfinite(l.y)) p = __int_as_float(0x7fc00000);
                    if (j < se.x || j >= se.y) p = ds = 0.f;
                }
                st[nt][e] = p;
                dpt[nt][e] = ds;
            }
        }
        if (mixed) scrub<T, kTB>(q_s + buf * kTB, do_s + buf * kTB, tid);
        mm::mma_xb2<T, D>(dv, st, dot, dk, dpt, qt, lane);  // dV += P^T dO, dK += dS^T Q
        __syncthreads();
        at = nx;
    }
    mm::cp_async_wait<0>();
    __syncthreads();
    mm::stage_rows<T, D>(k_s, dk, warp, lane);
    mm::stage_rows<T, D>(v_s, dv, warp, lane);
    __syncthreads();
    store_rows<T, D>(k_s, static_cast<T*>(const_cast<void*>(a.dk.data)) + b * a.dk.sb + hk * a.dk.sh, a.dk.ss, key0, a.Sk, tid);
    store_rows<T, D>(v_s, static_cast<T*>(const_cast<void*>(a.dv.data)) + b * a.dv.sb + hk * a.dv.sh, a.dv.ss, key0, a.Sk, tid);
}

template <typename T, int D, bool kCap, bool kBias>
cudaError_t passes(const DenseArgs& a, cudaStream_t st) {
    static thread_local unsigned long long raised = 0;  // devices (below 64) whose shared-memory limit this thread has raised for these kernels
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !((raised >> dev) & 1)) {
        e = cudaFuncSetAttribute(dense_dq_kernel<T, D, kCap, kBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, bwd_smem<D>());
        if (e == cudaSuccess) e = cudaFuncSetAttribute(dense_dkdv_kernel<T, D, kCap, kBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, bwd_smem<D>());
        if (e != cudaSuccess) return e;
        if (dev <= 63) raised |= 1ull << dev;
    }
    const ScoreShape shape = score_shape(a.scale, a.cap);
    const long long ctas_q = (long long)a.B * a.Hq * dense_units(a.Sq), ctas_k = (long long)a.B * a.Hk * dense_units(a.Sk);
    if (ctas_q > 0x7fffffffll || ctas_k > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    if (ctas_q > 0) dense_dq_kernel<T, D, kCap, kBias><<<(unsigned)ctas_q, kBwdThreads, bwd_smem<D>(), st>>>(a, shape);
    if (ctas_k > 0) dense_dkdv_kernel<T, D, kCap, kBias><<<(unsigned)ctas_k, kBwdThreads, bwd_smem<D>(), st>>>(a, shape);
    return cudaGetLastError();
}

template <typename T, int D>
cudaError_t backward(const DenseArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.B * a.Hq * a.Sq;
    if ((rows + 7) / 8 > 0x7fffffffll || a.B > 65535) return cudaErrorInvalidConfiguration;
    const int q_ctas = (dense_units(a.Sq) + 3) / 4, k_ctas = (dense_units(a.Sk) + 127) / 128;
    if (q_ctas + k_ctas > 0) dense_plan_kernel<<<dim3(q_ctas + k_ctas, a.B), 128, 0, st>>>(a, q_ctas);
    if (rows > 0) dense_delta_kernel<T, D><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
    if (cap) return bias ? passes<T, D, true, true>(a, st) : passes<T, D, true, false>(a, st);
    return bias ? passes<T, D, false, true>(a, st) : passes<T, D, false, false>(a, st);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t dense_bwd_workspace_bytes(const DenseArgs& a) {
    const size_t n_u = dense_units(a.Sq), n_k = dense_units(a.Sk);
    return align256(a.B * n_u * kTile * sizeof(int4)) + align256(a.B * n_u * sizeof(int4)) + align256(a.B * n_k * sizeof(int2)) +
           align256((size_t)a.B * a.Hq * a.Sq * sizeof(float));
}

cudaError_t launch_dense_bwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why) {
    if (a.B * a.Hq == 0) return cudaSuccess;
    const size_t n_u = dense_units(a.Sq), n_k = dense_units(a.Sk);
    unsigned char* w = static_cast<unsigned char*>(workspace);
    a.rows = reinterpret_cast<int4*>(w);
    w += align256(a.B * n_u * kTile * sizeof(int4));
    a.units = reinterpret_cast<int4*>(w);
    w += align256(a.B * n_u * sizeof(int4));
    a.hulls = reinterpret_cast<int2*>(w);
    w += align256(a.B * n_k * sizeof(int2));
    a.delta = reinterpret_cast<float*>(w);
    const cudaError_t e = a.dtype == LCBSA_BF16 ? (a.D == 128 ? backward<__nv_bfloat16, 128>(a, st) : backward<__nv_bfloat16, 64>(a, st))
                                                : (a.D == 128 ? backward<__half, 128>(a, st) : backward<__half, 64>(a, st));
    if (e == cudaErrorInvalidConfiguration) *why = "more CTAs than a launch takes";
    return e;
}

}  // namespace lcbsa
