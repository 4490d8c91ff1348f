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

// One warp per query row: rowsum(dout * out) in fp32, out with what its rounding left (a half step of out moves dS by as much as
// rounding dS does: dq of a causal row of 600 keys, bf16, is off by 1.53 times its own rounding without it, 1.46 with it).
template <typename T, int D>
__global__ void __launch_bounds__(256) dense_delta_kernel(const __grid_constant__ DenseArgs a) {
    constexpr int kPer = D / 32;
    const int lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= (long long)a.B * a.Hq * a.Sq) return;
    const int i = (int)(r % a.Sq), bh = (int)(r / a.Sq), b = bh / a.Hq, h = bh % a.Hq;
    const T* o = static_cast<const T*>(a.o.data) + b * a.o.sb + h * a.o.sh + i * a.o.ss + lane * kPer;
    const T* g = static_cast<const T*>(a.dout.data) + b * a.dout.sb + h * a.dout.sh + i * a.dout.ss + lane * kPer;
    const T* left = a.rest != nullptr ? static_cast<const T*>(a.rest) + r * D + lane * kPer : nullptr;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        float v = DType<T>::to_f32(o[e]);
        if (left != nullptr) v += DType<T>::to_f32(left[e]);
        s = fmaf(v, DType<T>::to_f32(g[e]), s);
    }
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
    if ((rows + 7) / 8 > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaError_t e = launch_dense_plan(a, st);
    if (e != cudaSuccess) return e;
    if (rows > 0) dense_delta_kernel<T, D><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
    if (cap) return bias ? passes<T, D, true, true>(a, st) : passes<T, D, true, false>(a, st);
    return bias ? passes<T, D, false, true>(a, st) : passes<T, D, false, false>(a, st);
}

}  // namespace

size_t dense_bwd_workspace_bytes(const DenseArgs& a) { return dense_plan_bytes(a, true) + (size_t)a.B * a.Hq * a.Sq * sizeof(float); }

cudaError_t launch_dense_bwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why) {
    if (a.B * a.Hq == 0) return cudaSuccess;
    dense_plan_carve(a, workspace, true);
    a.delta = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + dense_plan_bytes(a, true));
    const cudaError_t e = a.dtype == LCBSA_BF16 ? (a.D == 128 ? backward<__nv_bfloat16, 128>(a, st) : backward<__nv_bfloat16, 64>(a, st))
                                                : (a.D == 128 ? backward<__half, 128>(a, st) : backward<__half, 64>(a, st));
    if (e == cudaErrorInvalidConfiguration) *why = "more CTAs than a launch takes";
    return e;
}

}  // namespace lcbsa
