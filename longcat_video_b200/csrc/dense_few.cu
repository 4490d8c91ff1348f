// Dense attention forward for few queries (see dense_common.cuh for the formulas): a token, or a few drafted ones, of every sequence
// behind a long cache.  Bound by HBM: each key and value is read once for all queries and all heads that share it.
//
// The rows of a CTA's one or two 16-row MMA tiles are (query, head of the group) pairs, so a group of four heads and one query fill
// four of them and the cache is still read once.  The keys that the rows see are split evenly over the CTAs of a cluster, which join
// their partial results (fp32, relative to their maxima) through each other's shared memory: one launch, no workspace, one order.
// Where clusters of eight leave the chip idle and the keys are many, chunks of a fixed number of keys go to CTAs of their own
// instead, and a second kernel joins partial results from the workspace.  Inside a CTA four warps (eight at head_dim 64) take
// tiles of 16 keys in turn: a warp has a ring of its own in shared memory and nothing in the loop waits for another warp.  S, P and O
// stay in registers (mma.sync m16n8k16, fp32 accumulators; P is rounded to the input type for the product with V, as in the
// other attention kernels, the row sum is taken before the rounding); running maximum and sum per row in fp32.
//
// One token behind 32 caches of 8192 to 32768 keys, 8 key heads of 128 (2.8 GB): 395 us, 7.0 TB/s; 32 caches of 8192 keys under the profiler: 162
// us, 81 % of the DRAM rate.  Small calls are bound by latency, one chain of mask, copies, products and join: 6 us behind 1023 keys.
//
// Masked places hold anything: keys outside the union of the rows' runs are not loaded, a masked score is replaced (not
// multiplied), and in a tile that only some rows see the values that are not finite are added by hand to the rows that see
// them and are zero for the product, so that 0 * inf reaches no row that does not.
#include "dense_common.cuh"
#include "mma_common.cuh"

namespace lcbsa {

namespace {

template <int D> constexpr int kFewWarps = D == 64 ? 8 : 4;
constexpr int kFewStages = 3;   // tiles of a warp's ring, of K and V each
constexpr int kKeys = 16;       // keys of a warp's tile
constexpr int kMaxCluster = 8;  // CTAs of a cluster (16, which have to be asked for, start one after another: 20 us became 32)
constexpr int kMaxSplits = 256;
constexpr int few_step(int D) { return (D == 64 ? 8 : 4) * kKeys; }  // keys of a CTA's round

struct FewParams {
    DenseArgs a;
    ScoreShape shape;
    int rows;               // group * Sq rows of one key head
    int mt;                 // 16-row tiles of a CTA
    int tiles;              // CTAs' worth of rows
    int splits, chunk;      // CTAs that share the keys; chunk: keys of each, 0: a cluster, which splits evenly what its rows see
    float* part_o;          // [B*Hk*rows][splits][D], not yet divided by the row sum (chunks)
    float2* part_ml;        // [B*Hk*rows][splits]: maximum (log2), row sum
};

template <int D, int MT>
constexpr int few_smem() {
    return 16 * MT * D * 2 + kFewWarps<D> * kFewStages * 2 * kKeys * D * 2 + 16 * MT * 16;
}

// A warp's rows `first` .. of K or V into a swizzled tile; rows at `end` or behind are zero.  src: where this lane's 16 bytes of row
// first + lane / (chunks of a row) are, if there is such a row; head: an address that there is.
template <typename T, int D>
__device__ __forceinline__ void load_keys(uint32_t tile, const T* src, const T* head, long long ss, int first, int end, int lane) {
    constexpr int CPR = D * 2 / 16, kRowsAtOnce = 32 / CPR;
    const int r0 = lane / CPR, c = lane % CPR;
#pragma unroll
    for (int i = 0; i < kKeys / kRowsAtOnce; ++i, src += kRowsAtOnce * ss) {
        const int row = r0 + i * kRowsAtOnce;
        const bool there = first + row < end;
        mm::cp_async16(tile + row * (D * 2) + ((c ^ (row & 7)) << 4), there ? src : head, there);
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a float4 of another CTA's shared memory, at the address it has in this one
__device__ __forceinline__ float4 peer_float4(const void* mine, unsigned rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mm::smem_u32(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// Row `row` (of the key head's rows) of the result: n values per lane from column c on
template <typename T, int n>
__device__ __forceinline__ void write_row(const DenseArgs& a, int b, int hk, int row, int c, const float* x, float l, float m, int D, bool first_lane) {
    const int i = row / a.group, h = hk * a.group + row % a.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = static_cast<T*>(const_cast<void*>(a.o.data)) + (long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss + c;
    const long long at = ((long long)b * a.Hq + h) * a.Sq + i;
#pragma unroll
    for (int e = 0; e < n; ++e) {
        const float v = x[e] * inv;
        const T r = DType<T>::from_f32(v);
        dst[e] = r;
        if (a.rest != nullptr) static_cast<T*>(a.rest)[at * D + c + e] = DType<T>::from_f32(v - DType<T>::to_f32(r));
    }
    if (a.lse != nullptr && first_lane) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int D, int MT, bool kCap, bool kBias>
__global__ void __launch_bounds__(kFewWarps<D> * 32, 2) dense_few_kernel(const __grid_constant__ FewParams P) {
    constexpr int kN = kKeys, kTileBytes = kN * D * 2, kRows = 16 * MT, kStages = kFewStages, kStep = few_step(D), kW = kFewWarps<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const ring0 = smem + kRows * D * 2;
    int4* const seen_s = reinterpret_cast<int4*>(ring0 + kW * kStages * 2 * kTileBytes);  // [rows] lo, hi, pos
    const DenseArgs& a = P.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int split = blockIdx.x % P.splits;  // in a cluster: the CTA's rank
    const unsigned others = blockIdx.x / P.splits;
    const int tile = others % P.tiles;
    const int bh = others / P.tiles, b = bh / a.Hk, hk = bh % a.Hk;
    const int row0 = tile * kRows;

    const T* const qb = static_cast<const T*>(a.q.data) + (long long)b * a.q.sb;
    {   // the rows' queries into a swizzled tile, and what they see
        constexpr int CPR = D * 2 / 16;
        const uint32_t q_tile = mm::smem_u32(smem);
        for (int v = tid; v < kRows * CPR; v += kW * 32) {
            const int r = v / CPR, c = v % CPR, rr = row0 + r;
            const bool there = rr < P.rows;
            const int i = there ? rr / a.group : 0, h = hk * a.group + (there ? rr % a.group : 0);
            mm::cp_async16(q_tile + r * (D * 2) + ((c ^ (r & 7)) << 4), qb + (long long)h * a.q.sh + (long long)i * a.q.ss + c * 8, there);
        }
        mm::cp_async_commit();
        if (tid < kRows) {
            Seen s{0, 0, 0};
            if (row0 + tid < P.rows) s = dense_seen(a.mask, b, (row0 + tid) / a.group, a.Sq, a.Sk);
            seen_s[tid] = make_int4(s.lo, s.hi, s.pos, 0);
        }
        __syncthreads();
    }
    // union of the rows' runs, and the run that all rows see (rows that do not exist are masked out, nothing more)
    int u_lo = 0x7fffffff, u_hi = 0, all_lo = 0, all_hi = 0x7fffffff;
    for (int r = lane; r < kRows && row0 + r < P.rows; r += 32) {
        const int4 s = seen_s[r];
        if (s.x < s.y) {
            u_lo = s.x;
            u_hi = s.y;
            all_lo = s.x;
            all_hi = s.y;
        } else {
            all_hi = 0;
        }
    }
    u_lo = __reduce_min_sync(0xffffffffu, u_lo);
    u_hi = __reduce_max_sync(0xffffffffu, u_hi);
    all_lo = __reduce_max_sync(0xffffffffu, all_lo);
    all_hi = __reduce_min_sync(0xffffffffu, all_hi);
    int chunk = P.chunk;
    if (chunk == 0) chunk = u_hi > u_lo ? ((u_hi - u_lo + P.splits - 1) / P.splits + kStep - 1) / kStep * kStep : kStep;
    const long long c_lo = (long long)u_lo + (long long)split * chunk;
    const int first = (int)min(c_lo, (long long)u_hi), end = (int)min(c_lo + chunk, (long long)u_hi);  // keys of this CTA
    const int n_tiles = end > first ? (end - first + kN - 1) / kN : 0;

    const T* const kh = static_cast<const T*>(a.k.data) + (long long)b * a.k.sb + (long long)hk * a.k.sh;
    const T* const vh = static_cast<const T*>(a.v.data) + (long long)b * a.v.sb + (long long)hk * a.v.sh;
    unsigned char* const ring = ring0 + warp * kStages * 2 * kTileBytes;
    // First key of tile t.  With a bias the last keys, which weigh most behind a causal order, come first: the references move less.
    auto key_of = [&](int t) { return first + (kBias ? n_tiles - 1 - t : t) * kN; };
    // this lane's place in the warp's first tile; the tiles of a warp are kStep keys apart and asked for one after another
    constexpr int kCpr = D * 2 / 16, kApart = kBias ? -kStep : kStep;
    const T* k_src = kh + ((long long)key_of(warp) + lane / kCpr) * a.k.ss + lane % kCpr * 8;
    const T* v_src = vh + ((long long)key_of(warp) + lane / kCpr) * a.v.ss + lane % kCpr * 8;
    auto request = [&](int t, int slot) {
        if (t < n_tiles) {
            const uint32_t dst = mm::smem_u32(ring) + slot * 2 * kTileBytes;
            load_keys<T, D>(dst, k_src, kh, a.k.ss, key_of(t), end, lane);
            load_keys<T, D>(dst + kTileBytes, v_src, vh, a.v.ss, key_of(t), end, lane);
            k_src += (long long)kApart * a.k.ss;
            v_src += (long long)kApart * a.v.ss;
        }
        mm::cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) request(warp + i * kW, i);
    mm::cp_async_wait<kStages - 1>();  // the queries
    __syncthreads();

    // the thread's rows: lane / 4 + 8 k of the tiles, k = 0 .. 2 MT - 1
    constexpr int kMine = 2 * MT;
    int4 see[kMine];
    float slope[kMine], m[kMine], l[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
        const int r = (lane >> 2) + 8 * k;
        see[k] = seen_s[r];
        slope[k] = kBias && row0 + r < P.rows ? __ldg(a.slopes + hk * a.group + (row0 + r) % a.group) * kLog2e : 0.f;
        m[k] = -INFINITY;
        l[k] = 0.f;
    }
    float o[MT][D / 8][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    // the queries' fragments: in registers for one tile, read again for every tile of keys for two
    uint32_t qf[MT == 1 ? D / 16 : 1][4];
    auto load_q = [&](int t, int ks, uint32_t (&f)[4]) {
        const int row = 16 * t + (lane & 15), c = 2 * ks + (lane >> 4);
        mm::ldsm_x4(f, mm::smem_u32(smem) + row * (D * 2) + ((c ^ (row & 7)) << 4));
    };
    if (MT == 1) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) load_q(0, ks, qf[MT == 1 ? ks : 0]);
    }

    int slot = 0;
    for (int t = warp; t < n_tiles; t += kW) {
        request(t + (kStages - 1) * kW, slot >= 1 ? slot - 1 : kStages - 1);
        mm::cp_async_wait<kStages - 1>();
        __syncwarp();
        unsigned char* const v_ptr = ring + slot * 2 * kTileBytes + kTileBytes;
        const uint32_t kt = mm::smem_u32(ring) + slot * 2 * kTileBytes, vt = kt + kTileBytes;
        const int key0 = key_of(t);
        const bool mixed = key0 < all_lo || min(key0 + kN, end) > all_hi || key0 + kN > end;

        float s[MT][kN / 8][4];
#pragma unroll
        for (int q = 0; q < MT; ++q)
#pragma unroll
            for (int i = 0; i < kN / 8; ++i) s[q][i][0] = s[q][i][1] = s[q][i][2] = s[q][i][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t af[MT][4];
#pragma unroll
            for (int q = 0; q < MT; ++q) {
                if (MT > 1) load_q(q, ks, af[q]);
            }
#pragma unroll
            for (int np = 0; np < kN / 16; ++np) {
                const int mid = lane >> 3, row = np * 16 + (lane & 7) + (mid >> 1) * 8, c = 2 * ks + (mid & 1);
                uint32_t bf[4];
                mm::ldsm_x4(bf, kt + row * (D * 2) + ((c ^ (row & 7)) << 4));
#pragma unroll
                for (int q = 0; q < MT; ++q) {
                    const uint32_t(&f)[4] = MT == 1 ? qf[MT == 1 ? ks : 0] : af[q];
                    mm::mma16816<T>(s[q][2 * np], f, bf[0], bf[1]);
                    mm::mma16816<T>(s[q][2 * np + 1], f, bf[2], bf[3]);
                }
            }
        }
        float top[kMine];  // of this thread's scores
        bool moved = false;
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int q = k >> 1, e0 = 2 * (k & 1);  // row k's values: s[q][nt][e0], s[q][nt][e0 + 1]
            top[k] = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < kN / 8; ++nt) {
                const int j = key0 + nt * 8 + 2 * (lane & 3);
                float2 x = make_float2(s[q][nt][e0], s[q][nt][e0 + 1]);
                if (kCap) x = capped_any_plus(P.shape, x, make_float2(0.f, 0.f));
                else x = make_float2(x.x * P.shape.mul, x.y * P.shape.mul);
                if (kBias) {
                    x.x = fmaf(-slope[k], fabsf((float)(see[k].z - j)), x.x);
                    x.y = fmaf(-slope[k], fabsf((float)(see[k].z - j - 1)), x.y);
                }
                if (mixed) {
                    const int hi = min(see[k].y, end);
                    if (j < see[k].x || j >= hi) x.x = -INFINITY;
                    if (j + 1 < see[k].x || j + 1 >= hi) x.y = -INFINITY;
                }
                s[q][nt][e0] = x.x;
                s[q][nt][e0 + 1] = x.y;
                top[k] = fmaxf(top[k], fmaxf(x.x, x.y));
            }
            moved |= top[k] > m[k] + 8.f;
        }
        // The rows' references move only when a score is more than 2^8 above one (or the first that is seen): the maximum over the four
        // threads of a row, the sums and the accumulators are only touched then.
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int k = 0; k < kMine; ++k) {
                float n = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
                n = fmaxf(m[k], fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 2)));
                const float alpha = dense_ex2(m[k] - (n == -INFINITY ? 0.f : n));
                m[k] = n;
                l[k] *= alpha;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    o[k >> 1][i][2 * (k & 1)] *= alpha;
                    o[k >> 1][i][2 * (k & 1) + 1] *= alpha;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int q = k >> 1, e0 = 2 * (k & 1);
            const float base = m[k] == -INFINITY ? 0.f : m[k];
#pragma unroll
            for (int nt = 0; nt < kN / 8; ++nt) {
                s[q][nt][e0] = dense_ex2(s[q][nt][e0] - base);
                s[q][nt][e0 + 1] = dense_ex2(s[q][nt][e0 + 1] - base);
                l[k] += s[q][nt][e0] + s[q][nt][e0 + 1];  // this thread's keys; added up over the four threads of a row at the end
            }
        }
        if (mixed && tile_nonfinite<T, kTileBytes / 16>(reinterpret_cast<const uint4*>(v_ptr), lane)) {
#pragma unroll 1
            for (int r = 0; r < kN; ++r) {
                const int j = key0 + r;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const T* p = reinterpret_cast<const T*>(v_ptr + r * (D * 2) + ((i ^ (r & 7)) << 4)) + 2 * (lane & 3);
                    const float x0 = DType<T>::to_f32(p[0]), x1 = DType<T>::to_f32(p[1]);
#pragma unroll
                    for (int k = 0; k < kMine; ++k) {
                        const bool sees = j >= see[k].x && j < min(see[k].y, end);
                        if (sees && !isfinite(x0)) o[k >> 1][i][2 * (k & 1)] += x0;
                        if (sees && !isfinite(x1)) o[k >> 1][i][2 * (k & 1) + 1] += x1;
                    }
                }
            }
            __syncwarp();
            for (int v = lane; v < kTileBytes / 4; v += 32) {
                uint32_t* p = reinterpret_cast<uint32_t*>(v_ptr) + v;
                *p = zero_nonfinite<T>(*p);
            }
            __syncwarp();
        }
#pragma unroll
        for (int kk = 0; kk < kN / 16; ++kk) {
            uint32_t pa[MT][4];
#pragma unroll
            for (int q = 0; q < MT; ++q) {
                pa[q][0] = mm::pack2(T(), s[q][2 * kk][0], s[q][2 * kk][1]);
                pa[q][1] = mm::pack2(T(), s[q][2 * kk][2], s[q][2 * kk][3]);
                pa[q][2] = mm::pack2(T(), s[q][2 * kk + 1][0], s[q][2 * kk + 1][1]);
                pa[q][3] = mm::pack2(T(), s[q][2 * kk + 1][2], s[q][2 * kk + 1][3]);
            }
#pragma unroll
            for (int dp = 0; dp < D / 16; ++dp) {
                const int mid = lane >> 3, row = kk * 16 + (lane & 7) + (mid & 1) * 8, c = 2 * dp + (mid >> 1);
                uint32_t bf[4];
                mm::ldsm_x4_t(bf, vt + row * (D * 2) + ((c ^ (row & 7)) << 4));
#pragma unroll
                for (int q = 0; q < MT; ++q) {
                    mm::mma16816<T>(o[q][2 * dp], pa[q], bf[0], bf[1]);
                    mm::mma16816<T>(o[q][2 * dp + 1], pa[q], bf[2], bf[3]);
                }
            }
        }
        __syncwarp();  // all lanes are through with the slot that the next round's request overwrites
        if (++slot == kStages) slot = 0;
    }
    mm::cp_async_wait<0>();
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
    }

    // ---- join of the warps: their accumulators in the ring, [warp][rows][D + 4] fp32, and (m, l) behind them
    __syncthreads();
    constexpr int kPitch = D + 4;
    float* const acc_s = reinterpret_cast<float*>(ring0);
    float2* const ml_s = reinterpret_cast<float2*>(ring0 + kW * kRows * kPitch * 4);
    static_assert(kW * kRows * kPitch * 4 + kW * kRows * 8 <= kW * kStages * 2 * kTileBytes, "the join fits the ring");
    {
        float* const mine = acc_s + warp * kRows * kPitch;
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int r = (lane >> 2) + 8 * k;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(mine + r * kPitch + i * 8 + 2 * (lane & 3)) = make_float2(o[k >> 1][i][2 * (k & 1)], o[k >> 1][i][2 * (k & 1) + 1]);
            if ((lane & 3) == 0) ml_s[warp * kRows + r] = make_float2(m[k], l[k]);
        }
    }
    __syncthreads();
    constexpr int kPer = D / 32;  // values of a lane, a warp takes rows warp, warp + kW, ...
    const bool cluster = P.chunk == 0 && P.splits > 1;
    for (int r = warp; r < kRows && row0 + r < P.rows; r += kW) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kW; ++w) top = fmaxf(top, ml_s[w * kRows + r].x);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, x[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            const float2 ml = ml_s[w * kRows + r];
            const float f = dense_ex2(ml.x - base);
            sum += ml.y * f;
            const float* src = acc_s + (w * kRows + r) * kPitch + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] += src[e] * f;
        }
        if (cluster) {  // the CTA's result of the row takes the place of the first warp's
            float* dst = acc_s + r * kPitch + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) dst[e] = x[e];
            __syncwarp();
            if (lane == 0) *reinterpret_cast<float2*>(acc_s + r * kPitch + D) = make_float2(top, sum);
        } else if (P.part_o != nullptr) {
            const long long gr = (long long)bh * P.rows + row0 + r;
            float* dst = P.part_o + (gr * P.splits + split) * D + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) dst[e] = x[e];
            if (lane == 0) P.part_ml[gr * P.splits + split] = make_float2(top, sum);
        } else {
            write_row<T, kPer>(a, b, hk, row0 + r, lane * kPer, x, sum, top, D, lane == 0);
        }
    }
    if (!cluster) return;
    // ---- join of the cluster: CTA c takes rows c, c + splits, ..., D / 4 lanes a row
    cluster_sync();
    constexpr int kLanes = D / 4, kAtOnce = kW * 32 / kLanes;
    const int c4 = tid % kLanes;
    for (int r = split + P.splits * (tid / kLanes); r < kRows && row0 + r < P.rows; r += P.splits * kAtOnce) {
        float top = -INFINITY;
        for (int c = 0; c < P.splits; ++c) top = fmaxf(top, peer_float4(acc_s + r * kPitch + D, c).x);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = 0; c < P.splits; ++c) {
            const float4 ml = peer_float4(acc_s + r * kPitch + D, c), v = peer_float4(acc_s + r * kPitch + 4 * c4, c);
            const float f = dense_ex2(ml.x - base);
            sum += ml.y * f;
            x[0] += v.x * f;
            x[1] += v.y * f;
            x[2] += v.z * f;
            x[3] += v.w * f;
        }
        write_row<T, 4>(a, b, hk, row0 + r, 4 * c4, x, sum, top, D, c4 == 0);
    }
    cluster_sync();  // nobody leaves while another CTA reads its shared memory
}

// One warp per row: the chunks' partial results, relative to the row's maximum, in ascending order.
template <typename T, int D>
__global__ void __launch_bounds__(128) dense_combine_kernel(const __grid_constant__ FewParams P) {
    constexpr int kPer = D / 32;
    const DenseArgs& a = P.a;
    const int lane = threadIdx.x & 31;
    const long long gr = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (gr >= (long long)a.B * a.Hk * P.rows) return;
    const float2* ml = P.part_ml + gr * P.splits;
    float m = -INFINITY;
    for (int s = lane; s < P.splits; s += 32) m = fmaxf(m, ml[s].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, acc[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
    const float* src = P.part_o + gr * P.splits * D + lane * kPer;
    for (int s = 0; s < P.splits; ++s, src += D) {
        const float2 v = ml[s];
        if (v.x == -INFINITY && v.y == 0.f) continue;  // a chunk in which the row sees nothing
        const float f = dense_ex2(v.x - base);
        l += v.y * f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] += src[e] * f;
    }
    const int bh = (int)(gr / P.rows);
    write_row<T, kPer>(a, bh / a.Hk, bh % a.Hk, (int)(gr % P.rows), lane * kPer, acc, l, m, D, lane == 0);
}

// How the keys are shared out.  A cluster of CTAs for each 16 or 32 rows, as large as it takes for one CTA an SM, if there are keys for all of them; and
// larger where a CTA still has 64 rounds or more (GPU alone, without / with that second step: 32 caches of 32768 keys, 8 heads of 128, 652 / 614
// us, their lengths between a quarter and the whole 473 / 383; 24 ragged ones 404 / 305; 40 ragged ones of 20000 keys, 4 heads, 225 / 170; 16 heads of 64, 32 of
// 16384 keys, 322 / 326, ragged 227 / 211; 100 of 8192 keys, 8 heads, 481 / 487, ragged 338 / 326).
void few_plan(const DenseArgs& a, FewParams& P) {
    const int kStep = few_step(a.D);
    P.rows = a.group * a.Sq;
    P.mt = P.rows <= 16 ? 1 : 2;
    P.tiles = (P.rows + 16 * P.mt - 1) / (16 * P.mt);
    const long long units = (long long)a.B * a.Hk * P.tiles;
    P.chunk = 0;
    P.splits = 1;
    while (P.splits < kMaxCluster && units * P.splits < 148 && P.splits * kStep < a.Sk) P.splits *= 2;
    while (P.splits < kMaxCluster && units * P.splits < 148 * 8 && P.splits * kStep * 64 <= a.Sk) P.splits *= 2;
    if (units * P.splits >= 148 || a.Sk <= kMaxCluster * 16 * kStep) return;
    // clusters leave SMs idle, with more than 16 rounds to a CTA: chunks, some four for every SM
    long long splits = (148 * 4 + units - 1) / (units > 0 ? units : 1);
    const long long most = (a.Sk + 2 * kStep - 1) / (2 * kStep);
    splits = splits < most ? splits : most;
    splits = splits < kMaxSplits ? splits : kMaxSplits;
    P.chunk = (int)(((a.Sk + splits - 1) / splits + kStep - 1) / kStep * kStep);
    P.splits = (int)((a.Sk + P.chunk - 1) / P.chunk);
}

template <typename T, int D, int MT, bool kCap, bool kBias>
cudaError_t few_launch(const FewParams& P, cudaStream_t st) {
    const DenseArgs& a = P.a;
    auto kern = dense_few_kernel<T, D, MT, kCap, kBias>;
    static thread_local unsigned long long raised = 0;  // devices (below 64) whose shared-memory limit this thread has raised for this kernel
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !((raised >> dev) & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem<D, MT>());
        if (e != cudaSuccess) return e;
        if (dev <= 63) raised |= 1ull << dev;
    }
    const long long ctas = (long long)a.B * a.Hk * P.tiles * P.splits;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kFewWarps<D> * 32);
    cfg.dynamicSmemBytes = few_smem<D, MT>();
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = P.chunk == 0 ? P.splits : 1;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = P.chunk == 0 && P.splits > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, P);
    if (e != cudaSuccess || P.part_o == nullptr) return e;
    const long long rows = (long long)a.B * a.Hk * P.rows;
    dense_combine_kernel<T, D><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(P);
    return cudaGetLastError();
}

template <typename T, int D, int MT>
cudaError_t few_shape(const FewParams& P, cudaStream_t st) {
    const bool cap = P.a.cap > 0.f, bias = P.a.slopes != nullptr;
    if (cap) return bias ? few_launch<T, D, MT, true, true>(P, st) : few_launch<T, D, MT, true, false>(P, st);
    return bias ? few_launch<T, D, MT, false, true>(P, st) : few_launch<T, D, MT, false, false>(P, st);
}
template <typename T, int D>
cudaError_t few_rows(const FewParams& P, cudaStream_t st) { return P.mt == 1 ? few_shape<T, D, 1>(P, st) : few_shape<T, D, 2>(P, st); }

}  // namespace

bool dense_supported(const DenseArgs& a, const char** why) {
    if (a.dtype != LCBSA_BF16 && a.dtype != LCBSA_FP16) { *why = "takes bf16 or fp16"; return false; }
    if (a.D != 64 && a.D != 128) { *why = "takes head_dim 64 or 128"; return false; }
    if ((long long)a.group * a.Sq > 0x7ffffff0ll || a.Sk > 0x7fffff00) { *why = "more than 2^31 rows of a key head"; return false; }
    return true;
}

// Which kernel, from what the two cost in us: this one 5, for every key of a tile of 16 (32) rows 0.0100 (0.0145) over the
// SMs at head_dim 128 and half of it at 64, and 4 for every further wave of CTAs; the tcgen05 kernel 8 (a plan before it, tensor maps) and 0.55 for every
// unit of 64 keys of 128 rows of ONE head.  Measured (few / tcgen05, us): 8 sequences x 16 heads, head_dim 128: 4 x 512 10.1 / 13.9, 16 x 4096
// 50.2 / 51.0, 32 x 4096 53.4 / 50.5, 64 x 512 19.7 / 14.2; 2 x 16 heads sharing 4: 64 x 4096 31.7 / 39.6, 200 x 1000 29.0 / 17.8;
// head_dim 64, 8 heads: 200 x 200 8.4 / 11.0, 64 x 4096 13.6 / 37.9; 8 x 16: 128 x 128 15.1 / 10.9.
static bool few_queries(const DenseArgs& a) {
    if (a.impl != LCBSA_ATTN_AUTO) return a.impl == LCBSA_ATTN_MMA;
    FewParams P;
    few_plan(a, P);
    const double units = (double)a.B * a.Hk * P.tiles, items = (double)a.B * a.Hq * ((a.Sq + 127) / 128);
    const double few = 5 + units * a.Sk * (a.D / 128.0) * (P.mt == 1 ? 0.0100 : 0.0145) / 148 + 4 * (units > 296 ? units / 296 - 1 : 0);
    const double tc = 8 + 0.55 * (items <= 148 ? 1 : items / 148) * a.Sk / 64;
    return few <= tc;
}

size_t dense_fwd_workspace_bytes(const DenseArgs& a) {
    FewParams P;
    few_plan(a, P);
    const size_t plan = few_queries(a) ? 0 : dense_plan_bytes(a, false);
    if (P.chunk == 0) return plan;
    const size_t few = (size_t)a.B * a.Hk * P.rows * P.splits * (a.D + 2) * 4;
    return few > plan ? few : plan;
}

cudaError_t launch_dense_fwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why) {
    if (a.B == 0 || a.Hq == 0 || a.Sq == 0) return cudaSuccess;
    if (!few_queries(a) && a.impl == LCBSA_ATTN_TC && !dense_tc_supported(a)) {
        *why = "the tcgen05 kernel takes at least one query and one key, and tokens a stride apart";
        return cudaErrorInvalidValue;
    }
    if (!few_queries(a) && dense_tc_supported(a)) {
        dense_plan_carve(a, workspace, false);
        const cudaError_t e = launch_dense_plan(a, st);
        return e == cudaSuccess ? launch_dense_tc(a, st, why) : e;
    }
    FewParams P;
    P.a = a;
    P.shape = score_shape(a.scale, a.cap);
    few_plan(a, P);
    P.part_o = nullptr;
    P.part_ml = nullptr;
    if (P.chunk > 0) {
        P.part_o = static_cast<float*>(workspace);
        P.part_ml = reinterpret_cast<float2*>(P.part_o + (long long)a.B * a.Hk * P.rows * P.splits * a.D);
    }
    const cudaError_t e = a.dtype == LCBSA_BF16
                              ? (a.D == 128 ? few_rows<__nv_bfloat16, 128>(P, st) : few_rows<__nv_bfloat16, 64>(P, st))
                              : (a.D == 128 ? few_rows<__half, 128>(P, st) : few_rows<__half, 64>(P, st));
    if (e == cudaErrorInvalidConfiguration) *why = "more CTAs than a launch takes";
    return e;
}

}  // namespace lcbsa
