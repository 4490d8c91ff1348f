// Dense attention forward for few queries (see dense_common.cuh for the formulas): a token, or a few drafted ones, of every sequence
// behind a long cache.  Bound by HBM: each key and value is read once for all queries and all heads that share it.
//
// The rows of one 16-row MMA tile are (query, head of the group) pairs, so a group of four heads and one query fill four of
// them and the cache is still read once.  The keys are split over CTAs in chunks of a fixed number (an even load whatever the
// lengths; a chunk behind the last key that any row sees ends at once), and inside a CTA over four warps that take every fourth
// tile of 32 keys: a warp has a ring of its own in shared memory and nothing in the loop waits for another warp.  S, P and O
// stay in registers (mma.sync m16n8k16, fp32 accumulators; P is rounded to the input type for the product with V, as in the
// other attention kernels, the row sum is taken before the rounding); running maximum and sum per row in fp32, merged over the
// warps through shared memory and over the chunks by a second kernel from fp32 partial results.
//
// Masked places hold anything: keys outside the union of the rows' runs are not loaded, a masked score is replaced (not
// multiplied), and in a tile that only some rows see the values that are not finite are added by hand to the rows that see
// them and are zero for the product, so that 0 * inf reaches no row that does not.
#include "dense_common.cuh"
#include "mma_common.cuh"

namespace lcbsa {

namespace {

constexpr int kRows = 16;       // (query, head) rows of a CTA
constexpr int kFewWarps = 4;
constexpr int kKeys = 32;       // keys of a warp's tile
constexpr int kFewStages = 2;
constexpr int kMaxSplits = 256;

struct FewParams {
    DenseArgs a;
    ScoreShape shape;
    int rows;               // group * Sq rows of one key head
    int tiles;              // 16-row tiles of them
    int splits, chunk;      // chunks of the keys, keys of a chunk
    float* part_o;          // [B*Hk*rows][splits][D], not yet divided by the row sum; null: one chunk, straight to the output
    float2* part_ml;        // [B*Hk*rows][splits]: maximum (log2), row sum
};

template <int D>
constexpr int few_smem() {
    return kRows * D * 2 + kFewWarps * kFewStages * 2 * kKeys * D * 2 + kRows * 16;
}

// `n` rows of D values from row `first` on into a swizzled tile; rows at `end` or behind are zero
template <typename T, int D>
__device__ __forceinline__ void load_keys(uint32_t tile, const T* head, long long ss, int first, int end, int lane) {
    constexpr int CPR = D * 2 / 16;
#pragma unroll
    for (int v = lane; v < kKeys * CPR; v += 32) {
        const int row = v / CPR, c = v % CPR;
        const bool there = first + row < end;
        mm::cp_async16(tile + row * (D * 2) + ((c ^ (row & 7)) << 4), head + (there ? (long long)(first + row) * ss : 0) + c * 8, there);
    }
}

template <typename T, int D, bool kCap, bool kBias>
__global__ void __launch_bounds__(kFewWarps * 32) dense_few_kernel(const __grid_constant__ FewParams P) {
    constexpr int kTileBytes = kKeys * D * 2;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const ring0 = smem + kRows * D * 2;
    int4* const seen_s = reinterpret_cast<int4*>(ring0 + kFewWarps * kFewStages * 2 * kTileBytes);  // [16] lo, hi, pos
    const DenseArgs& a = P.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int split = blockIdx.x % P.splits;
    const unsigned rest = blockIdx.x / P.splits;
    const int tile = rest % P.tiles;
    const int bh = rest / P.tiles, b = bh / a.Hk, hk = bh % a.Hk;
    const int row0 = tile * kRows;

    const T* const qb = static_cast<const T*>(a.q.data) + (long long)b * a.q.sb;
    {   // the rows' queries into a swizzled tile, and what they see
        constexpr int CPR = D * 2 / 16;
        const uint32_t q_tile = mm::smem_u32(smem);
        for (int v = tid; v < kRows * CPR; v += kFewWarps * 32) {
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
        mm::cp_async_wait<0>();
        __syncthreads();
    }
    // union of the rows' runs, and the run that all rows see
    int u_lo = 0x7fffffff, u_hi = 0, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int4 s = seen_s[r];
        if (row0 + r >= P.rows) continue;
        if (s.x < s.y) {
            u_lo = min(u_lo, s.x);
            u_hi = max(u_hi, s.y);
            all_lo = max(all_lo, s.x);
            all_hi = min(all_hi, s.y);
        } else {
            all_hi = 0;
        }
    }
    const long long c_lo = (long long)u_lo + (long long)split * P.chunk;
    const int first = (int)min(c_lo, (long long)u_hi), end = (int)min(c_lo + P.chunk, (long long)u_hi);  // keys of this chunk
    const int n_tiles = end > first ? (end - first + kKeys - 1) / kKeys : 0;

    const int ra = lane >> 2, rb = ra + 8;  // the thread's two rows
    const int4 sa = seen_s[ra], sb = seen_s[rb];
    float slope_a = 0.f, slope_b = 0.f;
    if (kBias) {
        if (row0 + ra < P.rows) slope_a = __ldg(a.slopes + hk * a.group + (row0 + ra) % a.group) * kLog2e;
        if (row0 + rb < P.rows) slope_b = __ldg(a.slopes + hk * a.group + (row0 + rb) % a.group) * kLog2e;
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;

    const T* const kh = static_cast<const T*>(a.k.data) + (long long)b * a.k.sb + (long long)hk * a.k.sh;
    const T* const vh = static_cast<const T*>(a.v.data) + (long long)b * a.v.sb + (long long)hk * a.v.sh;
    unsigned char* const ring = ring0 + warp * kFewStages * 2 * kTileBytes;
    auto request = [&](int t, int slot) {
        const uint32_t dst = mm::smem_u32(ring) + slot * 2 * kTileBytes;
        load_keys<T, D>(dst, kh, a.k.ss, first + t * kKeys, end, lane);
        load_keys<T, D>(dst + kTileBytes, vh, a.v.ss, first + t * kKeys, end, lane);
    };
    if (warp < n_tiles) request(warp, 0);
    mm::cp_async_commit();

    uint32_t qf[D / 16][4];
    {
        const int row = lane & 15;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int c = 2 * ks + (lane >> 4);
            mm::ldsm_x4(qf[ks], mm::smem_u32(smem) + row * (D * 2) + ((c ^ (row & 7)) << 4));
        }
    }

    int slot = 0;
    for (int t = warp; t < n_tiles; t += kFewWarps, slot ^= 1) {
        if (t + kFewWarps < n_tiles) request(t + kFewWarps, slot ^ 1);
        mm::cp_async_commit();
        mm::cp_async_wait<1>();
        __syncwarp();
        unsigned char* const v_ptr = ring + slot * 2 * kTileBytes + kTileBytes;
        const uint32_t kt = mm::smem_u32(ring) + slot * 2 * kTileBytes, vt = kt + kTileBytes;
        const int key0 = first + t * kKeys;
        const bool mixed = key0 < all_lo || min(key0 + kKeys, end) > all_hi || key0 + kKeys > end;

        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
            for (int np = 0; np < 2; ++np) {
                const int mid = lane >> 3;
                const int row = np * 16 + (lane & 7) + (mid >> 1) * 8;
                const int c = 2 * ks + (mid & 1);
                uint32_t bf[4];
                mm::ldsm_x4(bf, kt + row * (D * 2) + ((c ^ (row & 7)) << 4));
                mm::mma16816<T>(s[2 * np], qf[ks], bf[0], bf[1]);
                mm::mma16816<T>(s[2 * np + 1], qf[ks], bf[2], bf[3]);
            }
        }
        float top_a = -INFINITY, top_b = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = key0 + nt * 8 + 2 * (lane & 3) + e;
                float2 x = make_float2(s[nt][e], s[nt][2 + e]), slack;
                if (kCap) x = capped_any(P.shape, x, slack);
                else x = make_float2(x.x * P.shape.mul, x.y * P.shape.mul);
                float xa = x.x, xb = x.y;
                if (kBias) {
                    xa = fmaf(-slope_a, fabsf((float)(sa.z - j)), xa);
                    xb = fmaf(-slope_b, fabsf((float)(sb.z - j)), xb);
                }
                if (mixed) {
                    if (j < sa.x || j >= min(sa.y, end)) xa = -INFINITY;
                    if (j < sb.x || j >= min(sb.y, end)) xb = -INFINITY;
                }
                s[nt][e] = xa;
                s[nt][2 + e] = xb;
                top_a = fmaxf(top_a, xa);
                top_b = fmaxf(top_b, xb);
            }
        }
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            top_a = fmaxf(top_a, __shfl_xor_sync(0xffffffffu, top_a, x));
            top_b = fmaxf(top_b, __shfl_xor_sync(0xffffffffu, top_b, x));
        }
        const float n_a = fmaxf(m_a, top_a), n_b = fmaxf(m_b, top_b);
        const float base_a = n_a == -INFINITY ? 0.f : n_a, base_b = n_b == -INFINITY ? 0.f : n_b;
        const float al_a = dense_ex2(m_a - base_a), al_b = dense_ex2(m_b - base_b);
        m_a = n_a;
        m_b = n_b;
        float sum_a = 0.f, sum_b = 0.f;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[nt][e] = dense_ex2(s[nt][e] - base_a);
                s[nt][2 + e] = dense_ex2(s[nt][2 + e] - base_b);
                sum_a += s[nt][e];
                sum_b += s[nt][2 + e];
            }
        }
        l_a = l_a * al_a + sum_a;  // this thread's keys; added up over the four threads of a row at the end
        l_b = l_b * al_b + sum_b;
        if (__any_sync(0xffffffffu, al_a != 1.f || al_b != 1.f)) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] *= al_a;
                o[i][1] *= al_a;
                o[i][2] *= al_b;
                o[i][3] *= al_b;
            }
        }
        if (mixed) {
            bool bad = false;
#pragma unroll 4
            for (int v = lane; v < kTileBytes / 16; v += 32) bad |= chunk_nonfinite<T>(*reinterpret_cast<const uint4*>(v_ptr + 16 * v));
            if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
                for (int r = 0; r < kKeys; ++r) {
                    const int j = key0 + r;
                    const bool ga = j >= sa.x && j < min(sa.y, end), gb = j >= sb.x && j < min(sb.y, end);
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const T* p = reinterpret_cast<const T*>(v_ptr + r * (D * 2) + ((i ^ (r & 7)) << 4)) + 2 * (lane & 3);
                        const float x0 = DType<T>::to_f32(p[0]), x1 = DType<T>::to_f32(p[1]);
                        if (!isfinite(x0)) {
                            if (ga) o[i][0] += x0;
                            if (gb) o[i][2] += x0;
                        }
                        if (!isfinite(x1)) {
                            if (ga) o[i][1] += x1;
                            if (gb) o[i][3] += x1;
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
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint32_t pa[4];
            pa[0] = mm::pack2(T(), s[2 * kk][0], s[2 * kk][1]);
            pa[1] = mm::pack2(T(), s[2 * kk][2], s[2 * kk][3]);
            pa[2] = mm::pack2(T(), s[2 * kk + 1][0], s[2 * kk + 1][1]);
            pa[3] = mm::pack2(T(), s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
            for (int dp = 0; dp < D / 16; ++dp) {
                const int mid = lane >> 3;
                const int row = kk * 16 + (lane & 7) + (mid & 1) * 8;
                const int c = 2 * dp + (mid >> 1);
                uint32_t bf[4];
                mm::ldsm_x4_t(bf, vt + row * (D * 2) + ((c ^ (row & 7)) << 4));
                mm::mma16816<T>(o[2 * dp], pa, bf[0], bf[1]);
                mm::mma16816<T>(o[2 * dp + 1], pa, bf[2], bf[3]);
            }
        }
        __syncwarp();  // all lanes are through with the slot that the next round's request overwrites
    }
    mm::cp_async_wait<0>();
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        l_a += __shfl_xor_sync(0xffffffffu, l_a, x);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, x);
    }

    // ---- merge of the four warps: their accumulators in the ring, [warp][16][D + 4] fp32, and (m, l) behind them
    __syncthreads();
    constexpr int kPitch = D + 4;
    float* const acc_s = reinterpret_cast<float*>(ring0);
    float2* const ml_s = reinterpret_cast<float2*>(ring0 + kFewWarps * kRows * kPitch * 4);
    static_assert(kFewWarps * kRows * kPitch * 4 + kFewWarps * kRows * 8 <= kFewWarps * kFewStages * 2 * kTileBytes, "the merge fits the ring");
    {
        float* const mine = acc_s + warp * kRows * kPitch;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const int col = i * 8 + 2 * (lane & 3);
            *reinterpret_cast<float2*>(mine + ra * kPitch + col) = make_float2(o[i][0], o[i][1]);
            *reinterpret_cast<float2*>(mine + rb * kPitch + col) = make_float2(o[i][2], o[i][3]);
        }
        if ((lane & 3) == 0) {
            ml_s[warp * kRows + ra] = make_float2(m_a, l_a);
            ml_s[warp * kRows + rb] = make_float2(m_b, l_b);
        }
    }
    __syncthreads();
    constexpr int kPer = D / 32;  // values of a lane, a warp takes rows warp, warp + 4, ...
    for (int r = warp; r < kRows && row0 + r < P.rows; r += kFewWarps) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, ml_s[w * kRows + r].x);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f, x[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float2 ml = ml_s[w * kRows + r];
            const float f = dense_ex2(ml.x - base);
            l += ml.y * f;
            const float* src = acc_s + (w * kRows + r) * kPitch + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] += src[e] * f;
        }
        const long long gr = (long long)bh * P.rows + row0 + r;
        if (P.part_o != nullptr) {
            float* dst = P.part_o + (gr * P.splits + split) * D + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) dst[e] = x[e];
            if (lane == 0) P.part_ml[gr * P.splits + split] = make_float2(m, l);
        } else {
            const int i = (row0 + r) / a.group, h = hk * a.group + (row0 + r) % a.group;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            T* dst = static_cast<T*>(const_cast<void*>(a.o.data)) + (long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const float v = x[e] * inv;
                dst[e] = DType<T>::from_f32(v);
                if (a.rest != nullptr)
                    static_cast<T*>(a.rest)[(((long long)b * a.Hq + h) * a.Sq + i) * D + lane * kPer + e] = DType<T>::from_f32(v - DType<T>::to_f32(dst[e]));
            }
            if (a.lse != nullptr && lane == 0) a.lse[((long long)b * a.Hq + h) * a.Sq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
    }
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
    const int bh = (int)(gr / P.rows), row = (int)(gr % P.rows);
    const int b = bh / a.Hk, h = bh % a.Hk * a.group + row % a.group, i = row / a.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = static_cast<T*>(const_cast<void*>(a.o.data)) + (long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const float v = acc[e] * inv;
        dst[e] = DType<T>::from_f32(v);
        if (a.rest != nullptr)
            static_cast<T*>(a.rest)[(((long long)b * a.Hq + h) * a.Sq + i) * D + lane * kPer + e] = DType<T>::from_f32(v - DType<T>::to_f32(dst[e]));
    }
    if (a.lse != nullptr && lane == 0) a.lse[((long long)b * a.Hq + h) * a.Sq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Chunks: about eight CTAs for every SM, none below 128 keys (a tile for each of the four warps).
void few_plan(const DenseArgs& a, FewParams& P) {
    P.rows = a.group * a.Sq;
    P.tiles = (P.rows + kRows - 1) / kRows;
    const long long units = (long long)a.B * a.Hk * P.tiles;
    long long splits = (148 * 8 + units - 1) / (units > 0 ? units : 1);
    const long long most = (a.Sk + 127) / 128;
    splits = splits < most ? splits : most;
    splits = splits < kMaxSplits ? splits : kMaxSplits;
    if (splits < 1) splits = 1;
    P.chunk = (int)(((a.Sk + splits - 1) / splits + 127) / 128 * 128);
    if (P.chunk < 128) P.chunk = 128;
    P.splits = a.Sk > 0 ? (int)((a.Sk + P.chunk - 1) / P.chunk) : 1;
}

template <typename T, int D, bool kCap, bool kBias>
cudaError_t few_launch(const FewParams& P, cudaStream_t st) {
    const DenseArgs& a = P.a;
    static thread_local unsigned long long raised = 0;  // devices (below 64) whose shared-memory limit this thread has raised for this kernel
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !((raised >> dev) & 1)) {
        e = cudaFuncSetAttribute(dense_few_kernel<T, D, kCap, kBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem<D>());
        if (e != cudaSuccess) return e;
        if (dev <= 63) raised |= 1ull << dev;
    }
    const long long ctas = (long long)a.B * a.Hk * P.tiles * P.splits;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    dense_few_kernel<T, D, kCap, kBias><<<(unsigned)ctas, kFewWarps * 32, few_smem<D>(), st>>>(P);
    e = cudaGetLastError();
    if (e != cudaSuccess || P.part_o == nullptr) return e;
    const long long rows = (long long)a.B * a.Hk * P.rows;
    dense_combine_kernel<T, D><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(P);
    return cudaGetLastError();
}

template <typename T, int D>
cudaError_t few_shape(const FewParams& P, cudaStream_t st) {
    const bool cap = P.a.cap > 0.f, bias = P.a.slopes != nullptr;
    if (cap) return bias ? few_launch<T, D, true, true>(P, st) : few_launch<T, D, true, false>(P, st);
    return bias ? few_launch<T, D, false, true>(P, st) : few_launch<T, D, false, false>(P, st);
}

}  // namespace

bool dense_supported(const DenseArgs& a, const char** why) {
    if (a.dtype != LCBSA_BF16 && a.dtype != LCBSA_FP16) { *why = "takes bf16 or fp16"; return false; }
    if (a.D != 64 && a.D != 128) { *why = "takes head_dim 64 or 128"; return false; }
    if ((long long)a.group * a.Sq > 0x7ffffff0ll || a.Sk > 0x7fffff00) { *why = "more than 2^31 rows of a key head"; return false; }
    return true;
}

// Which kernel: the tcgen05 kernel computes 128 rows of one head at a time, this one 16 rows of a group of heads.  (To be measured.)
static bool few_queries(const DenseArgs& a) { return (long long)a.group * a.Sq <= 64; }

size_t dense_fwd_workspace_bytes(const DenseArgs& a) {
    FewParams P;
    few_plan(a, P);
    const size_t plan = few_queries(a) ? 0 : dense_plan_bytes(a, false);
    if (P.splits == 1) return plan;
    const size_t few = (size_t)a.B * a.Hk * P.rows * P.splits * (a.D + 2) * 4;
    return few > plan ? few : plan;
}

cudaError_t launch_dense_fwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why) {
    if (a.B * a.Hq == 0 || a.Sq == 0) return cudaSuccess;
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
    if (P.splits > 1) {
        P.part_o = static_cast<float*>(workspace);
        P.part_ml = reinterpret_cast<float2*>(P.part_o + (long long)a.B * a.Hk * P.rows * P.splits * a.D);
    }
    const cudaError_t e = a.dtype == LCBSA_BF16
                              ? (a.D == 128 ? few_shape<__nv_bfloat16, 128>(P, st) : few_shape<__nv_bfloat16, 64>(P, st))
                              : (a.D == 128 ? few_shape<__half, 128>(P, st) : few_shape<__half, 64>(P, st));
    if (e == cudaErrorInvalidConfiguration) *why = "more CTAs than a launch takes";
    return e;
}

}  // namespace lcbsa
