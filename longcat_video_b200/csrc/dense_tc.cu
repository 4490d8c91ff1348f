// Dense attention forward for sm_100a (see dense_common.cuh for the formulas and the masks): TMA + tcgen05 + TMEM.
//
// One persistent CTA per SM; a work item is one tile of 128 queries of one head, and its keys are the union of the runs that its rows
// see, in units of 64 from the first such key on.  The items are taken off a counter (their lengths are known on the GPU
// alone), wave by wave of heads and in each the last queries first, since with a causal order they have most keys; one warp announces
// them in a ring.
//
//   warps 0-3, 4-7 : softmax warpgroups 0 and 1 (units of even / odd number; thread = one query row)
//   warp 8 : items, TMA producer of Q and K   warp 9 : S = Q K^T issuer   warp 10 : O += P V issuer   warp 11: TMA producer of V
//   warps 12-15 : Q to TMEM, merge and store of O (epilogue warps)
//
// The roles, the rings and the TMEM columns are those of the block-sparse kernel for 128-token blocks (attn_tc128.cu), where they
// are explained: per unit S = Q K^T (A = Q from TMEM) -> scores shaped, masked and exponentiated in registers (online softmax with a
// lazily moved reference) -> P in the input type into TMEM -> O += P V.  What differs: a unit is whole (every row sees all of its keys) or
// mixed, and only mixed units are masked element by element; heads share keys; scores are capped and biased on the arithmetic pipes
// (five operations per pair of scores for a cap, one for a bias: see ScoreShape and BiasLine).
//
// Bound by the latency of a unit's chain S -> registers -> exponentials -> P -> PV with two softmax warps on a scheduler, not by a pipe: the two
// products of a unit take 512 cycles of the tensor pipe and its 8192 exponentials 512 of the special functions', and a unit takes 1120 (37 heads of
// 2048 tokens, 128 units an SM: 144 000 cycles).  37 heads of 4096 tokens, head_dim 128: 540 ns a unit (1.1 PFLOP/s), 690 with a cap, 630
// with a bias, 760 with both; at 37 x 2048 under the profiler the tensor pipe is 46 % busy, 35 % with a cap, issue slots 43 and 45 %.  Every eighth
// pair of exponentials on the arithmetic pipes instead (a polynomial of degree 4): 455 us in the place of 447 at head_dim 128, 412 of 434 at 64;
// every fourth 471 and 413: not worth a second kind.
//
// Hidden values may be anything.  A score that is not finite stays in its column and is replaced there.  V enters the product of every row
// of the tile, so in mixed units its producer looks through the tile first: values that are not finite are set to zero, and the epilogue adds
// them by hand to the rows that see them.
//
// Every wait on an mbarrier is bounded, as in attn_tc.cu.
#include <type_traits>

#include "dense_common.cuh"
#include "tc_common.cuh"

namespace lcbsa {

namespace {

using namespace tc;

constexpr int kQRows = 128;     // queries of a work item: one M=128 tile
constexpr int kBlk = kDenseUnit;  // keys per unit
constexpr int kKSlots = 6, kVSlots = 6;
constexpr int kThreads = 512;
// setmaxnreg per warpgroup: (176 + 176 + 48 + 112) * 128 threads = the 64 K registers of the SM, 128 per thread at launch
constexpr int kRegsSoftmax = 176, kRegsOther = 48, kRegsEpilogue = 112;
constexpr int kItemRing = 4;    // items announced ahead
constexpr int kItemReaders = 15;  // warps that read an announced item: all but the one that writes it

// TMEM columns: O accumulator of warpgroup g at 128 * g, its S at 256 + 64 * g, its P (16-bit pairs) at 384 + 32 * g; Q (16-bit pairs)
constexpr uint32_t kTmO = 0, kTmS = 256, kTmP = 384, kTmQ = 448;

// shared memory map (offsets from the 1024-byte aligned base of dynamic shared memory)
template <int D> struct Lay {
    static constexpr int qTile = kQRows * D * 2;   // the Q tile, and the staged O tile
    static constexpr int qHalf = kQRows * 128;     // 64 columns of it: 128 rows x 128 B, 128B-swizzled
    static constexpr int tile = kBlk * D * 2;      // one K or V tile of 64 keys
    static constexpr int half = kBlk * 128;        // 64 columns of it
    static constexpr int offQ = 0;
    static constexpr int offK = offQ + qTile;
    static constexpr int offV = offK + kKSlots * tile;
    static constexpr int offBar = offV + kVSlots * tile;
    // barriers: k_full[6] k_empty[6] v_full[6] v_empty[6] q_full q_free s_full[2] s_free[2] p_full[2] pv_done[2]
    //           ml_ready o_free o_staged qt_full qt_free looked item_full[4] item_empty[4] v_ok[6]
    static constexpr int numBars = 2 * kKSlots + 3 * kVSlots + 2 + 8 + 6 + 2 * kItemRing;
    static constexpr int offMisc = offBar + numBars * 8;  // abort flag, TMEM base, whether a mixed unit held values that are not finite
    static constexpr int offItems = (offMisc + 96 + 31) / 32 * 32;  // [4] Item
    static constexpr int offMl = offItems + kItemRing * 32;         // [2 warpgroups][128 lanes] (maximum, row sum)
    static constexpr int smem = offMl + 2 * 128 * 8;
};

struct Item {  // n: units, -1: no more items.  All rows see the keys [all_lo, all_hi).
    int bh, tile, key0, n;
    int all_lo, all_hi;
    int near, pad;  // with a bias: number of the unit, counted from key0, that the tile's last query stands in or is nearest to
};

struct TcParams {
    CUtensorMap tm_q, tm_kv[2], tm_o;  // tm_kv[0]: K, [1]: V
    int fold_q, fold_k, fold_v, fold_o;  // bit 0: one head in the map, bit 1: one batch entry (axes with stride 0 or length 1)
    const int4* seen;
    const float* slopes;
    int* next_item;
    float* lse;
    void* rest;             // nullable, dense [B, Hq, Sq, D]: what rounding out to its type left
    const void* v;
    long long v_sb, v_sh, v_ss;
    unsigned int* status;
    int B, Hq, group, Sq, n_u, tiles, wave;
    uint32_t q_sign;        // flips the sign of Q: a negative scale
    ScoreShape shape;       // of the magnitude of the scale
};

// ------------------------------------------------------------------------------------------ kernel

__device__ __forceinline__ float2 get2(const uint32_t (&r)[64], int j) { return make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])); }
__device__ __forceinline__ void put2(uint32_t (&r)[64], int j, float2 v) {
    r[j] = __float_as_uint(v.x);
    r[j + 1] = __float_as_uint(v.y);
}
// the largest magnitude of a row of scores (a NaN is passed over: it stays one through the polynomial of the cap)
__device__ __forceinline__ float row_size(const uint32_t (&r)[64]) {
    float m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j += 2) m[k] = max3(m[k], fabsf(__uint_as_float(r[16 * k + j])), fabsf(__uint_as_float(r[16 * k + j + 1])));
    }
    return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

template <bool kBf16, int D, bool kCap, bool kBias>
__global__ void __launch_bounds__(kThreads, 1) dense_tc_kernel(const __grid_constant__ TcParams P) {
    using Ly = Lay<D>;
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar0 = sbase + Ly::offBar;
    auto bar_k_full = [&](int s) { return bar0 + 8u * s; };
    auto bar_k_empty = [&](int s) { return bar0 + 8u * (kKSlots + s); };
    auto bar_v_full = [&](int s) { return bar0 + 8u * (2 * kKSlots + s); };
    auto bar_v_empty = [&](int s) { return bar0 + 8u * (2 * kKSlots + kVSlots + s); };
    constexpr int kB0 = 2 * kKSlots + 2 * kVSlots;
    const uint32_t bar_q_full = bar0 + 8u * kB0, bar_q_free = bar0 + 8u * (kB0 + 1);
    auto bar_s_full = [&](int wg) { return bar0 + 8u * (kB0 + 2 + wg); };
    auto bar_s_free = [&](int wg) { return bar0 + 8u * (kB0 + 4 + wg); };
    auto bar_p_full = [&](int wg) { return bar0 + 8u * (kB0 + 6 + wg); };
    auto bar_pv_done = [&](int wg) { return bar0 + 8u * (kB0 + 8 + wg); };
    constexpr int kB1 = kB0 + 10;
    const uint32_t bar_ml_ready = bar0 + 8u * kB1, bar_o_free = bar0 + 8u * (kB1 + 1), bar_o_staged = bar0 + 8u * (kB1 + 2);
    const uint32_t bar_qt_full = bar0 + 8u * (kB1 + 3), bar_qt_free = bar0 + 8u * (kB1 + 4), bar_looked = bar0 + 8u * (kB1 + 5);
    auto bar_item_full = [&](unsigned n) { return bar0 + 8u * (kB1 + 6 + n % kItemRing); };
    auto bar_item_empty = [&](unsigned n) { return bar0 + 8u * (kB1 + 6 + kItemRing + n % kItemRing); };
    auto bar_v_ok = [&](int s) { return bar0 + 8u * (kB1 + 6 + 2 * kItemRing + s); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Ly::offMisc);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::offMisc + 32);
    volatile int* found_bad = reinterpret_cast<volatile int*>(smem + Ly::offMisc + 40);
    volatile int* slot_bad = reinterpret_cast<volatile int*>(smem + Ly::offMisc + 44);  // [6] of the tile in a V slot
    Item* items = reinterpret_cast<Item*>(smem + Ly::offItems);
    float2* ml = reinterpret_cast<float2*>(smem + Ly::offMl);  // [2][128]
    const Ctl ctl{abort_flag, P.status};

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same value, but provably warp-uniform

    if (tid == 0) {
        ctl_init(ctl);
        for (int s = 0; s < kKSlots; ++s) {
            mbar_init(bar_k_full(s), 1);
            mbar_init(bar_k_empty(s), 1);
        }
        for (int s = 0; s < kVSlots; ++s) {
            mbar_init(bar_v_full(s), 1);
            mbar_init(bar_v_empty(s), 1);
            mbar_init(bar_v_ok(s), 1);
        }
        mbar_init(bar_q_full, 1);
        mbar_init(bar_q_free, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_s_full(b), 1);
            mbar_init(bar_s_free(b), 4);
            mbar_init(bar_p_full(b), 4);  // one elected arrival per softmax warp
            mbar_init(bar_pv_done(b), 1);
        }
        mbar_init(bar_qt_full, 4);
        mbar_init(bar_qt_free, 1);
        mbar_init(bar_ml_ready, 8);
        mbar_init(bar_o_free, 4);
        mbar_init(bar_o_staged, 4);
        mbar_init(bar_looked, 1);
        for (int s = 0; s < kItemRing; ++s) {
            mbar_init(bar_item_full(s), 1);
            mbar_init(bar_item_empty(s), kItemReaders);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (sbase & 1023u) {  // the swizzled tiles need the base that the declaration asks for
            *abort_flag = 1;
            if (atomicCAS(P.status, 0u, 1u) == 0u) {
                P.status[1] = blockIdx.x;
                P.status[2] = sbase;
                P.status[3] = 0;
            }
        }
    }
    if (warp == 9) {  // TMEM: all 512 columns, allocated and freed by the S issuer
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const bool start_ok = *abort_flag == 0;
    const int bh_total = P.B * P.Hq;
    constexpr bool bf16 = kBf16;

    // Item number n of this CTA, as the first warp announced it.  Called by whole warps; each of the readers takes every item once.
    auto take_item = [&](unsigned n, Item& it) -> bool {
        if (!mbar_wait_warp(bar_item_full(n), (n / kItemRing) & 1, ctl, 14, n)) return false;
        const int4* p = reinterpret_cast<const int4*>(&items[n % kItemRing]);
        const int4 a = p[0], b = p[1];
        it.bh = a.x; it.tile = a.y; it.key0 = a.z; it.n = a.w;
        it.all_lo = b.x; it.all_hi = b.y; it.near = b.z;
        __syncwarp();
        mbar_arrive_elect(bar_item_empty(n));
        return true;
    };
    // First key of the unit that comes as number i.  With a bias the unit nearest to the tile's last query comes first, then those before it, going away,
    // then those behind it: scores grow towards a query's own place, and walking there would move its reference in every unit (16 heads,
    // 8192 tokens, causal: 392 us in ascending order, 270 in this one; every key seen: 630 and 528).
    auto unit_key = [](const Item& it, int i) { return it.key0 + kBlk * (!kBias || i > it.near ? i : it.near - i); };
    auto mixed_unit = [unit_key](const Item& it, int i) {
        const int k = unit_key(it, i);
        return k < it.all_lo || k + kBlk > it.all_hi;
    };
    // An item goes through an even number of units, at least two; those behind its own are empty.
    auto rounds = [](const Item& it) { return max(2, (it.n + 1) & ~1); };

    // Unit number gb (counted over the whole kernel) uses K slot gb % 6 and V slot gb % 6.  Within an item unit i belongs to warpgroup i & 1.
    if (!start_ok) {
    } else if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue));
        // ================================================================== epilogue warps (as in attn_tc.cu)
        const int wq = warp & 3;          // TMEM quadrant of this warp
        const int row = wq * 32 + lane;   // row of the tile = TMEM lane
        const uint32_t t_lane = (uint32_t)(wq * 32) << 16;
        unsigned char* const buf = smem + Ly::offQ + row * 128;  // this thread's row: chunk c at 16 * (c ^ (row & 7)), halves qHalf apart
        unsigned wk = 0, rr = 0;  // wk: items finished; rr: rounds of either softmax warpgroup over the whole kernel
        bool ok = true;
        Item cur, nx;
        cur.n = -1;
        for (unsigned n = 0;; ++n) {  // item n gets its Q, the one before (number wk) is finished
            ok = take_item(n, nx);
            if (!ok) break;
            const bool there = nx.n >= 0;
            if (there) {
                // the last S of the item before has read the columns
                if (n > 0) ok = mbar_wait_warp(bar_qt_free, (n - 1) & 1, ctl, 106, n);
                if (ok) ok = mbar_wait_warp(bar_q_full, n & 1, ctl, 108, n);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int half = 0; half < D / 64; ++half) {
                    uint32_t qr[32];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint4 v = *reinterpret_cast<const uint4*>(buf + half * Ly::qHalf + ((c ^ (row & 7)) << 4));
                        qr[4 * c + 0] = v.x ^ P.q_sign;
                        qr[4 * c + 1] = v.y ^ P.q_sign;
                        qr[4 * c + 2] = v.z ^ P.q_sign;
                        qr[4 * c + 3] = v.w ^ P.q_sign;
                    }
                    tc_st32(tmem + kTmQ + 32u * half + t_lane, qr);
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                mbar_arrive_elect(bar_qt_full);
            } else if (wk > 0) {
                // Behind the last item comes no Q, whose arrival would mean that the store of the item before has left the buffer.
                ok = mbar_wait_warp(bar_q_free, (wk - 1) & 1, ctl, 112, wk);
                if (!ok) break;
            }
            if (n > 0) {
                rr += rounds(cur) >> 1;
                // Both warpgroups have stored their last P, hence seen every PV but their last finish; no PV of the next item
                // starts before o_free, so the waits below are for exactly the item's last PVs.
                ok = mbar_wait_warp(bar_ml_ready, wk & 1, ctl, 104, wk);
                if (ok) ok = mbar_wait_warp(bar_looked, wk & 1, ctl, 105, wk);
                if (!ok) break;
                const bool bad = *found_bad != 0;
                const float2 ml0 = ml[row], ml1 = ml[128 + row];
                // merged scale of both partial sums: everything relative to the larger reference maximum.  A row with a NaN or an
                // infinite score has a NaN sum and comes out as NaN; a side that saw no key has the maximum -inf, hence the weight 0.
                const float m_all = fmaxf(ml0.x, ml1.x), m_base = m_all == -INFINITY ? 0.f : m_all;
                const float w0 = ex2(ml0.x - m_base), w1 = ex2(ml1.x - m_base);
                const float l_all = ml0.y * w0 + ml1.y * w1;
                const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
                const float f0 = w0 * inv, f1 = w1 * inv;
                const float2 f0_2 = make_float2(f0, f0), f1_2 = make_float2(f1, f1);
                const bool saw0 = cur.n > 0, saw1 = cur.n > 1;  // no unit: the accumulator holds garbage and is not used
                ok = mbar_wait_warp(bar_pv_done(0), (rr - 1) & 1, ctl, 100, wk);
                if (ok) ok = mbar_wait_warp(bar_pv_done(1), (rr - 1) & 1, ctl, 101, wk);
                if (!ok) break;
                tc_fence_after();
                const uint32_t tm_o = tmem + kTmO + t_lane;
                const int i_row = cur.tile * kQRows + row;
                const long long out_row = (long long)cur.bh * P.Sq + i_row;
#pragma unroll 1
                for (int cch = 0; cch < D / 32; ++cch) {
                    uint32_t oa[32], ob[32];
                    if (saw0) tc_ld32(tm_o + 32 * cch, oa);
                    if (saw1) tc_ld32(tm_o + 128 + 32 * cch, ob);
                    tc_wait_ld();
                    if (cch == D / 32 - 1) {  // both O accumulators may be overwritten by the next item's first PVs
                        tc_fence_before();
                        __syncwarp();
                        mbar_arrive_elect(bar_o_free);
                    }
                    if (LCBSA_UNLIKELY(!saw0)) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) oa[j] = 0u;
                    }
                    if (LCBSA_UNLIKELY(!saw1)) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) ob[j] = 0u;
                    }
                    unsigned char* const half = buf + (cch >> 1) * Ly::qHalf;
#pragma unroll
                    for (int q8 = 0; q8 < 4; ++q8) {
                        uint32_t pw[4], rw[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int e = q8 * 8 + 2 * j;
                            const float2 a2 = __fmul2_rn(make_float2(__uint_as_float(oa[e]), __uint_as_float(oa[e + 1])), f0_2);
                            const float2 v2 = __ffma2_rn(make_float2(__uint_as_float(ob[e]), __uint_as_float(ob[e + 1])), f1_2, a2);
                            pw[j] = pack2(bf16, v2.x, v2.y);
                            if (P.rest != nullptr) {
                                const T* r = reinterpret_cast<const T*>(&pw[j]);
                                rw[j] = pack2(bf16, v2.x - DType<T>::to_f32(r[0]), v2.y - DType<T>::to_f32(r[1]));
                            }
                        }
                        const int chunk = (cch & 1) * 4 + q8;
                        *reinterpret_cast<uint4*>(half + ((chunk ^ (row & 7)) << 4)) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
                        if (P.rest != nullptr && i_row < P.Sq)
                            *reinterpret_cast<uint4*>(static_cast<T*>(P.rest) + out_row * D + 32 * cch + 8 * q8) = make_uint4(rw[0], rw[1], rw[2], rw[3]);
                    }
                }
                if (LCBSA_UNLIKELY(bad)) {  // values of V that are not finite, to the rows that see them in mixed units
                    const int b = cur.bh / P.Hq, h = cur.bh - b * P.Hq;
                    const T* vh = static_cast<const T*>(P.v) + (long long)b * P.v_sb + (long long)(h / P.group) * P.v_sh;
                    const int4 see = i_row < P.Sq ? P.seen[((long long)b * P.n_u + i_row / kDenseUnit) * kSeenPitch + i_row % kDenseUnit] : make_int4(0, 0, 0, 0);
#pragma unroll 1
                    for (int i = 0; i < cur.n; ++i) {
                        if (!mixed_unit(cur, i)) continue;
                        const int k0 = unit_key(cur, i);
#pragma unroll 1
                        for (int key = max(k0, see.x); key < min(k0 + kBlk, see.y); ++key) {
#pragma unroll 1
                            for (int c = 0; c < D / 8; ++c) {
                                const uint4 raw = *reinterpret_cast<const uint4*>(vh + (long long)key * P.v_ss + c * 8);
                                if (!chunk_nonfinite<T>(raw)) continue;
                                T* dst = reinterpret_cast<T*>(buf + (c >> 3) * Ly::qHalf + (((c & 7) ^ (row & 7)) << 4));
                                const T* src = reinterpret_cast<const T*>(&raw);
#pragma unroll 1
                                for (int e = 0; e < 8; ++e) {
                                    const float x = DType<T>::to_f32(src[e]);
                                    if (!isfinite(x)) dst[e] = DType<T>::from_f32(DType<T>::to_f32(dst[e]) + x);
                                }
                            }
                        }
                    }
                }
                fence_proxy_async();
                __syncwarp();
                mbar_arrive_elect(bar_o_staged);
                if (P.lse != nullptr && i_row < P.Sq) P.lse[out_row] = l_all == 0.f ? -INFINITY : (m_all + log2f(l_all)) * kLn2;
                if (warp == 12) {  // the rows of all four warps are staged: off they go, then the buffer takes the Q after the next
                    ok = mbar_wait_warp(bar_o_staged, wk & 1, ctl, 110, wk);
                    if (!ok) break;
                    if (lane == 0) {
                        const int b = cur.bh / P.Hq, h = cur.bh - b * P.Hq;
                        const int ch = (P.fold_o & 1) ? 0 : h, cb = (P.fold_o & 2) ? 0 : b;
#pragma unroll
                        for (int half = 0; half < D / 64; ++half)
                            tma_store_5d(&P.tm_o, sbase + Ly::offQ + half * Ly::qHalf, 64 * half, cur.tile * kQRows, ch, cb, 0);
                        tma_store_commit();
                        tma_store_wait_read();
                        mbar_arrive(bar_q_free);
                    }
                    __syncwarp();
                }
                ++wk;
            }
            if (!there) break;
            cur = nx;
        }
        if (warp == 12 && lane == 0) tma_store_wait_all();
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
      if (warp == 8 || warp == 11) {
        // ================================================================== warp 8: items, Q and K; warp 11: V
        const bool is_k = warp == 8;
        const uint32_t ring = sbase + (is_k ? Ly::offK : Ly::offV), full0 = is_k ? bar_k_full(0) : bar_v_full(0), empty0 = is_k ? bar_k_empty(0) : bar_v_empty(0);
        const CUtensorMap* const tm = &P.tm_kv[is_k ? 0 : 1];
        const int fold = is_k ? P.fold_k : P.fold_v;
        unsigned gk = 0, wk = 0, nq_issued = 0;  // gk: units requested over the whole kernel
        int slot = 0, n_iter_done = 0;  // units of the item requested
        unsigned parity = 1;  // of the wait on an empty slot: the ring starts empty
        bool ok = true;
        auto request_q = [&](const Item& it) {  // Q tile of an item into the Q buffer
            if (lane == 0) {
                mbar_arrive_tx(bar_q_full, Ly::qTile);
                const int b = it.bh / P.Hq, h = it.bh - b * P.Hq;
                const int ch = (P.fold_q & 1) ? 0 : h, cb = (P.fold_q & 2) ? 0 : b;
#pragma unroll
                for (int half = 0; half < D / 64; ++half)
                    tma_load_5d(sbase + Ly::offQ + half * Ly::qHalf, &P.tm_q, bar_q_full, 64 * half, it.tile * kQRows, ch, cb, 0);
            }
            ++nq_issued;
            __syncwarp();
        };
        // Works out item `idx` of the launch and announces it as number n of this CTA.
        auto announce = [&](unsigned n, int idx, Item& it) -> bool {
            it.n = -1;
            it.bh = it.tile = it.key0 = it.all_lo = it.all_hi = it.near = 0;
            if (idx < bh_total * P.tiles) {
                dense_item(idx, bh_total, P.tiles, P.wave, it.bh, it.tile);
                it.tile = P.tiles - 1 - it.tile;
                const int4* u = P.seen + ((long long)(it.bh / P.Hq) * P.n_u + 2 * it.tile) * kSeenPitch + kDenseUnit;
                int4 a = __ldg(u), c = make_int4(0, 0, 0, 0x7fffffff);
                if (2 * it.tile + 1 < P.n_u) c = __ldg(u + kSeenPitch);
                const int lo = min(a.x < a.y ? a.x : 0x7fffffff, c.x < c.y ? c.x : 0x7fffffff), hi = max(a.y, c.y);
                it.n = hi > lo ? (hi - lo + kBlk - 1) / kBlk : 0;
                it.key0 = hi > lo ? lo : 0;
                it.all_lo = max(a.z, c.z);
                it.all_hi = min(a.w, c.w);
                if (kBias) {
                    const int last = min(it.tile * kQRows + kQRows, P.Sq) - 1;
                    const int pos = __ldg(&P.seen[((long long)(it.bh / P.Hq) * P.n_u + last / kDenseUnit) * kSeenPitch + last % kDenseUnit].z);
                    it.near = min(max((max(pos, 0) - it.key0) / kBlk, 0), max(it.n - 1, 0));
                }
            }
            if (!mbar_wait_warp(bar_item_empty(n), ((n / kItemRing) & 1) ^ 1, ctl, 16, n)) return false;
            if (lane == 0) {
                int4* p = reinterpret_cast<int4*>(&items[n % kItemRing]);
                p[0] = make_int4(it.bh, it.tile, it.key0, it.n);
                p[1] = make_int4(it.all_lo, it.all_hi, it.near, 0);
                mbar_arrive(bar_item_full(n));
            }
            __syncwarp();
            return true;
        };
        Item cur;
        if (is_k) {
            ok = announce(0, blockIdx.x, cur);
            if (ok && cur.n >= 0) request_q(cur);
        } else {
            ok = take_item(0, cur);
        }
        while (ok && cur.n >= 0) {
            const int b = cur.bh / P.Hq, h = (cur.bh - b * P.Hq) / P.group;
            const int ch = (fold & 1) ? 0 : h, cb = (fold & 2) ? 0 : b;
            const int n_iter = rounds(cur);
            // V of mixed units is looked through here, behind the copies: three units later, when it has come, and well before its P.
            auto look_at = [&](int j) -> bool {
                const unsigned g = gk - n_iter_done + j;  // number of unit j over the whole kernel
                const int vs = g % kVSlots;
                if (j < cur.n && mixed_unit(cur, j)) {
                    if (!mbar_wait_warp(bar_v_full(vs), (g / kVSlots) & 1, ctl, 24, g)) return false;
                    unsigned char* const v = smem + Ly::offV + vs * Ly::tile;
                    const bool bad = tile_nonfinite<T, Ly::tile / 16>(reinterpret_cast<const uint4*>(v), lane);
                    if (LCBSA_UNLIKELY(bad)) {
#pragma unroll 1
                        for (int c = lane; c < Ly::tile / 4; c += 32) {
                            uint32_t* p = reinterpret_cast<uint32_t*>(v) + c;
                            *p = zero_nonfinite<T>(*p);
                        }
                        fence_proxy_async();
                    }
                    if (lane == 0) slot_bad[vs] = bad;
                    __syncwarp();
                }
                mbar_arrive_elect(bar_v_ok(vs));
                return true;
            };
#pragma unroll 1
            for (int j = 0; j < n_iter; ++j) {
                ok = mbar_wait_warp(empty0 + 8u * slot, parity, ctl, is_k ? 20 : 22, gk);
                if (!ok) break;
                const uint32_t bar = full0 + 8u * slot, dst = ring + slot * Ly::tile;
                mbar_arrive_tx_elect(bar, j < cur.n ? Ly::tile : 0);
                if (j < cur.n) {
#pragma unroll
                    for (int half = 0; half < D / 64; ++half) tma_load_5d_elect(dst + half * Ly::half, tm, bar, 64 * half, unit_key(cur, j), ch, cb, 0);
                }
                ++gk;
                n_iter_done = j + 1;
                if (++slot == kKSlots) {
                    slot = 0;
                    parity ^= 1;
                }
                if (!is_k && j >= 3) {
                    ok = look_at(j - 3);
                    if (!ok) break;
                }
            }
            if (!ok) break;
            if (is_k) {
                // The next item, behind this one's last copies: six units of work are in the ring then.  Asked earlier, a CTA commits itself to
                // an item that it will not come to for long.
                int idx = 0;
                if (lane == 0) idx = (int)gridDim.x + atomicAdd(P.next_item, 1);
                ok = announce(wk + 1, __shfl_sync(0xffffffffu, idx, 0), cur);
                if (ok && cur.n >= 0) {  // its Q as soon as the buffer is free (see the epilogue warps)
                    ok = wk == 0 ? mbar_wait_warp(bar_qt_full, 0, ctl, 10, wk) : mbar_wait_warp(bar_q_free, (wk - 1) & 1, ctl, 11, wk);
                    if (ok) request_q(cur);
                }
            } else {
                for (int j = max(n_iter - 3, 0); j < n_iter && ok; ++j) ok = look_at(j);
                if (ok) ok = take_item(wk + 1, cur);
            }
            ++wk;
        }
        if (!ok && lane == 0) {
            // drain: give the copies this warp issued a bounded time to land before the CTA exits
            const long long t0 = clock64();
            for (unsigned r = gk > kKSlots ? gk - kKSlots : 0; r < gk; ++r)
                while (!mbar_try(full0 + 8u * (r % kKSlots), (r / kKSlots) & 1) && clock64() - t0 < 40000000ll) {
                }
            if (nq_issued > 0)
                while (!mbar_try(bar_q_full, (nq_issued - 1) & 1) && clock64() - t0 < 40000000ll) {
                }
        }
      } else if (warp == 9) {
        // ================================================================== S = Q K^T issuer
        const uint32_t idesc_s = instr_desc(bf16, kQRows, kBlk, 0);
        unsigned gb = 0, rr0 = 0, rr1 = 0;
        bool ok = true;
        Item cur;
        for (unsigned wk = 0; ok; ++wk) {
            ok = take_item(wk, cur);
            if (!ok || cur.n < 0) break;
            const int n_iter = rounds(cur);
            ok = mbar_wait_warp(bar_qt_full, wk & 1, ctl, 30, wk);  // Q of this item is in TMEM
            bool pre = false;
            for (int i = 0; i < n_iter && ok; ++i, ++gb) {
                const int wg = i & 1;
                const unsigned rr = wg ? rr1 : rr0;
                const int slot = gb % kKSlots;
                if (!pre) {  // not already seen ready by the look-ahead of the unit before
                    ok = mbar_wait_warp(bar_k_full(slot), (gb / kKSlots) & 1, ctl, 40, gb);
                    // the warpgroup has the S of its round before in registers
                    if (ok) ok = mbar_wait_warp(bar_s_free(wg), (rr & 1) ^ 1, ctl, 34 + wg, gb);
                    if (!ok) break;
                }
                // look ahead: probe the two barriers of the item's next unit now, read the answer after the MMAs
                bool nk = false, np = false;
                if (i + 1 < n_iter) {
                    nk = mbar_test(bar_k_full((gb + 1) % kKSlots), ((gb + 1) / kKSlots) & 1);
                    np = mbar_test(bar_s_free(wg ^ 1), ((wg ? rr0 : rr1) & 1) ^ 1);
                }
                tc_fence_after();
                if (i < cur.n) {
                    const uint64_t kd = smem_desc(sbase + Ly::offK + slot * Ly::tile, 16, 1024);
                    const uint32_t d = tmem + kTmS + 64u * wg;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        // 32 bytes per 16-column step inside a 64-column half
                        const uint64_t koff = (uint64_t)(((j >> 2) * Ly::half + (j & 3) * 32) >> 4);
                        tc_mma_ts(d, tmem + kTmQ + 8u * j, kd + koff, idesc_s, j > 0);
                    }
                }
                tc_commit(bar_k_empty(slot));  // K is free once these MMAs have read it
                tc_commit(bar_s_full(wg));
                __syncwarp();
                if (i == n_iter - 1) tc_commit(bar_qt_free);  // and so are Q's TMEM columns after the last S of the item
                if (wg) ++rr1; else ++rr0;
                pre = __all_sync(0xffffffffu, nk && np);
            }
        }
      } else if (warp == 10) {
        // ================================================================== O += P V issuer
        const uint32_t idesc_pv = instr_desc(bf16, kQRows, D, 1);
        unsigned gb = 0, rr0 = 0, rr1 = 0;
        bool ok = true;
        Item cur;
        for (unsigned wk = 0; ok; ++wk) {
            ok = take_item(wk, cur);
            if (!ok || cur.n < 0) break;
            const int n_iter = rounds(cur);
            // the epilogue of the previous item has read both O accumulators, and found_bad
            ok = mbar_wait_warp(bar_o_free, (wk & 1) ^ 1, ctl, 36, wk);
            if (!ok) break;
            int bad_item = 0;
            bool pre = false;
            for (int i = 0; i < n_iter && ok; ++i, ++gb) {
                const int wg = i & 1;
                const unsigned rr = wg ? rr1 : rr0;
                const int slot = gb % kVSlots;
                if (!pre) {
                    ok = mbar_wait_warp(bar_v_full(slot), (gb / kVSlots) & 1, ctl, 60, gb);
                    if (!ok) break;
                }
                if (i < cur.n && mixed_unit(cur, i)) {
                    ok = mbar_wait_warp(bar_v_ok(slot), (gb / kVSlots) & 1, ctl, 62, gb);
                    if (!ok) break;
                    bad_item |= slot_bad[slot];
                }
                if (i == n_iter - 1) {
                    if (lane == 0) {
                        *found_bad = bad_item;
                        mbar_arrive(bar_looked);
                    }
                    __syncwarp();
                }
                if (!pre) {
                    ok = mbar_wait_warp(bar_p_full(wg), rr & 1, ctl, 50 + wg, gb);
                    if (!ok) break;
                }
                bool nv = false, np = false;  // look ahead to the item's next unit
                if (i + 1 < n_iter) {
                    nv = mbar_test(bar_v_full((gb + 1) % kVSlots), ((gb + 1) / kVSlots) & 1);
                    np = mbar_test(bar_p_full(wg ^ 1), (wg ? rr0 : rr1) & 1);
                }
                tc_fence_after();
                // A: P in the warpgroup's 32 P columns, 8 columns per 16-key step.
                // B: V tile, MN-major: 64-column halves 8 KiB apart (LBO), 8-key groups 1 KiB apart (SBO).
                if (i < cur.n) {
                    const uint32_t pa = tmem + kTmP + 32u * wg;
                    const uint64_t vd = smem_desc(sbase + Ly::offV + slot * Ly::tile, Ly::half, 1024);
                    const uint32_t d = tmem + kTmO + 128u * wg;
#pragma unroll
                    for (int j = 0; j < kBlk / 16; ++j)
                        tc_mma_ts(d, pa + 8u * j, vd + (uint64_t)((j * 2048) >> 4), idesc_pv, (i > 1 || j > 0) ? 1u : 0u);
                }
                tc_commit(bar_v_empty(slot));
                tc_commit(bar_pv_done(wg));
                __syncwarp();
                if (wg) ++rr1; else ++rr0;
                pre = __all_sync(0xffffffffu, nv && np);
            }
        }
      }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ================================================================== softmax warpgroups
        const int wg = warp >> 2;         // warpgroup: takes units wg, wg + 2, ... of every work item
        const int wq = warp & 3;          // TMEM quadrant of this warp
        const int row = wq * 32 + lane;   // row of the tile = TMEM lane
        const uint32_t t_lane = (uint32_t)(wq * 32) << 16;
        const uint32_t tm_s = tmem + kTmS + 64u * wg + t_lane, tm_p = tmem + kTmP + 32u * wg + t_lane;
        const uint32_t tm_o_mine = tmem + kTmO + 128u * wg + t_lane;
        unsigned rr = 0;  // rounds of this warpgroup over the whole kernel
        bool ok = true;
        Item cur;
        for (unsigned wk = 0; ok; ++wk) {
            ok = take_item(wk, cur);
            if (!ok || cur.n < 0) break;
            const int n_iter = rounds(cur);
            const int b = cur.bh / P.Hq, i_row = cur.tile * kQRows + row;
            const int4 see = i_row < P.n_u * kDenseUnit ? P.seen[((long long)b * P.n_u + i_row / kDenseUnit) * kSeenPitch + i_row % kDenseUnit] : make_int4(0, 0, 0, 0);
            ScoreShape f = P.shape;
            if (kBias) f.slope2 = __ldg(P.slopes + (cur.bh - b * P.Hq)) * kLog2e;

            float m_ref = -INFINITY, l_sum = 0.f;
            bool first = true;  // no key of this item seen yet by this row in this warpgroup
            // S of the warpgroup's round into registers; the buffer is then free for the S of its next round
            uint32_t sr[64];
            ok = mbar_wait_warp(bar_s_full(wg), rr & 1, ctl, 80 + wg, rr);
            if (!ok) break;
            tc_fence_after();
            tc_ld64(tm_s, sr);
            tc_wait_ld();
            tc_fence_before();
            mbar_arrive_elect(bar_s_free(wg));
            for (int i = wg; i < n_iter && ok; i += 2, ++rr) {
                const bool active = i < cur.n;
                float alpha = 1.f;
                bool need = false;
                uint4 pk[8];  // this row of P in the input type, 8 keys per 16-byte chunk
                if (active) {
                    const int key0 = unit_key(cur, i);
                    // S -> exponents relative to the reference, in place (0 stands in for it until the row has seen a key)
                    const float m_eff = first ? 0.f : m_ref;
                    const float2 base = make_float2(-m_eff, -m_eff);
                    const float at = kBias ? (float)(see.z - key0) : 0.f;
                    const bool both_sides = kBias && __any_sync(0xffffffffu, at > 0.f && at < (float)(kBlk - 1));
                    auto plain = [&](float2 s, float2 c) { return __ffma2_rn(s, make_float2(f.mul, f.mul), c); };
                    auto small = [&](float2 s, float2 c) { return capped_small_plus(f, s, c); };
                    auto any = [&](float2 s, float2 c) { return capped_any_plus(f, s, c); };
                    auto row_max = [&]() {
                        float mx8[8];  // eight chains of eight values, three at a time
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            auto sv = [&](int i) { return __uint_as_float(sr[8 * i + k]); };
                            mx8[k] = fmaxf(max3(max3(max3(sv(0), sv(1), sv(2)), sv(3), sv(4)), sv(5), sv(6)), sv(7));
                        }
                        return fmaxf(max3(max3(mx8[0], mx8[1], mx8[2]), mx8[3], mx8[4]), max3(mx8[5], mx8[6], mx8[7]));
                    };
                    auto shift = [&](float by) {
                        const float2 b2 = make_float2(-by, -by);
#pragma unroll
                        for (int j = 0; j < 64; j += 2) put2(sr, j, __fadd2_rn(get2(sr, j), b2));
                    };
                    // Probabilities against the current reference, the row sum before their rounding.  exponent(pair number) gives two exponents.
                    auto probs = [&](float& rsum, auto exponent) {
                        float2 r01 = make_float2(0.f, 0.f), r23 = make_float2(0.f, 0.f);
#pragma unroll
                        for (int cch = 0; cch < 8; ++cch) {
                            float2 e[4];
#pragma unroll
                            for (int jp = 0; jp < 4; ++jp) {
                                const float2 x = exponent(cch * 4 + jp);
                                e[jp] = make_float2(ex2(x.x), ex2(x.y));
                            }
                            r01 = __fadd2_rn(r01, e[0]);
                            r23 = __fadd2_rn(r23, e[1]);
                            r01 = __fadd2_rn(r01, e[2]);
                            r23 = __fadd2_rn(r23, e[3]);
                            pk[cch].x = pack2(bf16, e[0].x, e[0].y);
                            pk[cch].y = pack2(bf16, e[1].x, e[1].y);
                            pk[cch].z = pack2(bf16, e[2].x, e[2].y);
                            pk[cch].w = pack2(bf16, e[3].x, e[3].y);
                        }
                        rsum = (r01.x + r01.y) + (r23.x + r23.y);
                    };
                    auto ready_made = [&](int pair) { return get2(sr, 2 * pair); };
                    bool large = false;
                    if constexpr (kCap) large = __any_sync(0xffffffffu, !(row_size(sr) <= f.s_fast));
                    const bool mixed = mixed_unit(cur, i);
                    float rs = 0.f;
                    // With a cap the exponents of the usual unit are made in the same pass as its probabilities, so that the arithmetic of one pair runs
                    // under the special functions of another (16 heads, 8192 tokens: 642 us in two passes, 549 in one).  Without one there
                    // is too little of it (453 and 467 us): the other units' way, exponents first, is every unit's.
                    constexpr bool kOnePass = kCap;
                    if (!kOnePass || LCBSA_UNLIKELY(mixed || large || both_sides || __any_sync(0xffffffffu, first))) {
                        auto exponents = [&](auto shaped, bool two_sides) {
                            BiasLine line;
                            if (kBias && !two_sides) line = bias_line(at, f.slope2, -m_eff);
#pragma unroll
                            for (int j = 0; j < 64; j += 2) {
                                float2 c = base;
                                if (kBias) {
                                    if (two_sides) c = __ffma2_rn(make_float2(fabsf(at - (float)j), fabsf(at - (float)(j + 1))), make_float2(-f.slope2, -f.slope2), base);
                                    else c = bias_next(line, j / 2);
                                }
                                put2(sr, j, shaped(get2(sr, j), c));
                            }
                        };
                        if constexpr (kCap) {
                            if (LCBSA_UNLIKELY(large)) exponents(any, true);
                            else exponents(small, true);
                        } else {
                            if (kBias && both_sides) exponents(plain, true);
                            else exponents(plain, false);
                        }
                        if (mixed) {
                            const int lo = min(max(see.x - key0, 0), kBlk), hi = min(max(see.y - key0, 0), kBlk);  // a run of bits
                            const uint64_t sees = hi > lo ? (~0ull >> (kBlk - (hi - lo))) << lo : 0ull;
                            const uint32_t s_lo = (uint32_t)sees, s_hi = (uint32_t)(sees >> 32);
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                if (!((s_lo >> j) & 1u)) sr[j] = 0xff800000u;  // -inf
                                if (!((s_hi >> j) & 1u)) sr[32 + j] = 0xff800000u;
                            }
                        }
                        // The first unit in which the row sees a key takes its own maximum as the reference.
                        if (LCBSA_UNLIKELY(first)) {
                            const float m = row_max();
                            if (m != -INFINITY) {
                                m_ref = m;
                                first = false;
                                shift(m);
                            }
                        }
                        probs(rs, ready_made);
                    } else {
                        BiasLine line;
                        if (kBias) line = bias_line(at, f.slope2, -m_eff);
                        probs(rs, [&](int pair) {
                            const float2 s = get2(sr, 2 * pair), c = kBias ? bias_next(line, pair) : base;
                            const float2 x = small(s, c);
                            put2(sr, 2 * pair, x);
                            return x;
                        });
                    }
                    // The row maximum was tracked beside them; only if it has moved by more than 2^8 is the pass repeated with the new reference.
                    const float m_top = row_max();
                    if (LCBSA_UNLIKELY(m_top > 8.f)) {
                        need = true;
                        alpha = ex2(-m_top);
                        m_ref += m_top;
                        shift(m_top);
                        probs(rs, ready_made);
                    }
                    l_sum = l_sum * alpha + rs;  // alpha is 1 unless this row's reference maximum moved
                }
                const bool any_need = __any_sync(0xffffffffu, need);
                // P may be overwritten, and O rescaled, once the warpgroup's PV of the round before has finished.  The next S
                // only waits for this one to be in registers, so it is usually there too: both barriers are probed at once
                // (a wait costs its warp 200 cycles even on a completed phase) and the next S is fetched under the store of P.
                const bool more = i + 2 < n_iter;
                const bool pv_ok = mbar_test(bar_pv_done(wg), (rr & 1) ^ 1), s_ok = !more || mbar_test(bar_s_full(wg), (rr + 1) & 1);
                const bool ready = __all_sync(0xffffffffu, pv_ok && s_ok);
                if (!ready) {
                    ok = mbar_wait_warp(bar_pv_done(wg), (rr & 1) ^ 1, ctl, 92 + wg, rr);
                    if (!ok) break;
                }
                tc_fence_after();  // orders the store of P behind the MMAs that read the columns (no other barrier does)
                uint32_t pr[32];  // all 32 lanes take part in the store (don't-cares for a unit that does not exist)
#pragma unroll
                for (int cch = 0; cch < 8; ++cch) {
                    pr[4 * cch + 0] = pk[cch].x;
                    pr[4 * cch + 1] = pk[cch].y;
                    pr[4 * cch + 2] = pk[cch].z;
                    pr[4 * cch + 3] = pk[cch].w;
                }
                if (LCBSA_UNLIKELY(any_need)) tc_scale_row<D>(tm_o_mine, alpha);  // rare: only when a row maximum jumps
                if (ready && more) {
                    tc_st32(tm_p, pr);
                    tc_ld64(tm_s, sr);
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive_elect(bar_p_full(wg));
                    tc_wait_ld();
                    tc_fence_before();
                    mbar_arrive_elect(bar_s_free(wg));
                } else {
                    tc_st32(tm_p, pr);
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive_elect(bar_p_full(wg));
                    if (more) {
                        ok = mbar_wait_warp(bar_s_full(wg), (rr + 1) & 1, ctl, 80 + wg, rr);
                        if (!ok) break;
                        tc_fence_after();
                        tc_ld64(tm_s, sr);
                        tc_wait_ld();
                        tc_fence_before();
                        mbar_arrive_elect(bar_s_free(wg));
                    }
                }
            }
            if (!ok) break;
            // The epilogue warps merge this item's partial results; they have read the (maximum, row sum) of the item before once
            // they have arrived on o_free.
            if (wk > 0) {
                if (!__all_sync(0xffffffffu, mbar_test(bar_o_free, (wk - 1) & 1))) {
                    ok = mbar_wait_warp(bar_o_free, (wk - 1) & 1, ctl, 102 + wg, wk);
                    if (!ok) break;
                }
            }
            ml[wg * 128 + row] = make_float2(first ? -INFINITY : m_ref, l_sum);  // no key seen: m_ref is a placeholder
            __syncwarp();
            mbar_arrive_elect(bar_ml_ready);
        }
    }

    // ---- teardown
    tc_fence_before();
    __syncthreads();
    if (tid == 0) ctl_report(ctl);
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

template <bool kBf16, int D, bool kCap, bool kBias>
cudaError_t tc_launch(const TcParams& P, int grid, cudaStream_t st) {
    static thread_local unsigned long long raised = 0;  // devices (below 64) whose shared-memory limit this thread has raised for this kernel
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !((raised >> dev) & 1)) {
        e = cudaFuncSetAttribute(dense_tc_kernel<kBf16, D, kCap, kBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::smem);
        if (e != cudaSuccess) return e;
        if (dev <= 63) raised |= 1ull << dev;
    }
    dense_tc_kernel<kBf16, D, kCap, kBias><<<grid, kThreads, Lay<D>::smem, st>>>(P);
    return cudaGetLastError();
}

template <bool kBf16, int D>
cudaError_t tc_shape(const TcParams& P, bool cap, int grid, cudaStream_t st) {
    if (cap) return P.slopes ? tc_launch<kBf16, D, true, true>(P, grid, st) : tc_launch<kBf16, D, true, false>(P, grid, st);
    return P.slopes ? tc_launch<kBf16, D, false, true>(P, grid, st) : tc_launch<kBf16, D, false, false>(P, grid, st);
}

}  // namespace

// A map over [B, H, S, D] rows, boxes of `box` rows x 64 columns.  Axes of length 1 or stride 0 become one entry (fold).
bool dense_rows_map(CUtensorMap* tm, int dtype, const View& v, int B, int H, int S, int D, int box, int* fold) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    *fold = (H == 1 || v.sh == 0 ? 1 : 0) | (B == 1 || v.sb == 0 ? 2 : 0);
    const long long row = S == 1 ? D : v.ss;
    const cuuint64_t one = (cuuint64_t)row * 2;  // any legal stride for an axis of one entry
    cuuint64_t dims[5] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)((*fold & 1) ? 1 : H), (cuuint64_t)((*fold & 2) ? 1 : B), 1};
    cuuint64_t strides[4] = {one, (*fold & 1) ? one : (cuuint64_t)v.sh * 2, (*fold & 2) ? one : (cuuint64_t)v.sb * 2, one};
    cuuint32_t boxes[5] = {64u, (cuuint32_t)box, 1u, 1u, 1u};
    cuuint32_t estr[5] = {1u, 1u, 1u, 1u, 1u};
    const CUtensorMapDataType dt = dtype == LCBSA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return fn(tm, dt, 5, const_cast<void*>(v.data), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool dense_tc_supported(const DenseArgs& a) {
    const View* vs[4] = {&a.q, &a.k, &a.v, &a.o};
    const int len[4] = {a.Sq, a.Sk, a.Sk, a.Sq};
    for (int i = 0; i < 4; ++i) {
        if (len[i] < 1 || (len[i] > 1 && vs[i]->ss == 0)) return false;
        if (vs[i]->ss * 2 >= (1ll << 40) || vs[i]->sh * 2 >= (1ll << 40) || vs[i]->sb * 2 >= (1ll << 40)) return false;
    }
    return (long long)a.B * a.Hq * ((a.Sq + kQRows - 1) / kQRows) < 0x7fff0000ll;
}

// The plan (rows, units, next_item zeroed) is in place when the kernel runs.
cudaError_t launch_dense_tc(const DenseArgs& a, cudaStream_t st, const char** why) {
    TcParams P;
    if (!dense_rows_map(&P.tm_q, a.dtype, a.q, a.B, a.Hq, a.Sq, a.D, kQRows, &P.fold_q) ||
        !dense_rows_map(&P.tm_kv[0], a.dtype, a.k, a.B, a.Hk, a.Sk, a.D, kBlk, &P.fold_k) ||
        !dense_rows_map(&P.tm_kv[1], a.dtype, a.v, a.B, a.Hk, a.Sk, a.D, kBlk, &P.fold_v) ||
        !dense_rows_map(&P.tm_o, a.dtype, a.o, a.B, a.Hq, a.Sq, a.D, kQRows, &P.fold_o)) {
        *why = "cuTensorMapEncodeTiled rejected a tensor";
        return cudaErrorInvalidValue;
    }
    P.seen = a.seen; P.slopes = a.slopes; P.next_item = a.next_item;
    P.lse = a.lse; P.rest = a.rest;
    P.v = a.v.data; P.v_sb = a.v.sb; P.v_sh = a.v.sh; P.v_ss = a.v.ss;
    P.status = a.status;
    P.B = a.B; P.Hq = a.Hq; P.group = a.group; P.Sq = a.Sq; P.n_u = dense_units(a.Sq);
    P.tiles = (a.Sq + kQRows - 1) / kQRows;
    P.wave = dense_wave(a.B * a.Hq, 4.0 * a.Sk * a.D / a.group);
    P.q_sign = a.scale < 0.f ? 0x80008000u : 0u;
    P.shape = score_shape(a.scale < 0.f ? -a.scale : a.scale, a.cap);
    int dev = 0, sm_count = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    const int usable = sm_count - attn_sm_reserve() > 0 ? sm_count - attn_sm_reserve() : 1;
    const long long work = (long long)a.B * a.Hq * P.tiles;
    const int grid = (int)(work < usable ? work : usable);
    const bool cap = a.cap > 0.f;
    if (a.dtype == LCBSA_BF16) return a.D == 128 ? tc_shape<true, 128>(P, cap, grid, st) : tc_shape<true, 64>(P, cap, grid, st);
    return a.D == 128 ? tc_shape<false, 128>(P, cap, grid, st) : tc_shape<false, 64>(P, cap, grid, st);
}

}  // namespace lcbsa
