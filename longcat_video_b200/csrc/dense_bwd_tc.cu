// Dense attention backward (see dense_common.cuh for the forward's formulas): dq, dk, dv from dout, the output and the lse.
//
//   delta_i = dout_i . o_i        p_ij = exp(x_ij - lse_i)        dv_j = sum_i p_ij dout_i
//   ds_ij = p_ij (dout_i . v_j - delta_i) (1 - tanh^2(s_ij / cap)) scale        dq_i = sum_j ds_ij k_j        dk_j = sum_i ds_ij q_i
//
// dk_j and dv_j also add up over the query heads that share the key head.  Two passes on TMA + tcgen05 + TMEM, so that every gradient is
// summed by one CTA in one order and nothing is added with atomics.  A CTA owns a tile pair (A1, A2) of 128 rows and walks pairs
// (B1, B2) of 64 rows:
//
//   dQ pass: A1 = Q  A2 = dO  B1 = K  B2 = V, over the keys that the rows see;   dK/dV pass: A1 = K  A2 = V  B1 = Q  B2 = dO, over
//   the query units that may see the keys, query head after query head of the group
//       S = A1 B1^T    dP = A2 B2^T    P, dS in registers, to TMEM in the input type    dQ += dS B1,  or  dV += P^T B2, dK += dS^T B1
//
// dS goes into its products without the factor scale, which the fp32 sums get when they are stored: a scale of 1 / sqrt(D) would move it three
// bits further into the subnormal numbers of fp16 (2048 keys, head_dim 64: dq off by 2.1 % for a dout of 10^-3 with it inside, 0.27 % outside; 0.21 and
// 0.038 % for 10^-2, 0.030 % for 1 either way).
// At the other end dS passes 65504 three bits earlier: at values of dout - which have the same limit - of some 10^4.
//
// The roles of the warps, the rings and the TMEM columns are those of the block-sparse backward for 128-token blocks (attn_bwd_tc.cu), where
// they are explained.  What differs: the walks are runs, so no lists are read; an entry is whole (all of its pairs are seen) or mixed, and
// only mixed ones are masked pair by pair; a query unit brings what its rows see along with its lse and delta.
//
// Hidden values may be anything.  A hidden pair's P and dS are set to zero; in mixed entries a producer looks through the tiles that are
// summed over, and once S and dP have read them the issuer of the gradient MMAs sets values that are not finite to zero (0 * inf is not 0).  A pair
// that is seen has its NaN from S and dP; for dV a mark in the place of the query's delta (kBadRow) says that dO is not finite.  (delta itself
// does not: it is the same where dO is finite and a value that the row sees is not, of which dV knows nothing.)
//
// Bound by the chain S -> P -> dP -> dS -> product and the operands' way from shared memory; two buffers of S and dP keep two entries in it.  37
// heads of 4096 tokens, head_dim 128 (ns for 128 x 64 pairs): dQ 650, with a cap 780; dK/dV 880 (1.4 PFLOP/s), with a cap 1040; tensor pipe 59
// and 61 % busy, 50 and 51 % with a cap.  Sixteen arithmetic warps with half a row of an entry each, not eight with a whole one, which
// leaves 104 registers a thread.  A third buffer of S^T in the place of the second dP^T: 920 in the place of 880.
//
// Every mbarrier wait is bounded; when one runs out the CTA flags the status word, drains its copies, frees TMEM, returns.
#include <cmath>
#include <type_traits>

#include "dense_common.cuh"
#include "tc_common.cuh"

namespace lcbsa {

namespace {

using namespace tc;

constexpr int kM = 128;                     // rows of an own tile
constexpr int kBlk = kDenseUnit;            // rows of a streamed tile
constexpr int kStatsBytes = kDenseStats * 4;  // of a query unit
constexpr int kSeenBytes = kSeenPitch * 16; // what its rows see
constexpr int kMathWarps = 16;
constexpr int kThreads = 32 * (kMathWarps + 4);
constexpr int kRegsMath = 104, kRegsOther = 64;  // setmaxnreg: (4 * 104 + 64) * 128 = the 60 K registers of the launch
constexpr int kItemRing = 4;

template <int D> struct Lay {
    static constexpr int aTile = kM * D * 2, aHalf = kM * 128;     // own tiles; a half: 64 columns, 128 B a row, 128B-swizzled
    static constexpr int bTile = kBlk * D * 2, bHalf = kBlk * 128;
    static constexpr int slots = D == 128 ? 4 : 8;                 // ring of (B1, B2) pairs
    static constexpr int extra = kStatsBytes + kSeenBytes;
    static constexpr int offA = 0;
    static constexpr int offB = offA + 2 * aTile;
    static constexpr int offExtra = offB + slots * 2 * bTile;
    static constexpr int offBar = offExtra + slots * extra;
    // barriers: full[slots], empty[slots], s_full[2], s_free[2], d_full[2], p_full[2], x_full[2], ts_done[2], a_full, a_empty, at_full,
    //           at_free, acc_done, acc_free, item_full[kItemRing], item_empty[kItemRing], looked[slots]
    static constexpr int numBars = 3 * slots + 12 + 6 + 2 * kItemRing;
    static constexpr int offMisc = (offBar + numBars * 8 + 15) / 16 * 16;  // abort flag, TMEM base
    static constexpr int offItems = offMisc + 80;
    static constexpr int smem = offItems + kItemRing * 32;
};
static_assert(Lay<128>::offExtra % 16 == 0 && Lay<128>::extra % 16 == 0 && Lay<128>::offBar % 8 == 0, "bulk copies and barriers are aligned");

// TMEM columns: two buffers of S and of dP.  P takes the columns of the S it comes from (dK/dV pass) and dS those of its dP, in two pieces of
// 16: the columns 32 h .. 32 h + 31 belong to the warps that work on half h, which have read them.
// dQ pass: dQ 0, S 128 and 192, dP 256 and 320, Q 384, dO 448.  dK/dV pass: dK 0, dV 128, S^T 256 and 320, dP^T 384 and 448; K and V stay in
// shared memory.
template <int kMode> struct Cols;
template <> struct Cols<0> {
    static constexpr uint32_t acc1 = 0, acc2 = 0, own1 = 384, own2 = 448;
    __device__ static __forceinline__ uint32_t s(int buf) { return 128u + 64u * buf; }
    __device__ static __forceinline__ uint32_t dp(int buf) { return 256u + 64u * buf; }
};
template <> struct Cols<1> {
    static constexpr uint32_t acc1 = 0, acc2 = 128, own1 = 0, own2 = 0;
    __device__ static __forceinline__ uint32_t s(int buf) { return 256u + 64u * buf; }
    __device__ static __forceinline__ uint32_t dp(int buf) { return 384u + 64u * buf; }
};
// 16-row step j of P or dS, relative to the columns of its S or dP
__device__ __forceinline__ uint32_t piece(int j) { return 32u * (j >> 1) + 8u * (j & 1); }

struct BwdParams {
    CUtensorMap tm_a1, tm_a2, tm_b1, tm_b2;
    int fold_a1, fold_a2, fold_b1, fold_b2;  // bit 0: one head in the map, bit 1: one batch entry
    const int4* seen;
    const int2* hulls;
    const float* stats;
    const float* slopes;
    int* next_item;
    unsigned int* status;
    void *out1, *out2;  // dQ pass: dq; dK/dV pass: dk, dv
    long long o1_sb, o1_sh, o1_ss, o2_sb, o2_sh, o2_ss;
    int B, Hq, Hk, group, n_u, n_k;  // query units, key units of an entry
    int heads, n_own, rows;          // heads, own tiles of a head and rows of the own axis
    // dK/dV pass: the query heads of a group are split over `splits` items of `walk` heads each, whose sums go to part [2][B * Hk * splits][Sk][D]
    int splits, walk;
    float* part;
    int n_items, wave;
    float scale;
    ScoreShape shape;
};

// called by a whole converged warp with warp-uniform operands, like the _elect copies of tc_common.cuh
__device__ __forceinline__ void bulk_load_elect(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}

// 32 columns of this thread's accumulator row -> 64 bytes of the row in global memory (input type)
template <bool kBf16>
__device__ __forceinline__ void store_row32(unsigned char* row_ptr, int col0, const uint32_t (&r)[32]) {
#pragma unroll
    for (int q8 = 0; q8 < 4; ++q8) {
        uint4 pk;
        pk.x = pack2(kBf16, __uint_as_float(r[q8 * 8 + 0]), __uint_as_float(r[q8 * 8 + 1]));
        pk.y = pack2(kBf16, __uint_as_float(r[q8 * 8 + 2]), __uint_as_float(r[q8 * 8 + 3]));
        pk.z = pack2(kBf16, __uint_as_float(r[q8 * 8 + 4]), __uint_as_float(r[q8 * 8 + 5]));
        pk.w = pack2(kBf16, __uint_as_float(r[q8 * 8 + 6]), __uint_as_float(r[q8 * 8 + 7]));
        *reinterpret_cast<uint4*>(row_ptr + (col0 + q8 * 8) * 2) = pk;
    }
}

// whether one of the scores is too large for the polynomial of the cap (a NaN is passed over: it stays one through it)
__device__ __forceinline__ bool any_large(const uint32_t (&r)[32], float s_fast) {
    float m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j += 2) m[k] = max3(m[k], fabsf(__uint_as_float(r[8 * k + j])), fabsf(__uint_as_float(r[8 * k + j + 1])));
    }
    return __any_sync(0xffffffffu, !(fmaxf(max3(m[0], m[1], m[2]), m[3]) <= s_fast));
}

// kMode 0: dQ pass, 1: dK/dV pass.  Persistent, one CTA per SM.
template <bool kBf16, int D, int kMode, bool kCap, bool kBias>
__global__ void __launch_bounds__(kThreads, 1) dense_bwd_tc_kernel(const __grid_constant__ BwdParams P) {
    using C = Cols<kMode>;
    using Ly = Lay<D>;
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    constexpr int kSlots = Ly::slots, kB = 2 * kSlots, kHalves = D / 64;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar0 = sbase + Ly::offBar;
    // Entries are numbered over the whole kernel: entry s uses ring slot s % kSlots, buffer s % 2 of S and dP, and is
    // worked on by the warpgroups 2 (s % 2) and 2 (s % 2) + 1, half of its columns each.  Items with entries
    // are numbered too, for the barriers that turn once an item.
    auto bar_full = [&](int s) { return bar0 + 8u * s; };
    auto bar_empty = [&](int s) { return bar0 + 8u * (kSlots + s); };
    auto bar_s_full = [&](int buf) { return bar0 + 8u * (kB + buf); };
    auto bar_s_free = [&](int buf) { return bar0 + 8u * (kB + 2 + buf); };  // dQ pass: S is in registers; dK/dV pass: P has been read
    auto bar_d_full = [&](int buf) { return bar0 + 8u * (kB + 4 + buf); };
    auto bar_p_full = [&](int buf) { return bar0 + 8u * (kB + 6 + buf); };
    auto bar_x_full = [&](int buf) { return bar0 + 8u * (kB + 8 + buf); };
    auto bar_ts_done = [&](int buf) { return bar0 + 8u * (kB + 10 + buf); };
    const uint32_t bar_a_full = bar0 + 8u * (kB + 12), bar_a_empty = bar0 + 8u * (kB + 13), bar_at_full = bar0 + 8u * (kB + 14);
    const uint32_t bar_at_free = bar0 + 8u * (kB + 15), bar_acc_done = bar0 + 8u * (kB + 16), bar_acc_free = bar0 + 8u * (kB + 17);
    auto bar_item_full = [&](int k) { return bar0 + 8u * (kB + 18 + k); };
    auto bar_item_empty = [&](int k) { return bar0 + 8u * (kB + 18 + kItemRing + k); };
    auto bar_looked = [&](int s) { return bar0 + 8u * (kB + 18 + 2 * kItemRing + s); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Ly::offMisc);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Ly::offMisc + 32);
    volatile int* slot_bad = reinterpret_cast<volatile int*>(smem + Ly::offMisc + 36);  // [slots] bit 0: B1, 1: B2 holds a value that is not finite
    int4* items = reinterpret_cast<int4*>(smem + Ly::offItems);
    const Ctl ctl{abort_flag, P.status};

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // provably warp-uniform
    if (tid == 0) {
        ctl_init(ctl);
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(bar_full(s), 2);  // one arrival per producer
            mbar_init(bar_empty(s), 1);
            mbar_init(bar_looked(s), 1);
        }
        for (int buf = 0; buf < 2; ++buf) {
            mbar_init(bar_s_full(buf), 1);
            mbar_init(bar_s_free(buf), kMode == 1 ? 1 : 8);  // one elected arrival per warp that works on an entry
            mbar_init(bar_d_full(buf), 1);
            mbar_init(bar_p_full(buf), 8);
            mbar_init(bar_x_full(buf), 8);
            mbar_init(bar_ts_done(buf), 1);
        }
        mbar_init(bar_a_full, 1);
        mbar_init(bar_a_empty, kMode == 1 ? 1 : kMathWarps);  // the arithmetic warps have moved it; dK/dV pass: the last S and dP have read it
        mbar_init(bar_at_full, kMathWarps);
        mbar_init(bar_at_free, 1);
        mbar_init(bar_acc_done, 1);
        mbar_init(bar_acc_free, kMathWarps);
        for (int k = 0; k < kItemRing; ++k) {
            mbar_init(bar_item_full(k), 1);
            mbar_init(bar_item_empty(k), kMathWarps + 3);  // every warp but the one that announces
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
    if (warp == kMathWarps + 1) {  // TMEM: all 512 columns, allocated and freed by the issuing warp
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const bool start_ok = *abort_flag == 0;  // else nothing runs, nothing is written

    // An item: own tile `own` of head bh, n entries.  dQ pass: keys from `first` on, all rows see [all_lo, all_hi).  dK/dV pass: `span` query units
    // from unit `first` on, for every query head of the group.  bh < 0: there is none, or the kernel is giving up.
    struct Item {
        int bh, own, first, n, all_lo, all_hi, span;
    };
    auto take_item = [&](unsigned k) {  // item number k of this CTA, for every warp but the one that announces
        Item it{-1, 0, 0, 0, 0, 0, 0};
        if (!mbar_wait_warp(bar_item_full(k % kItemRing), (k / kItemRing) & 1, ctl, 200, k)) return it;
        const int4 a = items[2 * (k % kItemRing)], c = items[2 * (k % kItemRing) + 1];
        __syncwarp();
        mbar_arrive_elect(bar_item_empty(k % kItemRing));
        return Item{a.x, a.y, a.z, a.w, c.x, c.y, c.z};
    };
    // Whether some pair of an entry is hidden.  dQ pass: entry e of the item; dK/dV pass: the unit's summary against the own keys
    auto mixed_keys = [](const Item& it, int e) {
        const int k = it.first + kBlk * e;
        return k < it.all_lo || k + kBlk > it.all_hi;
    };
    auto mixed_queries = [&P](const Item& it, const int4& unit) {
        const int k = it.own * kM;
        return k < unit.z || min(k + kM, P.rows) > unit.w;  // rows behind the last key are not stored
    };
    auto seen_of_slot = [&](int slot) { return reinterpret_cast<const int4*>(smem + Ly::offExtra + slot * Ly::extra + kStatsBytes); };

    if (warp >= kMathWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (!start_ok) {
        } else if (warp == kMathWarps || warp == kMathWarps + 3) {
            // ================================================================== TMA producers: one for items, own tiles, B1 and what comes with it, one for B2
            const bool is_b1 = warp == kMathWarps;
            const CUtensorMap* tm = is_b1 ? &P.tm_b1 : &P.tm_b2;
            const int fold = is_b1 ? P.fold_b1 : P.fold_b2;
            bool ok = true;
            unsigned s = 0, kk = 0;  // entries, items with entries
            int ahead2 = 0;          // number taken off the counter for the item behind the next
            Item ahead{-1, 0, 0, 0, 0, 0, 0};
            auto take = [&]() { return lane == 0 ? (int)gridDim.x + atomicAdd(P.next_item, 1) : 0; };
            auto look = [&](int id) {
                Item it{-1, 0, 0, 0, 0, 0, 0};
                if (id >= P.n_items) return it;
                dense_item(id, P.B * P.heads, P.n_own, P.wave, it.bh, it.own);
                const int b = it.bh / P.heads;
                if (kMode == 0) {  // the last queries first: with a causal order they have most keys
                    it.own = P.n_own - 1 - it.own;
                    const int4* u = P.seen + ((long long)b * P.n_u + 2 * it.own) * kSeenPitch + kBlk;
                    int4 x = __ldg(u), y = make_int4(0, 0, 0, 0x7fffffff);
                    if (2 * it.own + 1 < P.n_u) y = __ldg(u + kSeenPitch);
                    const int lo = min(x.x < x.y ? x.x : 0x7fffffff, y.x < y.y ? y.x : 0x7fffffff), hi = max(x.y, y.y);
                    it.n = hi > lo ? (hi - lo + kBlk - 1) / kBlk : 0;
                    it.first = hi > lo ? lo : 0;
                    it.all_lo = max(x.z, y.z);
                    it.all_hi = min(x.w, y.w);
                } else {  // the first keys first
                    const int2* hu = P.hulls + (long long)b * P.n_k + 2 * it.own;
                    int2 x = __ldg(hu);
                    if (2 * it.own + 1 < P.n_k) {
                        const int2 y = __ldg(hu + 1);
                        if (x.x >= x.y) x = y;
                        else if (y.x < y.y) x = make_int2(min(x.x, y.x), max(x.y, y.y));
                    }
                    if (x.x < x.y) {
                        it.first = x.x / kBlk;
                        it.span = (x.y - 1) / kBlk - it.first + 1;
                        it.n = it.span * P.walk;
                    }
                }
                return it;
            };
            if (is_b1) {
                ahead = look(blockIdx.x);
                ahead2 = take();
            }
            auto step = [&]() {
                ahead = look(__shfl_sync(0xffffffffu, ahead2, 0));
                ahead2 = take();
            };
            for (unsigned k = 0;; ++k) {
                Item it;
                if (is_b1) {
                    it = ahead;
                    ok = mbar_wait_warp(bar_item_empty(k % kItemRing), ((k / kItemRing) & 1) ^ 1, ctl, 201, k);
                    if (!ok) break;
                    if (lane == 0) {
                        items[2 * (k % kItemRing)] = make_int4(it.bh, it.own, it.first, it.n);
                        items[2 * (k % kItemRing) + 1] = make_int4(it.all_lo, it.all_hi, it.span, 0);
                        mbar_arrive(bar_item_full(k % kItemRing));
                    }
                    __syncwarp();
                } else {
                    it = take_item(k);
                }
                if (it.bh < 0) break;
                if (it.n == 0) {
                    if (is_b1) step();
                    continue;
                }
                const int b = it.bh / P.heads, h = it.bh % P.heads;
                if (is_b1) {
                    ok = mbar_wait_warp(bar_a_empty, (kk & 1) ^ 1, ctl, 202, kk);
                    if (!ok) break;
                    mbar_arrive_tx_elect(bar_a_full, 2 * Ly::aTile);
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        const int own_h = kMode == 0 ? h : h / P.splits;
                        tma_load_5d_elect(sbase + Ly::offA + half * Ly::aHalf, &P.tm_a1, bar_a_full, 64 * half, it.own * kM,
                                          (P.fold_a1 & 1) ? 0 : own_h, (P.fold_a1 & 2) ? 0 : b, 0);
                        tma_load_5d_elect(sbase + Ly::offA + Ly::aTile + half * Ly::aHalf, &P.tm_a2, bar_a_full, 64 * half, it.own * kM,
                                          (P.fold_a2 & 1) ? 0 : own_h, (P.fold_a2 & 2) ? 0 : b, 0);
                    }
                }
                ++kk;
                int e_done = 0;  // entries of the item requested
                // Tiles of mixed entries that are summed over (dQ pass: K; dK/dV pass: Q and dO) are looked through behind the copies, two entries
                // later, when they have come, and well before their dS.
                auto look_at = [&](int e) -> bool {
                    const unsigned g = s - e_done + e;  // number of entry e over the whole kernel
                    const int ls = g % kSlots;
                    bool mixed = kMode == 0 && mixed_keys(it, e);
                    if (kMode == 1 || mixed) {
                        if (!mbar_wait_warp(bar_full(ls), (g / kSlots) & 1, ctl, 214 + kMode, g)) return false;
                        if (kMode == 1) mixed = mixed_queries(it, seen_of_slot(ls)[kBlk]);
                    }
                    if (mixed) {
                        const uint4* t = reinterpret_cast<const uint4*>(smem + Ly::offB + ls * 2 * Ly::bTile);
                        int bad = tile_nonfinite<T, Ly::bTile / 16>(t, lane) ? 1 : 0;
                        if (kMode == 1 && tile_nonfinite<T, Ly::bTile / 16>(t + Ly::bTile / 16, lane)) bad |= 2;
                        if (lane == 0) slot_bad[ls] = bad;
                        __syncwarp();
                    }
                    mbar_arrive_elect(bar_looked(ls));
                    return true;
                };
                int unit = it.first, head = kMode == 0 ? h / P.group : h * P.walk;  // of the entry: dK/dV pass a query unit, dQ pass unused
                for (int e = 0; e < it.n; ++e) {
                    const int slot = s % kSlots;
                    ok = mbar_wait_warp(bar_empty(slot), ((s / kSlots) & 1) ^ 1, ctl, 210 + kMode, s);
                    if (!ok) break;
                    ++s;
                    const bool more = kMode == 1 && is_b1;
                    mbar_arrive_tx_elect(bar_full(slot), Ly::bTile + (more ? Ly::extra : 0));
                    const uint32_t dst = sbase + Ly::offB + slot * 2 * Ly::bTile + (is_b1 ? 0 : Ly::bTile);
                    const int row = kMode == 0 ? it.first + kBlk * e : unit * kBlk;
#pragma unroll
                    for (int half = 0; half < kHalves; ++half)
                        tma_load_5d_elect(dst + half * Ly::bHalf, tm, bar_full(slot), 64 * half, row, (fold & 1) ? 0 : head, (fold & 2) ? 0 : b, 0);
                    if (more) {
                        const uint32_t x = sbase + Ly::offExtra + slot * Ly::extra;
                        bulk_load_elect(x, P.stats + (((long long)b * P.Hq + head) * P.n_u + unit) * kDenseStats, kStatsBytes, bar_full(slot));
                        bulk_load_elect(x + kStatsBytes, P.seen + ((long long)b * P.n_u + unit) * kSeenPitch, kSeenBytes, bar_full(slot));
                    }
                    if (kMode == 1 && ++unit == it.first + it.span) {
                        unit = it.first;
                        ++head;
                    }
                    e_done = e + 1;
                    if (!is_b1 && e >= 2) {
                        ok = look_at(e - 2);
                        if (!ok) break;
                    }
                    if (is_b1 && e == it.n - 1) step();  // behind the item's last copies, none of which waits for the counter
                }
                if (!is_b1)
                    for (int e = max(it.n - 2, 0); e < it.n && ok; ++e) ok = look_at(e);
                if (!ok) break;
            }
            if ((!ok || *abort_flag != 0) && lane == 0) {
                // drain: give the copies this warp issued a bounded time to land before the CTA exits
                const long long t0 = clock64();
                while (is_b1 && kk > 0 && !mbar_try(bar_a_full, (kk - 1) & 1) && clock64() - t0 < 40000000ll) {
                }
                for (unsigned r = s > kSlots ? s - kSlots : 0; r < s; ++r)
                    while (!mbar_try(bar_full(r % kSlots), (r / kSlots) & 1) && clock64() - t0 < 40000000ll) {
                    }
            }
        } else if (warp == kMathWarps + 1) {
            // ================================================================== issuer of S and dP (S^T and dP^T)
            const uint32_t idesc_ss = instr_desc(kBf16, kM, kBlk, 0);
            const uint64_t a1d = smem_desc(sbase + Ly::offA, 16, 1024), a2d = smem_desc(sbase + Ly::offA + Ly::aTile, 16, 1024);  // dK/dV pass
            bool ok = true;
            unsigned s = 0, kk = 0;
            for (unsigned k = 0; ok; ++k) {
                const Item it = take_item(k);
                if (it.bh < 0) break;
                if (it.n == 0) continue;
                if (kMode == 0) ok = mbar_wait_warp(bar_at_full, kk & 1, ctl, 220, kk);  // the own tiles are in TMEM
                else ok = mbar_wait_warp(bar_a_full, kk & 1, ctl, 242, kk);
                ++kk;
                bool pre = false;
                for (int e = 0; e < it.n && ok; ++e, ++s) {
                    const int slot = s % kSlots, buf = s & 1;
                    const uint32_t before = ((s >> 1) & 1) ^ 1;  // parity of the buffer's use before
                    if (!pre) {  // not already seen ready by the look-ahead of the entry before
                        ok = mbar_wait_warp(bar_full(slot), (s / kSlots) & 1, ctl, 222 + kMode, s);
                        if (ok) ok = mbar_wait_warp(bar_s_free(buf), before, ctl, 226, s);
                        if (!ok) break;
                    }
                    tc_fence_after();
                    const uint32_t tile = sbase + Ly::offB + slot * 2 * Ly::bTile;
                    const uint64_t b1d = smem_desc(tile, 16, 1024), b2d = smem_desc(tile + Ly::bTile, 16, 1024);
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        // 32 bytes per 16-column step inside a 64-column half; 8 TMEM columns per step
                        const uint64_t off = (uint64_t)(((j >> 2) * Ly::bHalf + (j & 3) * 32) >> 4);
                        const uint64_t aoff = (uint64_t)(((j >> 2) * Ly::aHalf + (j & 3) * 32) >> 4);
                        if (kMode == 1) tc_mma(tmem + C::s(buf), a1d + aoff, b1d + off, idesc_ss, j > 0);
                        else tc_mma_ts(tmem + C::s(buf), tmem + C::own1 + 8u * j, b1d + off, idesc_ss, j > 0);
                    }
                    tc_commit(bar_s_full(buf));
                    __syncwarp();
                    // the gradient MMAs of entry s - 2 have read dS from dP's columns
                    if (!__all_sync(0xffffffffu, mbar_test(bar_ts_done(buf), before))) {
                        ok = mbar_wait_warp(bar_ts_done(buf), before, ctl, 227, s);
                        if (!ok) break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        const uint64_t off = (uint64_t)(((j >> 2) * Ly::bHalf + (j & 3) * 32) >> 4);
                        const uint64_t aoff = (uint64_t)(((j >> 2) * Ly::aHalf + (j & 3) * 32) >> 4);
                        if (kMode == 1) tc_mma(tmem + C::dp(buf), a2d + aoff, b2d + off, idesc_ss, j > 0);
                        else tc_mma_ts(tmem + C::dp(buf), tmem + C::own2 + 8u * j, b2d + off, idesc_ss, j > 0);
                    }
                    tc_commit(bar_d_full(buf));
                    if (e == it.n - 1) tc_commit(kMode == 1 ? bar_a_empty : bar_at_free);  // the own tiles have been read
                    __syncwarp();
                    bool nf = false, ns = false;
                    if (e + 1 < it.n) {
                        nf = mbar_test(bar_full((s + 1) % kSlots), ((s + 1) / kSlots) & 1);
                        ns = mbar_test(bar_s_free(buf ^ 1), (((s + 1) >> 1) & 1) ^ 1);
                    }
                    pre = __all_sync(0xffffffffu, nf && ns);
                }
            }
        } else if (warp == kMathWarps + 2) {
            // ================================================================== issuer of the gradient MMAs: A from TMEM (8 columns
            // per 16-row step), B the streamed tile, MN-major (64-column halves apart = LBO, 8-row groups 1 KiB apart = SBO, 16
            // rows = 2 KiB per step)
            const uint32_t idesc_ts = instr_desc(kBf16, kM, D, 1);
            bool ok = true;
            unsigned s = 0, kk = 0;
            for (unsigned k = 0; ok; ++k) {
                const Item it = take_item(k);
                if (it.bh < 0) break;
                if (it.n == 0) continue;
                ok = mbar_wait_warp(bar_acc_free, (kk & 1) ^ 1, ctl, 244, kk);  // the gradients of the item before have been read
                ++kk;
                bool pre = false;
                for (int e = 0; e < it.n && ok; ++e, ++s) {
                    const int slot = s % kSlots, buf = s & 1;
                    if (!pre) {
                        ok = mbar_wait_warp(bar_full(slot), (s / kSlots) & 1, ctl, 228 + kMode, s);
                        if (!ok) break;
                    }
                    unsigned char* const tiles = smem + Ly::offB + slot * 2 * Ly::bTile;
                    const uint32_t tile = sbase + Ly::offB + slot * 2 * Ly::bTile;
                    const uint64_t b1m = smem_desc(tile, Ly::bHalf, 1024), b2m = smem_desc(tile + Ly::bTile, Ly::bHalf, 1024);
                    const bool mixed = kMode == 0 ? mixed_keys(it, e) : mixed_queries(it, seen_of_slot(slot)[kBlk]);
                    // once S and dP of the entry have read the tile
                    auto clean = [&](int from) {
#pragma unroll 1
                        for (int c = lane; c < Ly::bTile / 4; c += 32) {
                            uint32_t* p = reinterpret_cast<uint32_t*>(tiles + from) + c;
                            *p = zero_nonfinite<T>(*p);
                        }
                        fence_proxy_async();
                        __syncwarp();
                    };
                    int bad = 0;
                    if (mixed) {
                        ok = mbar_wait_warp(bar_looked(slot), (s / kSlots) & 1, ctl, 247, s);
                        if (!ok) break;
                        bad = slot_bad[slot];
                    }
                    if (kMode == 1) {
                        if (!__all_sync(0xffffffffu, mbar_test(bar_p_full(buf), (s >> 1) & 1))) {
                            ok = mbar_wait_warp(bar_p_full(buf), (s >> 1) & 1, ctl, 245, s);
                            if (!ok) break;
                        }
                        if (LCBSA_UNLIKELY(bad & 2)) {
                            ok = mbar_wait_warp(bar_d_full(buf), (s >> 1) & 1, ctl, 246, s);  // dP has read dO
                            if (!ok) break;
                            clean(Ly::bTile);
                        }
                        tc_fence_after();
#pragma unroll
                        for (int j = 0; j < kBlk / 16; ++j)  // dV += P^T dO
                            tc_mma_ts(tmem + C::acc2, tmem + C::s(buf) + piece(j), b2m + (uint64_t)((j * 2048) >> 4), idesc_ts, (e > 0 || j > 0) ? 1u : 0u);
                        tc_commit(bar_s_free(buf));  // P's columns are S's
                        __syncwarp();
                    }
                    if (!pre) {
                        ok = mbar_wait_warp(bar_x_full(buf), (s >> 1) & 1, ctl, 224 + kMode, s);
                        if (!ok) break;
                    }
                    if (LCBSA_UNLIKELY(bad & 1)) clean(0);
                    bool nf = false, nx = false;
                    if (e + 1 < it.n) {
                        nf = mbar_test(bar_full((s + 1) % kSlots), ((s + 1) / kSlots) & 1);
                        nx = mbar_test(bar_x_full(buf ^ 1), ((s + 1) >> 1) & 1);
                    }
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < kBlk / 16; ++j)  // dQ += dS K, or dK += dS^T Q
                        tc_mma_ts(tmem + C::acc1, tmem + C::dp(buf) + piece(j), b1m + (uint64_t)((j * 2048) >> 4), idesc_ts, (e > 0 || j > 0) ? 1u : 0u);
                    tc_commit(bar_empty(slot));  // the streamed tiles are free once these MMAs have read them
                    tc_commit(bar_ts_done(buf)); // and so is dS
                    if (e == it.n - 1) tc_commit(bar_acc_done);
                    __syncwarp();
                    pre = __all_sync(0xffffffffu, nf && nx);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMath));
        // ================================================================== arithmetic warps
        const int wg = warp >> 3, half = (warp >> 2) & 1;  // entries of even or odd number, columns 32 half .. 32 half + 31 of them
        const int wq = warp & 3;   // TMEM quadrant of this warp
        const int row = wq * 32 + lane;  // row of the own tile = TMEM lane
        const uint32_t t_lane = (uint32_t)(wq * 32) << 16;
        bool ok = start_ok;
        unsigned s0 = 0, kk = 0;  // entries before the current item, items with entries before it
        // dQ pass: the own tiles go from shared memory to TMEM, where they are the A operands of every S and dP.  Warpgroup 2 g + h moves half h
        // of A1 (g = 0) or A2 (g = 1).
        auto own_to_tmem = [&](unsigned item) -> bool {
            if (kMode == 1) return true;
            if (!mbar_wait_warp(bar_a_full, item & 1, ctl, 242, item)) return false;
            if (item > 0 && !mbar_wait_warp(bar_at_free, (item - 1) & 1, ctl, 243, item)) return false;
            tc_fence_after();
            if (half < kHalves) {
                const unsigned char* src = smem + Ly::offA + wg * Ly::aTile + half * Ly::aHalf + row * 128;
                uint32_t ar[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 v = *reinterpret_cast<const uint4*>(src + ((c ^ (row & 7)) << 4));
                    ar[4 * c + 0] = v.x;
                    ar[4 * c + 1] = v.y;
                    ar[4 * c + 2] = v.z;
                    ar[4 * c + 3] = v.w;
                }
                tc_st32(tmem + (wg == 1 ? C::own2 : C::own1) + 32u * half + t_lane, ar);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            mbar_arrive_elect(bar_at_full);
            mbar_arrive_elect(bar_a_empty);
            return true;
        };
        // Two scores -> P, and 1 - tanh^2 with a cap.  c: -lse * log2(e), with a bias less the distance times the slope.
        auto probs = [&](float2 s, float2 c, bool large, float2& slack) {
            float2 x;
            if (kCap) x = __fadd2_rn(large ? capped_any(P.shape, s, slack) : capped_small(P.shape, s, slack), c);
            else x = __ffma2_rn(s, make_float2(P.shape.mul, P.shape.mul), c);
            return make_float2(ex2(x.x), ex2(x.y));
        };
        auto two = [](uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); };
        // dQ pass: what this thread's query sees, its -lse * log2(e) and -delta, the slope of its head; dK/dV pass: nothing yet
        struct Row {
            int4 see;
            float nl, nd, slope2;
        };
        auto row_of = [&](const Item& it) {
            Row r{make_int4(0, 0, 0, 0), 0.f, 0.f, 0.f};
            if (kMode == 0) {
                const int b = it.bh / P.heads, h = it.bh % P.heads, i = it.own * kM + row, u = i / kBlk;
                if (u < P.n_u) {
                    r.see = P.seen[((long long)b * P.n_u + u) * kSeenPitch + i % kBlk];
                    const float* st = P.stats + ((long long)it.bh * P.n_u + u) * kDenseStats + i % kBlk;
                    r.nl = st[0];
                    r.nd = st[kBlk];
                }
                if (kBias) r.slope2 = __ldg(P.slopes + h) * kLog2e;
            }
            return r;
        };
        auto entries = [&](const Item& it, const Row& me) {
            const unsigned n = it.n;
            const int key = it.own * kM + row;                 // dK/dV pass
            const int h0 = (it.bh % P.heads) * P.walk;
            int unit = (int)((s0 ^ wg) & 1), head = 0;         // of the entry, relative to the item's first
            float slope2 = me.slope2;
            auto wrap = [&]() {
                bool turned = false;
                while (unit >= it.span && head < P.walk) {
                    unit -= it.span;
                    ++head;
                    turned = true;
                }
                return turned;
            };
            if (kMode == 1) {
                wrap();
                if (kBias && head < P.walk) slope2 = __ldg(P.slopes + h0 + head) * kLog2e;
            }
            for (unsigned i = s0 + ((s0 ^ wg) & 1); i < s0 + n && ok; i += 2) {
                const unsigned r = i >> 1;
                const int slot = i % kSlots;
                // dK/dV pass: what came with the slot's tiles
                if (kMode == 1) ok = mbar_wait_warp(bar_full(slot), (i / kSlots) & 1, ctl, 234 + wg, i);
                if (ok) ok = mbar_wait_warp(bar_s_full(wg), r & 1, ctl, 230 + wg, i);
                if (!ok) break;
                tc_fence_after();
                uint32_t x[32], out[16];  // S, then dP
                float2 p[16];      // what dP - delta is multiplied by: P times 1 - tanh^2
                tc_ld32(tmem + C::s(wg) + 32u * half + t_lane, x);
                tc_wait_ld();
                if (kMode == 0) {
                    tc_fence_before();
                    mbar_arrive_elect(bar_s_free(wg));
                }
                const bool large = kCap && any_large(x, P.shape.s_fast);
                bool mixed;
                const float4* const st4 = reinterpret_cast<const float4*>(smem + Ly::offExtra + slot * Ly::extra) + 8 * half;  // dK/dV pass
                if constexpr (kMode == 0) {
                    const int first = it.first + kBlk * (int)(i - s0) + 32 * half;  // key of the warp's first column
                    mixed = mixed_keys(it, (int)(i - s0));
                    const float at = (float)(me.see.z - first);
                    const bool both_sides = kBias && __any_sync(0xffffffffu, at > 0.f && at < 31.f);
                    auto all = [&](bool lg, bool two_sides) {
                        BiasLine line;
                        if (kBias && !two_sides) line = bias_line(at, slope2, me.nl);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float2 c = make_float2(me.nl, me.nl), slack;
                            if (kBias) {
                                if (two_sides) c = __ffma2_rn(make_float2(fabsf(at - (float)(2 * k)), fabsf(at - (float)(2 * k + 1))), make_float2(-slope2, -slope2), c);
                                else c = bias_next(line, k);
                            }
                            p[k] = probs(two(x[2 * k], x[2 * k + 1]), c, lg, slack);
                            if (kCap) p[k] = __fmul2_rn(p[k], slack);
                        }
                    };
                    if (kCap && LCBSA_UNLIKELY(large)) all(true, true);
                    else if (kBias && (both_sides || (kCap && mixed))) all(false, true);  // mixed: the way of a tile that a hidden score makes large
                    else all(false, false);
                    if (mixed) {
                        const int lo = min(max(me.see.x - first, 0), 32), hi = min(max(me.see.y - first, 0), 32);  // a run of bits
                        const uint32_t sees = hi > lo ? (~0u >> (32 - (hi - lo))) << lo : 0u;
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            if (!((sees >> (2 * k)) & 1u)) p[k].x = 0.f;
                            if (!((sees >> (2 * k + 1)) & 1u)) p[k].y = 0.f;
                        }
                    }
                } else {
                    const int4* const see = seen_of_slot(slot);
                    mixed = mixed_queries(it, see[kBlk]);
                    // the queries of a whole entry belong to one document, so their places follow one another
                    const float at = kBias ? (float)(key - see[0].z - 32 * half) : 0.f;  // distance to column k: |at - k|
                    const bool both_sides = kBias && __any_sync(0xffffffffu, at > 0.f && at < 31.f);
                    auto all = [&](bool lg, bool mx, bool two_sides) {
                        BiasLine line;
                        if (kBias && !two_sides) line = bias_line(at, slope2, 0.f);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float4 l4 = st4[k >> 1];
                            float2 c = k & 1 ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y), slack;
                            int4 a = make_int4(0, 0, 0, 0), d = a;
                            if (mx) {
                                a = see[32 * half + 2 * k];
                                d = see[32 * half + 2 * k + 1];
                            }
                            if (kBias) {
                                float2 far = make_float2(fabsf(at - (float)(2 * k)), fabsf(at - (float)(2 * k + 1)));
                                if (mx) far = make_float2(fabsf((float)(a.z - key)), fabsf((float)(d.z - key)));
                                if (two_sides) c = __ffma2_rn(far, make_float2(-slope2, -slope2), c);
                                else c = __fadd2_rn(c, bias_next(line, k));
                            }
                            float2 w = probs(two(x[2 * k], x[2 * k + 1]), c, lg, slack);
                            p[k] = kCap ? __fmul2_rn(w, slack) : w;
                            if (mx) {
                                const float4 d4 = st4[16 + (k >> 1)];
                                if (__float_as_uint(k & 1 ? d4.z : d4.x) == kBadRow) w.x = p[k].x = __int_as_float(0x7fc00000);  // dO is not finite
                                if (__float_as_uint(k & 1 ? d4.w : d4.y) == kBadRow) w.y = p[k].y = __int_as_float(0x7fc00000);
                                if (key < a.x || key >= a.y) w.x = p[k].x = 0.f;  // last: the slack of a hidden score may be NaN
                                if (key < d.x || key >= d.y) w.y = p[k].y = 0.f;
                            }
                            out[k] = pack2(kBf16, w.x, w.y);
                        }
                    };
                    if (kCap && LCBSA_UNLIKELY(large)) all(true, true, true);
                    else if (mixed) all(false, true, true);
                    else if (kBias && both_sides) all(false, false, true);
                    else all(false, false, false);
                    unit += 2;
                    if (wrap() && kBias && head < P.walk) slope2 = __ldg(P.slopes + h0 + head) * kLog2e;
                    tc_st16(tmem + C::s(wg) + 32u * half + t_lane, out);  // the columns that this thread read
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive_elect(bar_p_full(wg));
                }
                ok = mbar_wait_warp(bar_d_full(wg), r & 1, ctl, 236 + wg, i);
                if (!ok) break;
                tc_fence_after();
                tc_ld32(tmem + C::dp(wg) + 32u * half + t_lane, x);
                tc_wait_ld();
                auto grads = [&](bool mx) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 nd = make_float2(me.nd, me.nd);
                        if (kMode == 1) {
                            const float4 d4 = st4[16 + (k >> 1)];
                            nd = k & 1 ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);
                        }
                        float2 ds = __fmul2_rn(p[k], __fadd2_rn(two(x[2 * k], x[2 * k + 1]), nd));
                        if (mx) {  // hidden, whatever dP is
                            if (p[k].x == 0.f) ds.x = 0.f;
                            if (p[k].y == 0.f) ds.y = 0.f;
                        }
                        out[k] = pack2(kBf16, ds.x, ds.y);
                    }
                };
                if (mixed) grads(true);
                else grads(false);
                tc_st16(tmem + C::dp(wg) + 32u * half + t_lane, out);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive_elect(bar_x_full(wg));
            }
            s0 += n;
        };
        // The accumulated gradients of an item's rows: TMEM -> registers, which frees the accumulators -> global memory, 32 columns at a
        // time.  dQ pass: warpgroup 2 g + h stores columns 32 (2 g + h) .. of dQ; dK/dV pass: half h of dK (g = 0) or dV (g = 1).
        auto store_item = [&](const Item& it, unsigned item) -> bool {
            const int b = it.bh / P.heads, h = it.bh % P.heads, i = it.own * kM + row;
            const bool second = kMode == 1 && wg == 1;
            unsigned char* base = static_cast<unsigned char*>(second ? P.out2 : P.out1);
            const long long sb = second ? P.o2_sb : P.o1_sb, sh = second ? P.o2_sh : P.o1_sh, ss = second ? P.o2_ss : P.o1_ss;
            unsigned char* row_ptr = base + ((long long)b * sb + (long long)h * sh + (long long)i * ss) * 2;
            const uint32_t t_acc = tmem + (second ? C::acc2 : C::acc1) + t_lane;
            if (it.n > 0) {
                if (!mbar_wait_warp(bar_acc_done, item & 1, ctl, 240 + kMode, item)) return false;
            }
            tc_fence_after();
            constexpr int kParts = kMode == 1 ? kHalves : 1;
#pragma unroll 1
            for (int part = 0; part < kParts; ++part) {
                const int col = kMode == 1 ? 32 * (half * kHalves + part) : 32 * (2 * wg + half);
                uint32_t acc[32];
                if (it.n > 0) {
                    tc_ld32(t_acc + (col < D ? col : 0), acc);
                    tc_wait_ld();
                    if (part == kParts - 1) {
                        tc_fence_before();
                        mbar_arrive_elect(bar_acc_free);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[j] = 0u;  // nobody sees these rows, or they see nothing
                }
                if (!second) {  // the scale that dS is without
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[j] = __float_as_uint(__uint_as_float(acc[j]) * P.scale);
                }
                if (i >= P.rows || col >= D) continue;
                if (kMode == 1 && P.splits > 1) {
                    float4* dst = reinterpret_cast<float4*>(P.part + (((long long)(second ? P.B * P.heads : 0) + it.bh) * P.rows + i) * D + col);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        dst[j] = make_float4(__uint_as_float(acc[4 * j]), __uint_as_float(acc[4 * j + 1]), __uint_as_float(acc[4 * j + 2]), __uint_as_float(acc[4 * j + 3]));
                } else {
                    store_row32<kBf16>(row_ptr, col, acc);
                }
            }
            return true;
        };
        // Item by item; the own tiles and row values of the next one are fetched before the gradients of this one are stored.
        unsigned k = 0;
        Item cur{-1, 0, 0, 0, 0, 0, 0};
        if (ok) cur = take_item(k++);
        bool moved = false;
        Row me = row_of(Item{0, P.n_own, 0, 0, 0, 0, 0}), me_n = me;
        while (ok && cur.bh >= 0) {
            if (cur.n > 0 && !moved) {
                me = row_of(cur);
                ok = own_to_tmem(kk);
                if (!ok) break;
            }
            if (cur.n > 0) {
                entries(cur, me);
                if (!ok) break;
            }
            const Item nx = take_item(k++);
            moved = cur.n > 0 && nx.bh >= 0 && nx.n > 0;
            if (moved) {
                me_n = row_of(nx);
                ok = own_to_tmem(kk + 1);
                if (!ok) break;
            }
            ok = store_item(cur, kk);
            if (cur.n > 0) ++kk;
            if (moved) me = me_n;
            cur = nx;
        }
    }

    // ---- teardown
    tc_fence_before();
    __syncthreads();
    if (tid == 0) ctl_report(ctl);
    if (warp == kMathWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// The split sums of dK and dV, added in order: a thread takes four values of a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) dense_join_kernel(const __grid_constant__ DenseArgs a, const float* part, int splits) {
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x, total = (long long)a.B * a.Hk * a.Sk * (D / 4);
    if (at >= total) return;
    const int c = (int)(at % (D / 4));
    const long long r = at / (D / 4), bh = r / a.Sk;
    const int i = (int)(r % a.Sk), b = (int)(bh / a.Hk), h = (int)(bh % a.Hk);
    const long long all = (long long)a.B * a.Hk * splits * a.Sk * D;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int sp = 0; sp < splits; ++sp) {
            const float4 v = *reinterpret_cast<const float4*>(part + t * all + ((bh * splits + sp) * a.Sk + i) * D + 4 * c);
            s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
        }
        const View& o = t ? a.dv : a.dk;
        uint2 w;
        w.x = pack2(DType<T>::code == LCBSA_BF16, s.x, s.y);
        w.y = pack2(DType<T>::code == LCBSA_BF16, s.z, s.w);
        *reinterpret_cast<uint2*>(static_cast<T*>(const_cast<void*>(o.data)) + b * o.sb + h * o.sh + i * o.ss + 4 * c) = w;
    }
}

// Items of the dK/dV pass are few where many query heads share a key head, and as long as all of them together: where there are less than
// four for an SM the heads are split: their fp32 sums go through the workspace and are joined in order.  Pass and join, 16 query heads on 4 key
// heads, nine documents in 5000 tokens: 222 us in one part, 131 + 10 in two, 109 + 16 in four; 16 heads on 8, 8192 tokens: 544 in one, 455 + 37 in two.
int dkdv_splits(const DenseArgs& a) {
    const long long items = (long long)a.B * a.Hk * ((a.Sk + kM - 1) / kM);
    int s = 1;
    while (s < a.group && items * s < 148 * 4) {
        do ++s; while (a.group % s != 0);
    }
    return s;
}

template <bool kBf16, int D, int kMode, bool kCap, bool kBias>
cudaError_t pass_launch(const BwdParams& P, cudaStream_t st) {
    static thread_local unsigned long long raised = 0;  // devices (below 64) whose shared-memory limit this thread has raised for this kernel
    int dev = 0, sm_count = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !((raised >> dev) & 1)) {
        e = cudaFuncSetAttribute(dense_bwd_tc_kernel<kBf16, D, kMode, kCap, kBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::smem);
        if (e != cudaSuccess) return e;
        if (dev <= 63) raised |= 1ull << dev;
    }
    const int usable = sm_count - attn_sm_reserve() > 0 ? sm_count - attn_sm_reserve() : 1;
    dense_bwd_tc_kernel<kBf16, D, kMode, kCap, kBias><<<P.n_items < usable ? P.n_items : usable, kThreads, Lay<D>::smem, st>>>(P);
    return cudaGetLastError();
}

template <bool kBf16, int D, int kMode>
cudaError_t pass_shape(const BwdParams& P, bool cap, cudaStream_t st) {
    if (cap) return P.slopes ? pass_launch<kBf16, D, kMode, true, true>(P, st) : pass_launch<kBf16, D, kMode, true, false>(P, st);
    return P.slopes ? pass_launch<kBf16, D, kMode, false, true>(P, st) : pass_launch<kBf16, D, kMode, false, false>(P, st);
}

template <bool kBf16, int D>
cudaError_t passes(const DenseArgs& a, cudaStream_t st, const char** why) {
    cudaError_t e = launch_dense_plan(a, st);
    if (e != cudaSuccess) return e;
    BwdParams P{};
    P.seen = a.seen; P.hulls = a.hulls; P.stats = a.stats; P.slopes = a.slopes; P.status = a.status;
    P.B = a.B; P.Hq = a.Hq; P.Hk = a.Hk; P.group = a.group; P.n_u = dense_units(a.Sq); P.n_k = dense_units(a.Sk);
    P.scale = a.scale;
    P.shape = score_shape(a.scale, a.cap);
    auto map = [&](CUtensorMap* tm, const View& v, int H, int S, int box, int* fold) {
        if (S == 0 || dense_rows_map(tm, a.dtype, v, a.B, H, S, D, box, fold)) return true;
        *why = "cuTensorMapEncodeTiled rejected a tensor";
        return false;
    };
    const bool cap = a.cap > 0.f;
    if (a.Sq > 0) {  // a call without keys still writes dq
        if (!map(&P.tm_a1, a.q, a.Hq, a.Sq, kM, &P.fold_a1) || !map(&P.tm_a2, a.dout, a.Hq, a.Sq, kM, &P.fold_a2) ||
            !map(&P.tm_b1, a.k, a.Hk, a.Sk, kBlk, &P.fold_b1) || !map(&P.tm_b2, a.v, a.Hk, a.Sk, kBlk, &P.fold_b2))
            return cudaErrorInvalidValue;
        P.out1 = const_cast<void*>(a.dq.data);
        P.o1_sb = a.dq.sb; P.o1_sh = a.dq.sh; P.o1_ss = a.dq.ss;
        P.heads = a.Hq; P.n_own = (a.Sq + kM - 1) / kM; P.rows = a.Sq;
        P.n_items = a.B * a.Hq * P.n_own;
        P.wave = dense_wave(a.B * a.Hq, 4.0 * a.Sk * D / a.group);
        P.next_item = a.next_item;
        e = pass_shape<kBf16, D, 0>(P, cap, st);
        if (e != cudaSuccess) return e;
    }
    if (a.Sk > 0) {
        if (!map(&P.tm_a1, a.k, a.Hk, a.Sk, kM, &P.fold_a1) || !map(&P.tm_a2, a.v, a.Hk, a.Sk, kM, &P.fold_a2) ||
            !map(&P.tm_b1, a.q, a.Hq, a.Sq, kBlk, &P.fold_b1) || !map(&P.tm_b2, a.dout, a.Hq, a.Sq, kBlk, &P.fold_b2))
            return cudaErrorInvalidValue;
        P.out1 = const_cast<void*>(a.dk.data);
        P.o1_sb = a.dk.sb; P.o1_sh = a.dk.sh; P.o1_ss = a.dk.ss;
        P.out2 = const_cast<void*>(a.dv.data);
        P.o2_sb = a.dv.sb; P.o2_sh = a.dv.sh; P.o2_ss = a.dv.ss;
        P.splits = dkdv_splits(a);
        P.walk = a.group / P.splits;
        P.part = a.part;
        P.heads = a.Hk * P.splits; P.n_own = (a.Sk + kM - 1) / kM; P.rows = a.Sk;
        P.n_items = a.B * P.heads * P.n_own;
        P.wave = dense_wave(a.B * P.heads, 4.0 * a.Sq * D * P.walk);
        P.next_item = a.next_item + 1;
        e = pass_shape<kBf16, D, 1>(P, cap, st);
        if (e == cudaSuccess && P.splits > 1) {
            using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
            const long long ctas = ((long long)a.B * a.Hk * a.Sk * (D / 4) + 255) / 256;
            if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
            dense_join_kernel<T, D><<<(unsigned)ctas, 256, 0, st>>>(a, a.part, P.splits);
            e = cudaGetLastError();
        }
    }
    return e;
}

}  // namespace

// Operands are read through tensor maps: rows a stride apart.
bool dense_bwd_supported(const DenseArgs& a, const char** why) {
    const View* vs[4] = {&a.q, &a.dout, &a.k, &a.v};
    const int len[4] = {a.Sq, a.Sq, a.Sk, a.Sk};
    for (int i = 0; i < 4; ++i) {
        if (len[i] > 1 && vs[i]->ss == 0) { *why = "tokens without a stride"; return false; }
        if (vs[i]->ss * 2 >= (1ll << 40) || vs[i]->sh * 2 >= (1ll << 40) || vs[i]->sb * 2 >= (1ll << 40)) { *why = "stride too large for a tensor map"; return false; }
    }
    if ((long long)a.B * a.Hq * ((a.Sq + kM - 1) / kM) > 0x7fff0000ll || (long long)a.B * a.Hk * ((a.Sk + kM - 1) / kM) > 0x7fff0000ll) {
        *why = "more tiles than a launch takes";
        return false;
    }
    return true;
}

size_t dense_bwd_workspace_bytes(const DenseArgs& a) {
    const int splits = dkdv_splits(a);
    return dense_plan_bytes(a, true) + (size_t)a.B * a.Hq * dense_units(a.Sq) * kStatsBytes +
           (splits > 1 ? 2 * (size_t)a.B * a.Hk * splits * a.Sk * a.D * sizeof(float) : 0);
}

cudaError_t launch_dense_bwd(DenseArgs a, void* workspace, cudaStream_t st, const char** why) {
    if (a.B == 0 || a.Hq == 0) return cudaSuccess;
    dense_plan_carve(a, workspace, true);
    a.stats = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + dense_plan_bytes(a, true));
    a.part = a.stats + (size_t)a.B * a.Hq * dense_units(a.Sq) * kDenseStats;
    const cudaError_t e = a.dtype == LCBSA_BF16 ? (a.D == 128 ? passes<true, 128>(a, st, why) : passes<true, 64>(a, st, why))
                                                : (a.D == 128 ? passes<false, 128>(a, st, why) : passes<false, 64>(a, st, why));
    if (e == cudaErrorInvalidConfiguration) *why = "more CTAs than a launch takes";
    return e;
}

}  // namespace lcbsa
