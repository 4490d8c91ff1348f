// Shared by the kernels that run on warp-level MMA (attn_mma.cu: the generic forward; attn_bwd.cu: the backward):
// cp.async / ldmatrix / mma.sync wrappers, the gather of a 3-D block's slots into a swizzled shared-memory tile.
#pragma once
#include "common.cuh"

namespace lcbsa {
namespace mm {

struct SlotEntry {
    int off;     // token offset of the slot relative to the block's first token
    int packed;  // lt | lh << 10 | lw << 20
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool pred) {
    const int n = pred ? 16 : 0;  // src-size 0 -> the 16 bytes are zero-filled
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(__half, float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ bool slot_present(const Geom& g, int packed, int t0, int h0, int w0) {
    return (t0 + (packed & 1023) < g.T) && (h0 + ((packed >> 10) & 1023) < g.H) && (w0 + (packed >> 20) < g.W);
}

// Gather ROWS block slots (starting at slot0) of block `blk` into a swizzled [ROWS][D] tile.
template <typename T, int D, int ROWS, int NTHREADS>
__device__ __forceinline__ void load_tile(unsigned char* tile, const T* head_base, long long ss, const Geom& g,
                                          const SlotEntry* tab, int blk, int slot0, int tid) {
    constexpr int CPR = D * 2 / 16;  // 16-byte chunks per row
    int bt, bh, bw;
    // a block number outside the grid (a caller's list may hold anything) is never turned into an address:
    // the whole tile is zero-filled and the caller of load_tile masks the block out of the softmax
    const bool blk_ok = (unsigned)blk < (unsigned)g.nblk;
    block_coords(g, blk_ok ? blk : 0, bt, bh, bw);
    const int t0 = bt * g.ct, h0 = bh * g.ch, w0 = bw * g.cw;
    const long long origin = ((long long)t0 * g.H + h0) * g.W + w0;
    const uint32_t sbase = smem_u32(tile);
#pragma unroll
    for (int v = tid; v < ROWS * CPR; v += NTHREADS) {
        const int row = v / CPR, c = v % CPR;
        const SlotEntry e = tab[slot0 + row];
        const bool present = blk_ok && (!g.ragged || slot_present(g, e.packed, t0, h0, w0));
        const T* src = head_base + (present ? (origin + e.off) * ss : 0) + c * 8;
        cp_async16(sbase + row * (D * 2) + ((c ^ (row & 7)) << 4), src, present);
    }
}

// ------------------------------------------------------------------------------------------ products of 64-row tiles (the backward passes)

// 16 rows x 64 columns (fp32 accumulators, 8 n-tiles) = A[16 x D] * B[64 x D]^T with A already in registers, twice at once (S and dP of
// the same tile pair): two independent accumulation chains in one instruction
// stream, which is what hides the ldmatrix -> mma latency with only two warps per scheduler.
template <typename T, int D>
__device__ __forceinline__ void mma_abt2(float (&acc0)[8][4], float (&acc1)[8][4], const uint32_t (&a0)[D / 16][4],
                                         const uint32_t (&a1)[D / 16][4], uint32_t b0_tile, uint32_t b1_tile, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        acc0[i][0] = acc0[i][1] = acc0[i][2] = acc0[i][3] = 0.f;
        acc1[i][0] = acc1[i][1] = acc1[i][2] = acc1[i][3] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int np = 0; np < 4; ++np) {
            const int mid = lane >> 3;
            const int row = np * 16 + (lane & 7) + (mid >> 1) * 8;
            const int c = 2 * ks + (mid & 1);
            const uint32_t off = row * (D * 2) + ((c ^ (row & 7)) << 4);
            uint32_t bf0[4], bf1[4];
            ldsm_x4(bf0, b0_tile + off);
            ldsm_x4(bf1, b1_tile + off);
            mma16816<T>(acc0[2 * np], a0[ks], bf0[0], bf0[1]);
            mma16816<T>(acc1[2 * np], a1[ks], bf1[0], bf1[1]);
            mma16816<T>(acc0[2 * np + 1], a0[ks], bf0[2], bf0[3]);
            mma16816<T>(acc1[2 * np + 1], a1[ks], bf1[2], bf1[3]);
        }
    }
}

// The same with the A operands read from shared tiles step by step (this warp's 16 rows of a0_tile and a1_tile)
template <typename T, int D>
__device__ __forceinline__ void mma_abt2_sa(float (&acc0)[8][4], float (&acc1)[8][4], uint32_t a0_tile, uint32_t a1_tile, uint32_t b0_tile,
                                            uint32_t b1_tile, int warp, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        acc0[i][0] = acc0[i][1] = acc0[i][2] = acc0[i][3] = 0.f;
        acc1[i][0] = acc1[i][1] = acc1[i][2] = acc1[i][3] = 0.f;
    }
    const int arow = warp * 16 + (lane & 15);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a0[4], a1[4];
        {
            const int c = 2 * ks + (lane >> 4);
            const uint32_t off = arow * (D * 2) + ((c ^ (arow & 7)) << 4);
            ldsm_x4(a0, a0_tile + off);
            ldsm_x4(a1, a1_tile + off);
        }
#pragma unroll
        for (int np = 0; np < 4; ++np) {
            const int mid = lane >> 3;
            const int row = np * 16 + (lane & 7) + (mid >> 1) * 8;
            const int c = 2 * ks + (mid & 1);
            const uint32_t off = row * (D * 2) + ((c ^ (row & 7)) << 4);
            uint32_t bf0[4], bf1[4];
            ldsm_x4(bf0, b0_tile + off);
            ldsm_x4(bf1, b1_tile + off);
            mma16816<T>(acc0[2 * np], a0, bf0[0], bf0[1]);
            mma16816<T>(acc1[2 * np], a1, bf1[0], bf1[1]);
            mma16816<T>(acc0[2 * np + 1], a0, bf0[2], bf0[3]);
            mma16816<T>(acc1[2 * np + 1], a1, bf1[2], bf1[3]);
        }
    }
}

// A fragments (16 rows of this warp, all of D) of a swizzled [64][D] tile
template <int D>
__device__ __forceinline__ void load_a_frags(uint32_t (&af)[D / 16][4], uint32_t tile, int warp, int lane) {
    const int row = warp * 16 + (lane & 15);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const int c = 2 * ks + (lane >> 4);
        ldsm_x4(af[ks], tile + row * (D * 2) + ((c ^ (row & 7)) << 4));
    }
}

// out[16 x D] += X[16 x 64] * B[64 x D], X given as fp32 accumulators of the layout mma_abt2 produces (rounded to T here)
template <typename T, int D>
__device__ __forceinline__ void mma_xb(float (&out)[D / 8][4], const float (&x)[8][4], uint32_t b_tile, int lane) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        uint32_t pa[4];
        pa[0] = pack2(T(), x[2 * kk][0], x[2 * kk][1]);
        pa[1] = pack2(T(), x[2 * kk][2], x[2 * kk][3]);
        pa[2] = pack2(T(), x[2 * kk + 1][0], x[2 * kk + 1][1]);
        pa[3] = pack2(T(), x[2 * kk + 1][2], x[2 * kk + 1][3]);
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
            const int mid = lane >> 3;
            const int row = kk * 16 + (lane & 7) + (mid & 1) * 8;
            const int c = 2 * dp + (mid >> 1);
            uint32_t bf[4];
            ldsm_x4_t(bf, b_tile + row * (D * 2) + ((c ^ (row & 7)) << 4));
            mma16816<T>(out[2 * dp], pa, bf[0], bf[1]);
            mma16816<T>(out[2 * dp + 1], pa, bf[2], bf[3]);
        }
    }
}

// Two of those at once: out0 += X0 * B0 and out1 += X1 * B1 (dV and dK of one tile pair)
template <typename T, int D>
__device__ __forceinline__ void mma_xb2(float (&out0)[D / 8][4], const float (&x0)[8][4], uint32_t b0_tile, float (&out1)[D / 8][4],
                                        const float (&x1)[8][4], uint32_t b1_tile, int lane) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        uint32_t pa0[4], pa1[4];
        pa0[0] = pack2(T(), x0[2 * kk][0], x0[2 * kk][1]);
        pa0[1] = pack2(T(), x0[2 * kk][2], x0[2 * kk][3]);
        pa0[2] = pack2(T(), x0[2 * kk + 1][0], x0[2 * kk + 1][1]);
        pa0[3] = pack2(T(), x0[2 * kk + 1][2], x0[2 * kk + 1][3]);
        pa1[0] = pack2(T(), x1[2 * kk][0], x1[2 * kk][1]);
        pa1[1] = pack2(T(), x1[2 * kk][2], x1[2 * kk][3]);
        pa1[2] = pack2(T(), x1[2 * kk + 1][0], x1[2 * kk + 1][1]);
        pa1[3] = pack2(T(), x1[2 * kk + 1][2], x1[2 * kk + 1][3]);
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
            const int mid = lane >> 3;
            const int row = kk * 16 + (lane & 7) + (mid & 1) * 8;
            const int c = 2 * dp + (mid >> 1);
            const uint32_t off = row * (D * 2) + ((c ^ (row & 7)) << 4);
            uint32_t bf0[4], bf1[4];
            ldsm_x4_t(bf0, b0_tile + off);
            ldsm_x4_t(bf1, b1_tile + off);
            mma16816<T>(out0[2 * dp], pa0, bf0[0], bf0[1]);
            mma16816<T>(out1[2 * dp], pa1, bf1[0], bf1[1]);
            mma16816<T>(out0[2 * dp + 1], pa0, bf0[2], bf0[3]);
            mma16816<T>(out1[2 * dp + 1], pa1, bf1[2], bf1[3]);
        }
    }
}

// fp32 accumulators of this warp's 16 rows (all of D) -> a swizzled [64][D] tile in T
template <typename T, int D>
__device__ __forceinline__ void stage_rows(unsigned char* tile, const float (&o)[D / 8][4], int warp, int lane) {
    const int r0 = warp * 16 + (lane >> 2), r1 = r0 + 8;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
        const int col = i * 8 + 2 * (lane & 3);
        const int c = col >> 3, within = (col & 7) * 2;
        *reinterpret_cast<uint32_t*>(tile + r0 * (D * 2) + ((c ^ (r0 & 7)) << 4) + within) = pack2(T(), o[i][0], o[i][1]);
        *reinterpret_cast<uint32_t*>(tile + r1 * (D * 2) + ((c ^ (r1 & 7)) << 4) + within) = pack2(T(), o[i][2], o[i][3]);
    }
}

}  // namespace mm
}  // namespace lcbsa
