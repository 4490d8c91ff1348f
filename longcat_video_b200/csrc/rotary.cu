// Rotary positions along one axis: pair p of a head turns by position * frequency[p].
//
//   (a, b) -> (a cos - b sin, b cos + a sin) * factor,  angle = position * frequency;  the gradient turns the other way.
//
// Pairs lie next to each other (2p, 2p + 1) or half of the turning part apart (p, p + pairs); the rest of the head is copied.  Reads every
// element once and writes it once: bound by HBM (2 bytes in, 2 bytes out per element).
//
// The angle is kept as a fraction of a turn in 64-bit fixed point: frequency = F / 2^64 turns per position, and position * F modulo 2^64
// is the fraction, with no rounding but F's own, where position * frequency in fp32 is off by 0.03 radians at position 10^6.
// Its upper 32 bits, rounded to 24, go to sincospif: off by 2^-24 of half a turn at most.  F is off by up to 2^-65 turns, which makes 2^-25 of a turn,
// as much as that, at position 2^40 and doubles with every power of two beyond.  No table: the frequencies are an argument
// of the launch, so a call reads nothing but its rows and its positions.
//
// A thread owns one 16-byte vector of a token (half layout: the two vectors that its eight pairs lie in) and walks over a group
// of heads, four at a time, so the angles are worked out once for all of them.
// A call takes q and k together: one launch.  q and k of 2 x 32 heads of 8192 tokens, head_dim 128: 80 us, 74 % of the DRAM rate under the
// profiler; a prompt of 5003 tokens 9.2 us with four heads' vectors in flight, 11.8 with one head's.
#include "common.cuh"

namespace lcbsa {

namespace {

constexpr int kRotThreads = 256;
constexpr int kBatch = 4;  // heads whose vectors a thread has in flight

template <typename T> struct Two;
template <> struct Two<__nv_bfloat16> {
    __device__ static __forceinline__ float2 get(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
    __device__ static __forceinline__ uint32_t put(float x, float y) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
};
template <> struct Two<__half> {
    __device__ static __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    __device__ static __forceinline__ uint32_t put(float x, float y) {
        const __half2 t = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
};

// The eight values of a vector against their partners: interleaved, pairs inside `a` (b unused); else a[i] with b[i].
template <typename T, bool kInter>
__device__ __forceinline__ void turn(uint4& a, uint4& b, const float* cs, const float* sn) {
    uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
    uint32_t* pb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (kInter) {
            const float2 v = Two<T>::get(pa[i]);
            pa[i] = Two<T>::put(fmaf(v.x, cs[i], -v.y * sn[i]), fmaf(v.y, cs[i], v.x * sn[i]));
        } else {
            const float2 x = Two<T>::get(pa[i]), y = Two<T>::get(pb[i]);
            pa[i] = Two<T>::put(fmaf(x.x, cs[2 * i], -y.x * sn[2 * i]), fmaf(x.y, cs[2 * i + 1], -y.y * sn[2 * i + 1]));
            pb[i] = Two<T>::put(fmaf(y.x, cs[2 * i], x.x * sn[2 * i]), fmaf(y.y, cs[2 * i + 1], x.y * sn[2 * i + 1]));
        }
    }
}

template <typename T, bool kInter>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryArgs P) {
    constexpr int kAngles = kInter ? 4 : 8;
    const long long item = (long long)blockIdx.x * kRotThreads + threadIdx.x;
    if (item >= P.items) return;
    const int slot = (int)(item % P.slots);
    const long long tok = item / P.slots;
    const int s = (int)(tok % P.S), b = (int)(tok / P.S);
    int g = blockIdx.y, j = 0;
    while (g >= P.job[j].groups) g -= P.job[j++].groups;
    const RotaryJob& J = P.job[j];
    const int h0 = g * P.hpc, h1 = min(h0 + P.hpc, J.H);
    // where the thread's vectors lie: the turning slots first, then those that are copied
    const int turning = kInter ? P.pairs / 4 : P.pairs / 8;
    const bool turns = slot < turning;
    const int at = turns ? slot * 8 : 2 * P.pairs + (slot - turning) * 8;
    const T* src = static_cast<const T*>(J.x.data) + b * J.x.sb + s * J.x.ss + h0 * J.x.sh + at;
    T* dst = static_cast<T*>(const_cast<void*>(J.out.data)) + b * J.out.sb + s * J.out.ss + h0 * J.out.sh + at;
    const bool both = !kInter && turns;
    // kBatch heads at a time, all of their vectors in flight together; those of the first batch under the angles
    uint4 v[kBatch], w[kBatch];
    auto fetch = [&](int h) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (h + i < h1) {
                v[i] = *reinterpret_cast<const uint4*>(src);
                if (both) w[i] = *reinterpret_cast<const uint4*>(src + P.pairs);
                src += J.x.sh;
            }
        }
    };
    fetch(h0);
    float cs[kAngles], sn[kAngles];
    if (turns) {
        long long pos = P.offset + s;
        if (P.pos != nullptr) {
            const long long e = b * P.pos_sb + s * P.pos_ss;
            pos = P.pos64 ? __ldg(static_cast<const long long*>(P.pos) + e) : (long long)__ldg(static_cast<const int*>(P.pos) + e);
        }
        const int p0 = slot * kAngles;
#pragma unroll
        for (int i = 0; i < kAngles; ++i) {
            const unsigned long long phase = (unsigned long long)pos * P.turns[p0 + i];
            sincospif((float)(int)(phase >> 32) * 4.656612873077393e-10f, &sn[i], &cs[i]);  // 2^-31: half turns
            cs[i] *= P.factor;
            sn[i] *= P.inverse ? -P.factor : P.factor;
        }
    }
#pragma unroll 1
    for (int h = h0; h < h1; h += kBatch) {
        if (h > h0) fetch(h);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (h + i < h1) {
                if (turns) turn<T, kInter>(v[i], w[i], cs, sn);
                *reinterpret_cast<uint4*>(dst) = v[i];
                if (both) *reinterpret_cast<uint4*>(dst + P.pairs) = w[i];
                dst += J.out.sh;
            }
        }
    }
}

}  // namespace

cudaError_t launch_rotary(int dtype, RotaryArgs& P, int B, int D, cudaStream_t st, const char** why) {
    P.slots = P.interleaved ? D / 8 : (D - 2 * P.pairs) / 8 + P.pairs / 8;
    P.items = (long long)B * P.S * P.slots;
    int heads = 0;
    for (int i = 0; i < P.n; ++i) heads += P.job[i].H;
    if (P.items == 0 || heads == 0) return cudaSuccess;
    const long long ctas = (P.items + kRotThreads - 1) / kRotThreads;
    if (ctas > 0x7fffffffll) {
        *why = "more CTAs than a launch takes";
        return cudaErrorInvalidConfiguration;
    }
    // A thread takes up to 16 heads, over which its angles are spread; small calls take fewer, since its heads are a chain of loads.
    P.hpc = 16;
    auto groups = [&] {
        int n = 0;
        for (int i = 0; i < P.n; ++i) n += P.job[i].groups = (P.job[i].H + P.hpc - 1) / P.hpc;
        return n;
    };
    while (P.hpc > 1 && ctas * groups() < 148 * 4) P.hpc /= 2;
    const int n = groups();
    if (n > 65535) {
        *why = "more heads than a launch takes";
        return cudaErrorInvalidConfiguration;
    }
    const dim3 grid((unsigned)ctas, (unsigned)n);
    if (dtype == LCBSA_BF16) {
        if (P.interleaved) rotary_kernel<__nv_bfloat16, true><<<grid, kRotThreads, 0, st>>>(P);
        else rotary_kernel<__nv_bfloat16, false><<<grid, kRotThreads, 0, st>>>(P);
    } else {
        if (P.interleaved) rotary_kernel<__half, true><<<grid, kRotThreads, 0, st>>>(P);
        else rotary_kernel<__half, false><<<grid, kRotThreads, 0, st>>>(P);
    }
    return cudaGetLastError();
}

}  // namespace lcbsa
