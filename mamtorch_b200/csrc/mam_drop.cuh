// The counter-based generator of the dropout masks: a mask is a function of (seed, element index), formed again wherever
// it is needed -- forward, backward, weight drop -- and never stored.
#pragma once
#include <cuda_runtime.h>

#include "mam_vec.cuh"

namespace mamb200 {

// The splitmix64 generator: a mixing function on seed + counter * golden ratio.
constexpr unsigned long long MAM_DROP_STEP = 0x9E3779B97F4A7C15ull;
__device__ __forceinline__ unsigned long long mam_drop_finish(unsigned long long z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
__device__ __forceinline__ unsigned long long mam_drop_mix(unsigned long long seed, unsigned long long counter) {
    return mam_drop_finish(seed + counter * MAM_DROP_STEP);
}

// The keep / drop decision of element `idx` in the MAM forward's epilogue and in mam_drop_f32: one mix an element, its
// high 32 bits.  Dropped with probability threshold / 2^32.
__device__ __forceinline__ bool mam_drop_keeps(unsigned long long seed, unsigned long long idx, unsigned threshold) {
    return (unsigned)(mam_drop_mix(seed, idx) >> 32) >= threshold;
}

// Dropout of the memory-bound operators (layer norm with residual, GELU, residual addition), where the mix would take
// longer than the bytes: one mix gives two elements, its low 32 bits the even one's draw, its high 32 bits the odd
// one's.  The elements of a tensor are counted in its contiguous order.
struct DropArgs {
    unsigned long long seed;     // added to *seed_at where that is given
    const long long* seed_at;    // device memory, read by the kernel: a captured graph takes a new seed from it
    unsigned threshold;          // rate * 2^32
    float scale;                 // 1 / (1 - rate)
    int on;                      // 0: nothing is dropped
    __device__ __forceinline__ unsigned long long seed_now() const {
        return seed + (seed_at ? (unsigned long long)*seed_at : 0ull);
    }
};

// where the mixes of the elements from `idx` on begin: the one of pair j is of start + j * MAM_DROP_STEP
__device__ __forceinline__ unsigned long long mam_drop_start(unsigned long long seed, long long idx) {
    return seed + ((unsigned long long)idx >> 1) * MAM_DROP_STEP;
}
// x = kept ? x * scale : 0 for N pairs of elements from `start` on; `odd`: the first of them is the odd element of its
// pair.  A select, not a product: what is dropped leaves nothing behind, an infinity or NaN neither.
//
// In 16-bit tensors the mixes are what bounds it (shifts, xors, compares and selects share a pipe of half rate).  The last
// step of the mix only flips the lowest bit of the high half, where its highest bit is set, and is left out there: up to
// a threshold of 2^31 such a half is kept either way, and a higher threshold is even (the rate, a float from 1/2 on, is
// a multiple of 2^-24), so that it does not tell the two apart.
template <int N>
__device__ __forceinline__ void mam_drop_pairs(float2 (&x)[N], unsigned long long start, bool odd, unsigned threshold,
                                               float scale) {
    const float2 sc = make_float2(scale, scale);
    const auto draw = [&](int j, unsigned& lo, unsigned& hi) {
        // the 64-bit steps of mam_drop_finish in 32-bit ones
        const unsigned long long z = start + (unsigned long long)j * MAM_DROP_STEP;
        unsigned l = (unsigned)z, h = (unsigned)(z >> 32);
        const auto times = [&](unsigned cl, unsigned ch) {
            const unsigned long long w = (unsigned long long)l * cl;
            h = l * ch + (h * cl + (unsigned)(w >> 32));
            l = (unsigned)w;
        };
        const auto fold = [&](int k) {
            l ^= __funnelshift_r(l, h, k);
            h ^= h >> k;
        };
        fold(30);
        times(0x1CE4E5B9u, 0xBF58476Du);
        fold(27);
        times(0x133111EBu, 0x94D049BBu);
        lo = l ^ __funnelshift_r(l, h, 31);
        hi = h;
    };
    if (!odd) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            unsigned lo, hi;
            draw(j, lo, hi);
            const float2 y = mul2(x[j], sc);
            x[j] = make_float2(lo >= threshold ? y.x : 0.f, hi >= threshold ? y.y : 0.f);
        }
    } else {
        unsigned lo, high;
        draw(0, lo, high);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            unsigned hi;
            draw(j + 1, lo, hi);
            const float2 y = mul2(x[j], sc);
            x[j] = make_float2(high >= threshold ? y.x : 0.f, lo >= threshold ? y.y : 0.f);
            high = hi;
        }
    }
}

}  // namespace mamb200
