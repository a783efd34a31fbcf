// The counter-based generator of the dropout masks: a mask is a function of (seed, element index), formed again wherever
// it is needed -- forward, backward, weight drop -- and never stored.
#pragma once
#include <cuda_runtime.h>

namespace mamb200 {

// the splitmix64 mixing function on seed + counter * golden ratio
__device__ __forceinline__ unsigned long long mam_drop_mix(unsigned long long seed, unsigned long long counter) {
    unsigned long long z = seed + counter * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
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

// x[j] = kept ? x[j] * scale : 0 for the VEC elements from `idx` on; VEC > 1 needs an even idx.  A select, not a product:
// what is dropped leaves nothing behind, an infinity or NaN neither.
template <int VEC>
__device__ __forceinline__ void mam_drop_vec(float (&x)[VEC], unsigned long long seed, unsigned long long idx,
                                             unsigned threshold, float scale) {
    if constexpr (VEC == 1) {
        const unsigned long long z = mam_drop_mix(seed, idx >> 1);
        const unsigned draw = (idx & 1) ? (unsigned)(z >> 32) : (unsigned)z;
        x[0] = draw >= threshold ? __fmul_rn(x[0], scale) : 0.f;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const unsigned long long z = mam_drop_mix(seed, (idx + j) >> 1);
            x[j] = (unsigned)z >= threshold ? __fmul_rn(x[j], scale) : 0.f;
            x[j + 1] = (unsigned)(z >> 32) >= threshold ? __fmul_rn(x[j + 1], scale) : 0.f;
        }
    }
}

}  // namespace mamb200
