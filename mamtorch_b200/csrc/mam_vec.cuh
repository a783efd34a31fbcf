// Loads and stores of VEC consecutive elements of fp32, fp16 or bf16, with the arithmetic in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace mamb200 {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& a, float (&f)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = to_f32(a.v[j]);
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&f)[VEC]) {
    Pack<T, VEC> a;
#pragma unroll
    for (int j = 0; j < VEC; ++j) a.v[j] = from_f32<T>(f[j]);
    return a;
}
template <typename T, int VEC>
__device__ __forceinline__ void load_f32(const T* p, float (&f)[VEC]) {
    unpack(load_pack<T, VEC>(p), f);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_f32(T* p, const float (&f)[VEC]) {
    *reinterpret_cast<Pack<T, VEC>*>(p) = pack<T, VEC>(f);
}

// Weights and biases of a norm: fp32, or the activations' type.  The branch is the same for the whole grid.
// A missing weight is one, a missing bias zero.
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, bool is_f32, long long c, float missing, float (&f)[VEC]) {
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = missing;
    } else if (is_f32) {
        const float* q = static_cast<const float*>(p) + c;
        if constexpr (VEC == 8) {
            const float4 lo = *reinterpret_cast<const float4*>(q), hi = *reinterpret_cast<const float4*>(q + 4);
            f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
            f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
        } else {
            load_f32<float, VEC>(q, f);
        }
    } else {
        load_f32<T, VEC>(static_cast<const T*>(p) + c, f);
    }
}

}  // namespace mamb200
