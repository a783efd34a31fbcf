// GELU with dropout, and dropout with a residual addition, over flat tensors; forward and backward.
//
//   gelu:     y = drop(x Phi(x))             dx = drop(gy (Phi(x) + x phi(x)))        Phi, phi: the normal distribution
//   dropout:  y = residual + drop(x)         dx = drop(gy)
//
// Bound by memory: each tensor is read or written once.  Arithmetic in fp32, rounded once.
#pragma once
#include "mam_drop.cuh"
#include "mam_vec.cuh"

namespace mamb200 {

struct PointParams {
    const void* x;
    const void* other;     // residual (or nullptr), or the upstream gradient
    void* out;
    long long n;
    DropArgs drop;
};

enum PointOp { POINT_DROPOUT, POINT_GELU, POINT_GELU_BWD };

__device__ __forceinline__ float gelu_cdf(float x) { return 0.5f * (1.f + erff(x * 0.70710678118654752f)); }

template <int OP, int VEC>
__device__ __forceinline__ void point_apply(float (&x)[VEC], const float (&o)[VEC], bool has_other, const DropArgs& d,
                                            unsigned long long seed, unsigned long long idx) {
    if constexpr (OP == POINT_DROPOUT) {
        if (d.on) mam_drop_vec<VEC>(x, seed, idx, d.threshold, d.scale);
        if (has_other) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[j] = __fadd_rn(o[j], x[j]);
        }
    } else if constexpr (OP == POINT_GELU) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] *= gelu_cdf(x[j]);
        if (d.on) mam_drop_vec<VEC>(x, seed, idx, d.threshold, d.scale);
    } else {
        // the mask last: what the forward dropped gets a zero whatever its x was
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float slope = fmaf(x[j] * 0.39894228040143268f, expf(-0.5f * x[j] * x[j]), gelu_cdf(x[j]));
            x[j] = o[j] * slope;
        }
        if (d.on) mam_drop_vec<VEC>(x, seed, idx, d.threshold, d.scale);
    }
}

// NV vectors a thread, all loads first; the ragged end element by element.
template <typename T, int VEC, int NV, int OP>
__global__ void __launch_bounds__(256) mam_point_kernel(const __grid_constant__ PointParams p) {
    const T* x = static_cast<const T*>(p.x);
    const T* o = static_cast<const T*>(p.other);
    T* out = static_cast<T*>(p.out);
    const unsigned long long seed = p.drop.on ? p.drop.seed_now() : 0;
    const bool has = o != nullptr;
    const long long base = ((long long)blockIdx.x * NV * 256 + threadIdx.x) * VEC;
    Pack<T, VEC> px[NV], po[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long at = base + (long long)i * 256 * VEC;
        if (at + VEC <= p.n) {
            px[i] = load_pack<T, VEC>(x + at);
            if (has) po[i] = load_pack<T, VEC>(o + at);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long at = base + (long long)i * 256 * VEC;
        if (at + VEC <= p.n) {
            float f[VEC], q[VEC];
            unpack(px[i], f);
            if (has) unpack(po[i], q);
            point_apply<OP, VEC>(f, q, has, p.drop, seed, (unsigned long long)at);
            store_f32<T, VEC>(out + at, f);
        } else if (VEC > 1) {
            for (long long e = at; e < p.n && e < at + VEC; ++e) {
                float f[1] = {to_f32(x[e])}, q[1] = {has ? to_f32(o[e]) : 0.f};
                point_apply<OP, 1>(f, q, has, p.drop, seed, (unsigned long long)e);
                out[e] = from_f32<T>(f[0]);
            }
        }
    }
}

}  // namespace mamb200
