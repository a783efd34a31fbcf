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
    int tail;              // elements behind the n of the whole vectors (TAIL)
    DropArgs drop;
};

enum PointOp { POINT_DROPOUT, POINT_GELU, POINT_GELU_BWD };

// q = -erfc(a / sqrt(2)) / 2 and e = exp(-a^2 / 2) for a = min(|x|, 15), pairwise: the form of Abramowitz and Stegun, 7.1.26,
// t P(t) e with t = 1 / (1 + k a), and coefficients of our own fits.  erff and expf took 33 instructions an element and twice
// the time of the bytes in bf16; this takes a reciprocal, an exponential and the rest in packed pairs.  15: beyond it q is
// zero in fp32; min.NaN passes a NaN on.
//
// 16-bit types: k = 0.28, six coefficients (as they stand off by 1.1e-8 at most, at a = 1.09; roundings make it 2e-7 at
// a = 0, where q is of the order of one half).
// fp32: there that absolute error would show (x Phi(x) off by 4.7e-7 relative, rms 1.0e-7, where erff's form has 2.2e-7 and 4.6e-8),
// and for a < 1 q = a R(a^2) - 1/2, R a polynomial, off by 7e-9.  From a = 1 on R's form is too high, more and more so; the
// other one, k = 0.37 with five coefficients fitted from a = 1 on (a q off by 4.6e-9), is too high below it, by more than
// its roundings from 0.9 down.  So the lower of the two is the one that counts, and close to 1 either is: 2.9e-7, rms 4.0e-8.
// 12608x4096 with dropout, forward and backward: 151.5 -> 150.2 us; under load for seconds, where the power limit takes the
// clock to 1.5 GHz and instructions count, 163.7 -> 173.5 (28.2 -> 31.5 and 31.3 -> 35.2 an element).  erff and expf took 202.
template <typename T>
__device__ __forceinline__ void normal_tail(float2 x, float2& a, float2& q, float2& e) {
    float u, v;
    split2(x, u, v);
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(u) : "f"(fabsf(u)), "f"(15.f));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(fabsf(v)), "f"(15.f));
    a = make_float2(u, v);
    split2(fma2(a, splat2(sizeof(T) == 2 ? 0.28f : 0.37f), splat2(1.f)), u, v);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(u));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v));
    const float2 t = make_float2(u, v), aa = mul2(a, a);
    split2(mul2(aa, splat2(-0.72134752044448170f)), u, v);    // -a^2 / 2 in base 2
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(u));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(v));
    e = make_float2(u, v);
    if constexpr (sizeof(T) == 2) {
        float2 s = fma2(splat2(0.105807796f), t, splat2(-0.389872253f));
        s = fma2(s, t, splat2(0.23699066f));
        s = fma2(s, t, splat2(-0.268907934f));
        s = fma2(s, t, splat2(-0.0674976185f));
        s = fma2(s, t, splat2(-0.116520643f));
        q = mul2(mul2(s, t), e);
    } else {
        float2 s = fma2(splat2(0.10187085717916489f), t, splat2(-0.23629137873649597f));
        s = fma2(s, t, splat2(-0.05451401323080063f));
        s = fma2(s, t, splat2(-0.16487039625644684f));
        s = fma2(s, t, splat2(-0.14599835872650146f));
        s = mul2(mul2(s, t), e);
        float2 r = fma2(splat2(9.171009151032194e-05f), aa, splat2(-0.0011636228300631046f));
        r = fma2(r, aa, splat2(0.009962853975594044f));
        r = fma2(r, aa, splat2(-0.0664883628487587f));
        r = fma2(r, aa, splat2(0.39894217252731323f));
        r = fma2(a, r, splat2(-0.5f));
        q = make_float2(fminf(r.x, s.x), fminf(r.y, s.y));      // a NaN is in both
    }
}
// x Phi(x) = max(x, 0) + |x| q: zero at minus infinity, its limit
template <typename T>
__device__ __forceinline__ float2 gelu2(float2 x) {
    float2 a, q, e;
    normal_tail<T>(x, a, q, e);
    float u, v;
    split2(x, u, v);
    return fma2(a, q, make_float2(fmaxf(u, 0.f), fmaxf(v, 0.f)));
}
__device__ __forceinline__ float flip(float u, float sign) {
    return __uint_as_float(__float_as_uint(u) ^ (__float_as_uint(sign) & 0x80000000u));
}
// Phi(x) + x phi(x) = 1/2 + sign(x) (1/2 + q + a phi(a))
template <typename T>
__device__ __forceinline__ float2 gelu_slope2(float2 x) {
    float2 a, q, e;
    normal_tail<T>(x, a, q, e);
    float u, v, xu, xv;
    split2(add2(fma2(mul2(a, splat2(0.39894228040143268f)), e, splat2(0.5f)), q), u, v);
    split2(x, xu, xv);
    return add2(make_float2(flip(u, xu), flip(v, xv)), splat2(0.5f));
}

template <typename T, int OP, int N>
__device__ __forceinline__ void point_apply(float2 (&x)[N], const float2 (&o)[N], bool has_other, const DropArgs& d,
                                            unsigned long long start) {
    if constexpr (OP != POINT_DROPOUT) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = OP == POINT_GELU ? gelu2<T>(x[j]) : mul2(o[j], gelu_slope2<T>(x[j]));
    }
    // in the backward the mask comes last: what the forward dropped gets a zero whatever its x was
    if (d.on) mam_drop_pairs<N>(x, start, false, d.threshold, d.scale);
    if (OP == POINT_DROPOUT && has_other) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = add2(o[j], x[j]);
    }
}

constexpr int POINT_THREADS = 128;
// CTAs on an SM: the forward of GELU in fp32 needs 40 registers, and twelve CTAs take 67.7 us where eight or ten take 69.8
// (12608x4096 with dropout)
template <typename T, int OP, int MODE>
constexpr int POINT_CTAS = sizeof(T) == 4 && OP == POINT_GELU && MODE == ALIGNED ? 12 : 8;

// NV vectors a thread, all loads first; a CTA a block (CTAs that walk over several blocks took a sixth fewer instructions and
// a tenth longer: their loads wait for the stores before them).  ALIGNED: whole vectors only, n is a multiple of them; with TAIL
// one thread of a last CTA does the elements behind them, pair by pair (an instance of its own: the loop's registers cost the
// others a tenth).
// RAGGED: any n and any alignment, with the loads and stores of ragged rows, the whole tensor being one row.
template <typename T, int NV, int OP, int MODE, bool TAIL>
__global__ void __launch_bounds__(POINT_THREADS, POINT_CTAS<T, OP, MODE>) mam_point_kernel(const __grid_constant__ PointParams p) {
    constexpr int V = VEC<T>;
    const bool has = p.other != nullptr;
    const RowSrc<T, MODE> x(static_cast<const T*>(p.x), 0, 1, p.n, static_cast<const T*>(p.x)),
        o(static_cast<const T*>(p.other), 0, 1, p.n, static_cast<const T*>(p.other));
    T* out = static_cast<T*>(p.out);
    // ragged, a warp's vectors follow one another
    constexpr int STEP = MODE == RAGGED ? 32 * V : POINT_THREADS * V;
    const long long base = MODE == RAGGED
        ? (((long long)blockIdx.x * (POINT_THREADS / 32) + (threadIdx.x >> 5)) * (NV * 32) + (threadIdx.x & 31)) * V
        : ((long long)blockIdx.x * NV * POINT_THREADS + threadIdx.x) * V;
    if constexpr (TAIL) {
        if (blockIdx.x == gridDim.x - 1) {
            if (threadIdx.x > 0) return;
            const unsigned long long seed = p.drop.on ? p.drop.seed_now() : 0;
            const T *xt = static_cast<const T*>(p.x) + p.n, *ot = static_cast<const T*>(p.other) + p.n;
#pragma unroll 1
            for (int e = 0; e < p.tail; e += 2) {
                const bool two = e + 1 < p.tail;
                float2 f[1] = {make_float2(to_f32(xt[e]), two ? to_f32(xt[e + 1]) : 0.f)}, g[1] = {splat2(0.f)};
                if (has) g[0] = make_float2(to_f32(ot[e]), two ? to_f32(ot[e + 1]) : 0.f);
                point_apply<T, OP>(f, g, has, p.drop, mam_drop_start(seed, p.n + e));
                out[p.n + e] = from_f32<T>(f[0].x);
                if (two) out[p.n + e + 1] = from_f32<T>(f[0].y);
            }
            return;
        }
    }
    const unsigned long long start = p.drop.on ? mam_drop_start(p.drop.seed_now(), base) : 0;
    uint4 px[NV], po[NV], carry = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long at = base + i * STEP;
        if (at < p.n) {
            const int n = MODE == RAGGED ? (int)min((long long)V, p.n - at) : V;
            px[i] = x.template load<false>(at, n);
            if (has) po[i] = o.template load<false>(at, n);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long at = base + i * STEP;
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (at < p.n) {
            float2 f[V / 2], g[V / 2];
            unpack<T>(px[i], f);
            if (has) unpack<T>(po[i], g);
            point_apply<T, OP>(f, g, has, p.drop, start + (unsigned long long)(i * (STEP / 2)) * MAM_DROP_STEP);
            q = pack<T>(f);
        }
        const int rest = MODE == RAGGED ? (int)max(min(p.n - at, 2LL * V), 0LL) : at < p.n ? V : 0;
        store_vec<T, MODE>(out + at, q, rest, threadIdx.x & 31, 32, i == 0, i == NV - 1, carry);
    }
}

}  // namespace mamb200
