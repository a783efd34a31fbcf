// Sixteen-byte vectors of fp32, fp16 or bf16, with the arithmetic on packed pairs of fp32 (one instruction for two
// elements: the operators that use this file are close to the card's issue rate where their tensors are 16-bit).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>


namespace mamb200 {

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ void split2(float2 v, float& a, float& b) {
    a = v.x;
    b = v.y;
}
__device__ __forceinline__ float2 splat2(float x) { return make_float2(x, x); }
__device__ __forceinline__ float sum2(float2 v) {
    float lo, hi;
    split2(v, lo, hi);
    return lo + hi;
}

template <typename T>
constexpr int VEC = 16 / sizeof(T);      // elements of a vector
// Where a row's vectors lie: FULL, 16-byte aligned and one for each of a thread's; ALIGNED, but some threads have fewer;
// RAGGED, at any element, the last one cut short.
enum { RAGGED, ALIGNED, FULL };
template <typename T>
using Vals = float2[VEC<T> / 2];        // its values

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

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, Vals<T>& f) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
        f[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        f[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                f[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
            } else {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                f[j] = make_float2(v.x, v.y);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const Vals<T>& f) {
    unsigned w[4];
    if constexpr (sizeof(T) == 4) {
        float a, b;
        split2(f[0], a, b);
        w[0] = __float_as_uint(a);
        w[1] = __float_as_uint(b);
        split2(f[1], a, b);
        w[2] = __float_as_uint(a);
        w[3] = __float_as_uint(b);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a, b;
            split2(f[j], a, b);
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
                w[j] = *reinterpret_cast<const unsigned*>(&v);
            } else {
                const __half2 v = __floats2half2_rn(a, b);
                w[j] = *reinterpret_cast<const unsigned*>(&v);
            }
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// element j of a vector, j a constant after unrolling
template <typename T>
__device__ __forceinline__ T element(const uint4& q, int j) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(w[j]);
    } else {
        const unsigned short h = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
        return *reinterpret_cast<const T*>(&h);
    }
}

// values from n on become zero
template <typename T>
__device__ __forceinline__ void keep_first(Vals<T>& f, int n) {
#pragma unroll
    for (int j = 0; j < VEC<T> / 2; ++j) {
        float a, b;
        split2(f[j], a, b);
        f[j] = make_float2(2 * j < n ? a : 0.f, 2 * j + 1 < n ? b : 0.f);
    }
}

// The 16 bytes that begin `off` bytes (0 .. 16, a multiple of the element) into the 32 bytes of a and b.
template <typename T>
__device__ __forceinline__ uint4 cut(const uint4& a, const uint4& b, unsigned off) {
    unsigned w[9] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, 0u};
    const unsigned q = off >> 2;
    if (q & 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = w[j + 4];
        w[4] = 0u;
    }
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = (q & 2) ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = (q & 1) ? w[j + 1] : w[j];
    if constexpr (sizeof(T) == 2) {
        const unsigned bits = (off & 2u) * 8u;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], bits);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A tensor's row as it is read.  Rows whose starts are not 16-byte aligned (odd widths, slices) are read with aligned
// vectors all the same: a thread loads the two that hold its 16 bytes (the second one comes from L1, its neighbour reads it
// too) and shifts them together, by the same distance all along the row.  Element by element it took 8 times the loads.
// The aligned blocks are read only where they lie inside the tensor, [lo, hi): a row that may reach its ends (`inside`
// false) tests each of them, and reads element by element where one does not.
template <typename T, int MODE>
struct RowSrc {
    const T* row;
    uintptr_t lo, hi;
    unsigned off;
    bool inside;
    // a row of `width` elements at `at`, in a tensor of `rows` of them, `pitch` apart, at `base`
    __device__ __forceinline__ RowSrc(const T* base, long long pitch, long long rows, long long width, const T* at) {
        row = at;
        if constexpr (MODE == RAGGED) {
            lo = reinterpret_cast<uintptr_t>(base);
            hi = reinterpret_cast<uintptr_t>(base + (rows - 1) * pitch + width);
            off = (unsigned)(reinterpret_cast<uintptr_t>(row) & 15u);
            inside = reinterpret_cast<uintptr_t>(row) - off >= lo && reinterpret_cast<uintptr_t>(row + width) + 32 <= hi;
        }
    }
    // the vector at column c (a multiple of VEC), of which n (1 .. VEC) elements lie in the row; the others are undefined
    // STREAM: past L1, where the parameters are to stay; for tensors that the kernel does not write
    template <bool STREAM = true>
    __device__ __forceinline__ uint4 load(long long c, int n) const {
        const T* p = row + c;
        if constexpr (MODE != RAGGED && !STREAM) {
            return *reinterpret_cast<const uint4*>(p);
        } else if constexpr (MODE != RAGGED) {
            return __ldcg(reinterpret_cast<const uint4*>(p));
        } else {
            const uintptr_t a = reinterpret_cast<uintptr_t>(p) - off;
            if (inside || (a >= lo && a + 32 <= hi))
                return cut<T>(*reinterpret_cast<const uint4*>(a), *reinterpret_cast<const uint4*>(a + 16), off);
            unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < VEC<T>; ++j)
                if (j < n) {
                    if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(p[j]);
                    else w[j >> 1] |= (unsigned)*reinterpret_cast<const unsigned short*>(p + j) << (16 * (j & 1));
                }
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// Stores a row's vectors.  The lanes of a warp hold consecutive vectors of one row, or of one row each group of `lanes`, and
// call it together (shuffles), vector after vector where the warp has several: lane t for the vector at p, of which `rest`
// elements lie in the row from there on (<= 0: none; it joins in the shuffles).  Unaligned, a lane writes the aligned block
// that ends inside its vector, with the end of the vector before it in front (its neighbour's, or for lane 0 the last
// lane's of the call before, in `carry`); only what has no such neighbour, at the ends of the warp's columns and of the
// row, is written element by element.
template <typename T, int MODE>
__device__ __forceinline__ void store_vec(T* p, const uint4& o, int rest, int t, int lanes, bool first, bool last,
                                          uint4& carry) {
    constexpr int V = VEC<T>;
    if constexpr (MODE != RAGGED) {
        if (rest > 0) *reinterpret_cast<uint4*>(p) = o;
    } else {
        const unsigned off = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u);
        const int head = (int)((16u - off) / sizeof(T));     // elements of the vector in its first aligned block
        const int from = (int)(threadIdx.x & 31 & ~(lanes - 1)) | ((t - 1) & (lanes - 1));   // the lane before, or the last
        uint4 prev;
        prev.x = __shfl_sync(~0u, o.x, from);
        prev.y = __shfl_sync(~0u, o.y, from);
        prev.z = __shfl_sync(~0u, o.z, from);
        prev.w = __shfl_sync(~0u, o.w, from);
        const uint4 wrapped = prev;
        if (!first && t == 0) prev = carry;
        carry = wrapped;
        int j0 = 0, j1 = rest < V ? rest : V;                // the elements that are left to write one by one
        if (rest >= V && (t > 0 || !first || off == 0)) {
            *reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(p) - off) = cut<T>(prev, o, 16u - off);
            j0 = head;
        }
        if (rest >= 2 * V && (t < lanes - 1 || !last)) j1 = head;   // the next vector's lane writes the rest
        if (j0 < j1) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j >= j0 && j < j1) p[j] = element<T>(o, j);
        }
    }
}

// Weights and biases of a norm: fp32, or the activations' type.  The branches are the same for the whole grid.
// A missing weight is one, a missing bias zero.
template <typename T, int MODE>
__device__ __forceinline__ void load_param(const void* p, bool is_f32, int c, int n, float missing, Vals<T>& f) {
    constexpr int V = VEC<T>;
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) f[j] = splat2(missing);
    } else if (MODE == RAGGED && (n < V || (reinterpret_cast<uintptr_t>(p) & 15u))) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (2 * j + k < n)
                    v[k] = is_f32 ? static_cast<const float*>(p)[c + 2 * j + k]
                                  : to_f32(static_cast<const T*>(p)[c + 2 * j + k]);
            f[j] = make_float2(v[0], v[1]);
        }
    } else if (sizeof(T) == 2 && is_f32) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + c);
        const float4 a = q[0], b = q[1];
        f[0] = make_float2(a.x, a.y);
        f[1] = make_float2(a.z, a.w);
        f[V / 2 - 2] = make_float2(b.x, b.y);
        f[V / 2 - 1] = make_float2(b.z, b.w);
    } else {
        unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p) + c), f);
    }
}

}  // namespace mamb200
