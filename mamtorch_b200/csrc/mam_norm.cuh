// Layer norm over the rows of [rows, width], alone or behind a residual addition with dropout, forward and backward.
//
//   s = residual + drop(x), rounded to the type (or s = x)        mu = mean(s)      r = 1 / sqrt(mean((s - mu)^2) + eps)
//   h = (s - mu) r                                                y = h w + b
//   a = gy w    ds = r (a - mean(a) - h mean(a h)) + gs           dx = drop(ds)     dw = sum_rows gy h    db = sum_rows gy
//
// The norm reads the sum as it is stored, rounded: the fused call then equals the residual addition followed by the norm
// bit for bit, and the backward, which has only the stored sum, differentiates exactly what the forward computed.
//
// Bound by memory: forward one read and one write of the rows (two and two with the residual), backward two reads and one
// write (three and two).  A row stays in registers between its load and its store; statistics take two reductions, the
// mean first and the deviations from it second, so that a mean far from zero costs no digits.
#pragma once
#include "mam_drop.cuh"
#include "mam_vec.cuh"

namespace mamb200 {

struct NormFwdParams {
    const void* x;
    const void* residual;      // nullptr: s = x
    const void* weight;        // nullptr: ones
    const void* bias;          // nullptr: zeros
    void* y;
    void* sum;                 // s, with a residual
    float2* stats;             // (mu, r) of each row, or nullptr
    long long rows, width, x_pitch, res_pitch;
    float eps;
    bool params_f32;
    DropArgs drop;
};

struct NormBwdParams {
    const void* gy;            // nullptr: zeros
    const void* gs;            // gradient of the stored sum, or nullptr
    const void* s;             // what the forward normalised
    const float2* stats;
    const void* weight;
    void* ds;
    void* dx;                  // drop(ds), or nullptr
    float* partial;            // [blocks][2][width]: sums of gy h and of gy over the block's rows, or nullptr
    long long rows, width, s_pitch;
    bool params_f32;
    DropArgs drop;
};

// Sum of two values over a row's threads: the lanes of one warp, or all warps of the CTA.  `slot` is shared memory of
// one float2 a warp, another one for each reduction that may still be read.
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float a, float b, float2* slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(~0u, a, o);
        b += __shfl_xor_sync(~0u, b, o);
    }
    if constexpr (WARP) return make_float2(a, b);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slot[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const float2 v = lane < warps ? slot[lane] : make_float2(0.f, 0.f);
    a = v.x;
    b = v.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(~0u, a, o);
        b += __shfl_xor_sync(~0u, b, o);
    }
    return make_float2(a, b);
}

// s = round(residual + drop(x)), each step rounded by itself
template <typename T, int VEC>
__device__ __forceinline__ void add_residual(const Pack<T, VEC>& px, const Pack<T, VEC>& pr, const DropArgs& d,
                                             unsigned long long seed, unsigned long long idx, Pack<T, VEC>& ps) {
    float x[VEC], r[VEC];
    unpack(px, x);
    unpack(pr, r);
    if (d.on) mam_drop_vec<VEC>(x, seed, idx, d.threshold, d.scale);
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = __fadd_rn(r[j], x[j]);
    ps = pack<T, VEC>(x);
}

// mean, and 1 / sqrt(variance + eps), of `width` values of which this thread holds v[NV][VEC] (live(i): vector i is inside)
template <bool WARP, int NV, int VEC, class Live>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][VEC], Live live, long long width, float eps, float2* slot) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (!live(i)) continue;
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t += v[i][j];
        s += t;
    }
    const float n = (float)width;
    float mu = row_sum<WARP>(s, 0.f, slot).x / n;
    float d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (!live(i)) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float d = v[i][j] - mu;
            d1 += d;
            d2 = fmaf(d, d, d2);
        }
    }
    const float2 t = row_sum<WARP>(d1, d2, slot + 32);
    // the deviations' own mean is what rounding left in mu: with it a row of equal values comes out as exactly zero
    const float off = t.x / n;
    const float var = fmaxf(t.y / n - off * off, 0.f);
    return make_float2(mu + off, __frsqrt_rn(var + eps));
}

// Rows of up to NV * VEC * threads values: one warp a row, or one CTA.
template <typename T, int VEC, int NV, bool ADD, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) mam_norm_fwd_kernel(const __grid_constant__ NormFwdParams p) {
    __shared__ float2 slot[64];
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x, nt = WARP ? 32 : blockDim.x;
    const long long row = WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= p.rows) return;
    const int width = (int)p.width;
    auto col = [&](int i) { return (i * nt + t) * VEC; };
    auto live = [&](int i) { return col(i) < width; };
    const T* x = static_cast<const T*>(p.x) + row * p.x_pitch;
    float v[NV][VEC];
    if constexpr (ADD) {
        const T* r = static_cast<const T*>(p.residual) + row * p.res_pitch;
        T* sum = static_cast<T*>(p.sum) + row * p.width;
        const unsigned long long seed = p.drop.on ? p.drop.seed_now() : 0;
        Pack<T, VEC> px[NV], pr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
                px[i] = load_pack<T, VEC>(x + col(i));
                pr[i] = load_pack<T, VEC>(r + col(i));
            }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
                Pack<T, VEC> ps;
                add_residual(px[i], pr[i], p.drop, seed, (unsigned long long)(row * p.width + col(i)), ps);
                *reinterpret_cast<Pack<T, VEC>*>(sum + col(i)) = ps;
                unpack(ps, v[i]);
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) load_f32<T, VEC>(x + col(i), v[i]);
    }
    const float2 st = row_stats<WARP>(v, live, p.width, p.eps, slot);
    if (p.stats && t == 0) p.stats[row] = st;
    T* y = static_cast<T*>(p.y) + row * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live(i)) {
            float w[VEC], b[VEC];
            load_param<T, VEC>(p.weight, p.params_f32, col(i), 1.f, w);
            load_param<T, VEC>(p.bias, p.params_f32, col(i), 0.f, b);
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[j] = fmaf((v[i][j] - st.x) * st.y, w[j], b[j]);
            store_f32<T, VEC>(y + col(i), w);
        }
}

// Rows of any width: one CTA a row, which reads it again for each of its steps (from L2 mostly).
template <typename T, int VEC, bool ADD>
__global__ void __launch_bounds__(1024) mam_norm_fwd_wide_kernel(const __grid_constant__ NormFwdParams p) {
    __shared__ float2 slot[64];
    const long long row = blockIdx.x, step = (long long)blockDim.x * VEC;
    const long long c0 = (long long)threadIdx.x * VEC;
    const T* src = static_cast<const T*>(p.x) + row * p.x_pitch;
    float s = 0.f;
    if constexpr (ADD) {
        const T* r = static_cast<const T*>(p.residual) + row * p.res_pitch;
        T* sum = static_cast<T*>(p.sum) + row * p.width;
        const unsigned long long seed = p.drop.on ? p.drop.seed_now() : 0;
        for (long long c = c0; c < p.width; c += step) {
            Pack<T, VEC> ps;
            float v[VEC];
            add_residual(load_pack<T, VEC>(src + c), load_pack<T, VEC>(r + c), p.drop, seed,
                         (unsigned long long)(row * p.width + c), ps);
            *reinterpret_cast<Pack<T, VEC>*>(sum + c) = ps;
            unpack(ps, v);
            float q = 0.f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) q += v[j];
            s += q;
        }
        src = sum;   // each thread reads back what it wrote itself
    } else {
        for (long long c = c0; c < p.width; c += step) {
            float v[VEC], q = 0.f;
            load_f32<T, VEC>(src + c, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) q += v[j];
            s += q;
        }
    }
    const float n = (float)p.width;
    const float mu = row_sum<false>(s, 0.f, slot).x / n;
    float d1 = 0.f, d2 = 0.f;
    for (long long c = c0; c < p.width; c += step) {
        float v[VEC], q1 = 0.f, q2 = 0.f;
        load_f32<T, VEC>(src + c, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float d = v[j] - mu;
            q1 += d;
            q2 = fmaf(d, d, q2);
        }
        d1 += q1;
        d2 += q2;
    }
    const float2 t = row_sum<false>(d1, d2, slot + 32);
    const float off = t.x / n;
    const float2 st = make_float2(mu + off, __frsqrt_rn(fmaxf(t.y / n - off * off, 0.f) + p.eps));
    if (p.stats && threadIdx.x == 0) p.stats[row] = st;
    T* y = static_cast<T*>(p.y) + row * p.width;
    for (long long c = c0; c < p.width; c += step) {
        float v[VEC], w[VEC], b[VEC];
        load_f32<T, VEC>(src + c, v);
        load_param<T, VEC>(p.weight, p.params_f32, c, 1.f, w);
        load_param<T, VEC>(p.bias, p.params_f32, c, 0.f, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = fmaf((v[j] - st.x) * st.y, w[j], b[j]);
        store_f32<T, VEC>(y + c, w);
    }
}

// Backward of rows of up to NV * VEC * group values.  blockDim.x / group groups of `group` threads (a multiple of 32)
// walk the rows; a thread keeps its columns' sums of gy h and gy in registers over all of them, and the CTA leaves one
// partial row of each.
template <typename T, int VEC, int NV, bool ADD>
__global__ void __launch_bounds__(1024) mam_norm_bwd_kernel(const __grid_constant__ NormBwdParams p, int group) {
    extern __shared__ float cols[];    // [2][width], with several groups
    __shared__ float2 slot[2][32];
    const int groups = blockDim.x / group, g = threadIdx.x / group, t = threadIdx.x % group;
    const int warps = group >> 5, lane = threadIdx.x & 31, first = (g * group) >> 5;
    const int width = (int)p.width;
    auto col = [&](int i) { return (i * group + t) * VEC; };
    auto live = [&](int i) { return col(i) < width; };
    const unsigned long long seed = ADD && p.drop.on ? p.drop.seed_now() : 0;
    float w[NV][VEC], aw[NV][VEC], ab[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (live(i)) load_param<T, VEC>(p.weight, p.params_f32, col(i), 1.f, w[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) aw[i][j] = ab[i][j] = 0.f;
    }
    const float inv_n = 1.f / (float)p.width;
    const long long step = (long long)gridDim.x * groups;
    int parity = 0;
    for (long long row = (long long)blockIdx.x * groups + g; row < p.rows; row += step) {
        const T* s = static_cast<const T*>(p.s) + row * p.s_pitch;
        const float2 st = p.stats[row];
        float h[NV][VEC], a[NV][VEC];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
                load_f32<T, VEC>(s + col(i), h[i]);
                if (p.gy) load_f32<T, VEC>(static_cast<const T*>(p.gy) + row * p.width + col(i), a[i]);
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j) a[i][j] = 0.f;
            }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    h[i][j] = (h[i][j] - st.x) * st.y;
                    aw[i][j] = fmaf(a[i][j], h[i][j], aw[i][j]);
                    ab[i][j] += a[i][j];
                    a[i][j] *= w[i][j];
                    s1 += a[i][j];
                    s2 = fmaf(a[i][j], h[i][j], s2);
                }
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s1 += __shfl_xor_sync(~0u, s1, o);
            s2 += __shfl_xor_sync(~0u, s2, o);
        }
        if (warps > 1) {
            // two sets of slots in turn: a set is written again only behind the next row's barrier
            if (lane == 0) slot[parity][threadIdx.x >> 5] = make_float2(s1, s2);
            asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "r"(group) : "memory");
            const float2 v = lane < warps ? slot[parity][first + lane] : make_float2(0.f, 0.f);
            s1 = v.x;
            s2 = v.y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                s1 += __shfl_xor_sync(~0u, s1, o);
                s2 += __shfl_xor_sync(~0u, s2, o);
            }
            parity ^= 1;
        }
        s1 *= inv_n;
        s2 *= inv_n;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
                const long long at = row * p.width + col(i);
                float d[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] = st.y * (a[i][j] - s1 - h[i][j] * s2);
                if constexpr (ADD) {
                    if (p.gs) {
                        float q[VEC];
                        load_f32<T, VEC>(static_cast<const T*>(p.gs) + at, q);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) d[j] += q[j];
                    }
                }
                store_f32<T, VEC>(static_cast<T*>(p.ds) + at, d);
                if constexpr (ADD) {
                    if (p.dx) {
                        mam_drop_vec<VEC>(d, seed, (unsigned long long)at, p.drop.threshold, p.drop.scale);
                        store_f32<T, VEC>(static_cast<T*>(p.dx) + at, d);
                    }
                }
            }
    }
    if (!p.partial) return;
    float* out = p.partial + (long long)blockIdx.x * 2 * p.width;
    // the groups add to the columns one after the other: a fixed order
    for (int k = 0; k < groups; ++k) {
        if (g == k) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (live(i)) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int c = col(i) + j;
                        if (k > 0) {
                            aw[i][j] += cols[c];
                            ab[i][j] += cols[width + c];
                        }
                        if (k < groups - 1) {
                            cols[c] = aw[i][j];
                            cols[width + c] = ab[i][j];
                        } else {
                            out[c] = aw[i][j];
                            out[width + c] = ab[i][j];
                        }
                    }
                }
        }
        if (groups > 1) __syncthreads();
    }
}

// Backward of rows of any width: gradients of the rows, one CTA a row, without the columns' sums.
template <typename T, int VEC, bool ADD>
__global__ void __launch_bounds__(1024) mam_norm_bwd_wide_kernel(const __grid_constant__ NormBwdParams p) {
    __shared__ float2 slot[32];
    const long long row = blockIdx.x, step = (long long)blockDim.x * VEC, c0 = (long long)threadIdx.x * VEC;
    const T* s = static_cast<const T*>(p.s) + row * p.s_pitch;
    const T* gy = p.gy ? static_cast<const T*>(p.gy) + row * p.width : nullptr;
    const float2 st = p.stats[row];
    const unsigned long long seed = ADD && p.drop.on ? p.drop.seed_now() : 0;
    float s1 = 0.f, s2 = 0.f;
    if (gy)
        for (long long c = c0; c < p.width; c += step) {
            float h[VEC], a[VEC], w[VEC], q1 = 0.f, q2 = 0.f;
            load_f32<T, VEC>(s + c, h);
            load_f32<T, VEC>(gy + c, a);
            load_param<T, VEC>(p.weight, p.params_f32, c, 1.f, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                a[j] *= w[j];
                q1 += a[j];
                q2 = fmaf(a[j], (h[j] - st.x) * st.y, q2);
            }
            s1 += q1;
            s2 += q2;
        }
    const float2 m = row_sum<false>(s1, s2, slot);
    s1 = m.x / (float)p.width;
    s2 = m.y / (float)p.width;
    for (long long c = c0; c < p.width; c += step) {
        const long long at = row * p.width + c;
        float h[VEC], d[VEC], w[VEC];
        load_f32<T, VEC>(s + c, h);
        if (gy) load_f32<T, VEC>(gy + c, d);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[j] = 0.f;
        load_param<T, VEC>(p.weight, p.params_f32, c, 1.f, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[j] = st.y * (d[j] * w[j] - s1 - (h[j] - st.x) * st.y * s2);
        if constexpr (ADD) {
            if (p.gs) {
                load_f32<T, VEC>(static_cast<const T*>(p.gs) + at, h);
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] += h[j];
            }
        }
        store_f32<T, VEC>(static_cast<T*>(p.ds) + at, d);
        if constexpr (ADD) {
            if (p.dx) {
                mam_drop_vec<VEC>(d, seed, (unsigned long long)at, p.drop.threshold, p.drop.scale);
                store_f32<T, VEC>(static_cast<T*>(p.dx) + at, d);
            }
        }
    }
}

constexpr int NORM_COLS = 32, NORM_LANES = 8;

// The columns' sums of gy h and gy over slabs of rows, for rows wider than a CTA's registers hold: grid (column groups,
// slabs), into partial[slab][2][width].
template <typename T>
__global__ void __launch_bounds__(NORM_COLS * NORM_LANES)
mam_norm_bwd_cols_kernel(const __grid_constant__ NormBwdParams p, long long rows_per) {
    __shared__ float2 part[NORM_LANES][NORM_COLS];
    const int c = threadIdx.x % NORM_COLS, l = threadIdx.x / NORM_COLS;
    const long long n = (long long)blockIdx.x * NORM_COLS + c;
    const long long m0 = (long long)blockIdx.y * rows_per, m1 = min(m0 + rows_per, p.rows);
    float2 sum = make_float2(0.f, 0.f);
    if (n < p.width && p.gy)
        for (long long m = m0 + l; m < m1; m += NORM_LANES) {
            const float2 st = p.stats[m];
            const float a = to_f32(static_cast<const T*>(p.gy)[m * p.width + n]);
            sum.x = fmaf(a, (to_f32(static_cast<const T*>(p.s)[m * p.s_pitch + n]) - st.x) * st.y, sum.x);
            sum.y += a;
        }
    part[l][c] = sum;
    __syncthreads();
    if (l == 0 && n < p.width) {
        for (int i = 1; i < NORM_LANES; ++i) {
            sum.x += part[i][c].x;
            sum.y += part[i][c].y;
        }
        float* out = p.partial + (long long)blockIdx.y * 2 * p.width;
        out[n] = sum.x;
        out[p.width + n] = sum.y;
    }
}

// dw and db: the partial rows added in a fixed order, rounded once to the parameters' type.
template <typename T>
__global__ void __launch_bounds__(NORM_COLS * NORM_LANES)
mam_norm_params_kernel(const float* __restrict__ partial, void* dweight, void* dbias, long long parts, long long width,
                       bool params_f32) {
    __shared__ float part[NORM_LANES][NORM_COLS];
    const int c = threadIdx.x % NORM_COLS, l = threadIdx.x / NORM_COLS;
    const long long n = (long long)blockIdx.x * NORM_COLS + c;      // 0 .. 2 * width - 1: weight, then bias
    float s = 0.f;
    if (n < 2 * width)
        for (long long m = l; m < parts; m += NORM_LANES) s += partial[m * 2 * width + n];
    part[l][c] = s;
    __syncthreads();
    if (l != 0 || n >= 2 * width) return;
    for (int i = 1; i < NORM_LANES; ++i) s += part[i][c];
    void* out = n < width ? dweight : dbias;
    if (!out) return;
    const long long at = n < width ? n : n - width;
    if (params_f32) static_cast<float*>(out)[at] = s;
    else static_cast<T*>(out)[at] = from_f32<T>(s);
}

}  // namespace mamb200
