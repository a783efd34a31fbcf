// Layer norm over the rows of [rows, width], alone or behind a residual addition with dropout, forward and backward.
//
//   s = residual + drop(x), rounded to the type (or s = x)        mu = mean(s)      r = 1 / sqrt(mean((s - mu)^2) + eps)
//   h = (s - mu) r                                                y = h w + b
//   a = gy w    ds = r (a - mean(a) - h mean(a h)) + gs           dx = drop(ds)     dw = sum_rows gy h    db = sum_rows gy
//
// The norm reads the sum as it is stored, rounded: the fused call then equals the residual addition followed by the norm (s bit
// for bit, y up to the order of a row's sums), and the backward, which has only the stored sum, differentiates exactly what
// the forward computed.
//
// Bound by memory: forward one read and one write of the rows (two and two with the residual), backward two reads and one
// write (three and two).  A row stays in registers between its load and its store; statistics take two reductions, the
// mean first and the deviations from it second, so that a mean far from zero costs no digits.
#pragma once
#include "mam_drop.cuh"
#include "mam_host.cuh"
#include "mam_ptx.cuh"
#include "mam_vec.cuh"

namespace mamb200 {

// threads of a CTA that an SM's registers hold, by the values each keeps in the forward's ring
template <int PER>
constexpr int FWD_RING_THREADS = PER == 8 ? 1024 : PER == 16 ? 768 : 640;


struct NormFwdParams {
    const void* x;
    const void* residual;      // nullptr: s = x
    const void* weight;        // nullptr: ones
    const void* bias;          // nullptr: zeros
    void* y;
    void* sum;                 // s, with a residual
    float2* stats;             // (mu, r) of each row, or nullptr
    long long rows, width, x_pitch, res_pitch;
    float eps, inv_width;
    bool params_f32;
    WaitWords wait;            // set where a bounded wait ran out
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
    float inv_width;
    bool params_f32;
    WaitWords wait;            // set where a bounded wait ran out
    DropArgs drop;
};

// Sums over a row's threads: LANES neighbouring lanes (8, 16 or 32), and with CTA all its warps.  `slot` is shared memory of
// one value a warp, another one for each reduction that may still be read.
template <int LANES>
__device__ __forceinline__ float lane_sum(float a) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
    return a;
}
// Two sums at once: the first exchange leaves a in one half of the lanes and b in the other, six shuffles instead of ten.
template <int LANES>
__device__ __forceinline__ float2 lane_sum2(float a, float b) {
    const bool upper = threadIdx.x & (LANES / 2);
    const float v = lane_sum<LANES / 2>((upper ? b : a) + __shfl_xor_sync(~0u, upper ? a : b, LANES / 2));
    const float w = __shfl_xor_sync(~0u, v, LANES / 2);
    return upper ? make_float2(w, v) : make_float2(v, w);
}
// MOST: as many warps as the CTA can have, 16 or 32
template <bool CTA, int LANES, int MOST>
__device__ __forceinline__ float row_sum(float a, float* slot) {
    a = lane_sum<LANES>(a);
    if constexpr (CTA) {
        const int k = threadIdx.x & (MOST - 1);
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = a;
        __syncthreads();
        a = lane_sum<MOST>(k < (int)(blockDim.x >> 5) ? slot[k] : 0.f);
    }
    return a;
}
template <bool CTA, int LANES, int MOST>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* slot) {
    float2 v = lane_sum2<LANES>(a, b);
    if constexpr (CTA) {
        const int k = threadIdx.x & (MOST - 1);
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = k < (int)(blockDim.x >> 5) ? slot[k] : make_float2(0.f, 0.f);
        v = lane_sum2<MOST>(v.x, v.y);
    }
    return v;
}

// s = round(residual + drop(x)), each step rounded by itself
template <typename T>
__device__ __forceinline__ uint4 add_residual(const uint4& qx, const uint4& qr, const DropArgs& d,
                                              unsigned long long start, bool odd) {
    Vals<T> x, r;
    unpack<T>(qx, x);
    unpack<T>(qr, r);
    if (d.on) mam_drop_pairs<VEC<T> / 2>(x, start, odd, d.threshold, d.scale);
#pragma unroll
    for (int j = 0; j < VEC<T> / 2; ++j) x[j] = add2(r[j], x[j]);
    return pack<T>(x);
}

template <typename T>
__device__ __forceinline__ float2 total(const Vals<T>& v) {
    float2 s = v[0];
#pragma unroll
    for (int j = 1; j < VEC<T> / 2; ++j) s = add2(s, v[j]);
    return s;
}

// (mean, r) from the mean `mu` of the first reduction and the sums d1 of the deviations from it and d2 of their squares.  The
// deviations' own mean is what rounding left in mu; `off` is the step from mu to the corrected mean as it is stored, so
// that deviation - off is s - mean, the same as in the backward, and zero for a row of equal values whatever r is.
__device__ __forceinline__ float2 row_stats(float mu, float d1, float d2, float inv_n, float eps, float& off) {
    const float mean = fmaf(d1, inv_n, mu);
    off = mean - mu;
    return make_float2(mean, rsqrtf(fmaxf(d2 * inv_n - off * (2.f * (d1 * inv_n) - off), 0.f) + eps));
}

// Rows of up to NV vectors a thread, held in registers.  CTA: a CTA a row; else LANES lanes a row, 128 / LANES rows a CTA.
// Loads of a whole row at once and as many threads on an SM as the registers allow keep the memory busy: 85 % of the copy rate at
// [32768, 4096] bf16 (97 us; four vectors a thread instead of eight 108, for the reductions' instructions are paid per
// thread), 94 % at [4096, 8192] fp32.  FULL leaves out the tests for columns: 28 -> 14 instructions an element with the packed
// pairs.
template <typename T, int NV, bool ADD, int MODE, bool CTA, int LANES>
__global__ void __launch_bounds__(!CTA ? 128 : NV <= 2 ? 1024 : 512)
mam_norm_fwd_kernel(const __grid_constant__ NormFwdParams p) {
    __shared__ float2 slot[64];
    constexpr int V = VEC<T>, nt = LANES, MOST = NV <= 2 ? 32 : 16;
    const int t = threadIdx.x & (LANES - 1);
    const long long row = CTA ? (long long)blockIdx.x
                              : (long long)blockIdx.x * (128 / LANES) + threadIdx.x / LANES;
    const int width = CTA || row < p.rows ? (int)p.width : 0;    // no columns beyond the last row
    const int first = CTA ? (int)(threadIdx.x >> 5) * NV * 32 * V + t * V : t * V;    // a warp's vectors follow one another
    auto col = [&](int i) { return first + i * nt * V; };
    auto count = [&](int i) { return MODE == FULL ? (CTA || width ? V : 0) : min(V, width - col(i)); };
    uint4 carry = make_uint4(0u, 0u, 0u, 0u);
    const T* x0 = static_cast<const T*>(p.x);
    const RowSrc<T, MODE> x(x0, p.x_pitch, p.rows, p.width, x0 + row * p.x_pitch);
    uint4 qx[NV];
    float2 v[NV][V / 2];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (count(i) > 0) qx[i] = x.load(col(i), count(i));
    if constexpr (ADD) {
        const T* r0 = static_cast<const T*>(p.residual);
        const RowSrc<T, MODE> r(r0, p.res_pitch, p.rows, p.width, r0 + row * p.res_pitch);
        const long long at = row * p.width + first;
        const unsigned long long start = p.drop.on ? mam_drop_start(p.drop.seed_now(), at) : 0;
        const bool odd = MODE == RAGGED && (at & 1);
        uint4 qr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (count(i) > 0) qr[i] = r.load(col(i), count(i));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint4 qs = make_uint4(0u, 0u, 0u, 0u);
            if (count(i) > 0) {
                qs = add_residual<T>(qx[i], qr[i], p.drop, start + (unsigned long long)(i * nt * (V / 2)) * MAM_DROP_STEP, odd);
                unpack<T>(qs, v[i]);
            }
            store_vec<T, MODE>(static_cast<T*>(p.sum) + at + i * nt * V, qs, width - col(i), t, nt, i == 0, i == NV - 1, carry);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (count(i) > 0) unpack<T>(qx[i], v[i]);
    }
    float2 s = splat2(0.f), d1 = s, d2 = s;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (count(i) > 0) {
            if (MODE == RAGGED && count(i) < V) keep_first<T>(v[i], count(i));
            s = add2(s, total<T>(v[i]));
        }
    const float mu = row_sum<CTA, LANES, MOST>(sum2(s), reinterpret_cast<float*>(slot)) * p.inv_width;
    const float2 minus = splat2(-mu);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (count(i) > 0) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) v[i][j] = add2(v[i][j], minus);
            if (MODE == RAGGED && count(i) < V) keep_first<T>(v[i], count(i));
#pragma unroll
            for (int j = 0; j < V / 2; ++j) d2 = fma2(v[i][j], v[i][j], d2);
            d1 = add2(d1, total<T>(v[i]));
        }
    const float2 d = row_sum2<CTA, LANES, MOST>(sum2(d1), sum2(d2), slot + 32);
    float off;
    const float2 st = row_stats(mu, d.x, d.y, p.inv_width, p.eps, off);
    if (p.stats && first == 0 && width) p.stats[row] = st;
    const float2 r2 = splat2(st.y), o2 = splat2(-off);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (count(i) > 0) {
            float2 w[V / 2], b[V / 2];
            load_param<T, MODE>(p.weight, p.params_f32, col(i), count(i), 1.f, w);
            load_param<T, MODE>(p.bias, p.params_f32, col(i), count(i), 0.f, b);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) w[j] = fma2(mul2(add2(v[i][j], o2), r2), w[j], b[j]);
            q = pack<T>(w);
        }
        store_vec<T, MODE>(static_cast<T*>(p.y) + row * p.width + col(i), q, width - col(i), t, nt, i == 0, i == NV - 1, carry);
    }
}

// Places in shared memory of a ring of rows: `stages` rows of each of `groups` groups of `group` threads (whole warps) are
// there or on their way by bulk copies, so that loads go on whatever the registers leave room for.
struct NormRing {
    int group, groups, stages;
    unsigned slot_bytes;                   // of one tensor's row
    unsigned weights_at, bars_at, bytes;   // the parameters, the barriers; the whole
    unsigned late;                         // 1: the first wait counts as run out (tests)
};

constexpr unsigned RING_POLLS = 1u << 22;      // of a wait for a row; each may suspend the thread for a while

// A wait for a row ran out.  The results are void, which the flag says; the thread waits no more, but it meets every barrier of its
// group.  Where it is thread 0, which arms the barriers and sends for the rows, that ends here too (a barrier whose copy is
// pending must not be armed again), and it waits for the copies on their way, of `sent` rows from `row` on: they write
// to shared memory that the CTA may reuse or leave.  Another thread needs no such care: its stage is sent for again only
// behind its group's barrier, after thread 0 has seen it full.
__device__ __forceinline__ void ring_late(const WaitWords& w, uint64_t* full, int stages, int stage, unsigned phase, int sent,
                                          long long row, long long step, long long rows) {
    *w.flag = 1;
    *reinterpret_cast<volatile int*>(w.image) = 1;
    __threadfence_system();
    for (int k = 0; k < sent && row < rows; ++k, row += step) {
        mbar_wait_bounded(full + stage, phase, RING_POLLS);
        if (++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
}
// The same as a call: in the forward's kernels the code in line cost the loop its schedule ([32768,4096] bf16 behind a residual
// 205 us, with the call 180); in the backward's it is the faster one ([5003,1283] bf16 38.5 us for 40.3, [16384,5120] 170.6 for
// 175.5, with dropout and residual).
__device__ __noinline__ void ring_late_call(const WaitWords& w, uint64_t* full, int stages, int stage, unsigned phase, int sent,
                                            long long row, long long step, long long rows) {
    ring_late(w, full, stages, stage, phase, sent, row, step, rows);
}

// Many rows that are ragged, or too wide for the next kernel's loads to be held: one CTA an SM walks them with the parameters
// in shared memory, in fp32.  A group's row leaves its stage for the
// registers before the first reduction; behind that barrier thread 0 sends for the row `stages` ahead.  RAGGED rows are
// copied with the aligned 16 bytes at either end, which belong to the rows beside them; the first and the last row have no
// such neighbours and are brought element by element.
template <typename T, int NV, bool ADD, int MODE>
__global__ void __launch_bounds__(FWD_RING_THREADS<NV * VEC<T>>)
mam_norm_fwd_ring_kernel(const __grid_constant__ NormFwdParams p, const __grid_constant__ NormRing ring) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 slot[2][32];
    constexpr int V = VEC<T>, HALVES = V / 4, TENSORS = ADD ? 2 : 1, MOST = 32;
    const int group = ring.group, groups = ring.groups, g = threadIdx.x / group, t = threadIdx.x - g * group;
    const int lane = threadIdx.x & 31, warps = group >> 5, slot0 = (g * group) >> 5;
    const int width = (int)p.width;
    const int vec0 = (t >> 5) * NV * 32 + lane;     // a warp's vectors follow one another
    auto col = [&](int i) { return (vec0 + i * 32) * V; };
    auto count = [&](int i) { return MODE == FULL ? V : min(V, width - col(i)); };
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring.bars_at) + g * ring.stages;
    unsigned char* mine = smem + (size_t)g * ring.stages * TENSORS * ring.slot_bytes;      // [stage][x, residual][row]
    // weight and bias, the halves of a vector of eight apart: a warp's 16-byte reads then meet no bank twice
    float4* params = reinterpret_cast<float4*>(smem + ring.weights_at);
    const int vecs = (width + V - 1) / V;
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
        float2 w[V / 2], b[V / 2];
        load_param<T, MODE>(p.weight, p.params_f32, v * V, min(V, width - v * V), 1.f, w);
        load_param<T, MODE>(p.bias, p.params_f32, v * V, min(V, width - v * V), 0.f, b);
#pragma unroll
        for (int k = 0; k < HALVES; ++k) {
            params[k * vecs + v] = make_float4(w[2 * k].x, w[2 * k].y, w[2 * k + 1].x, w[2 * k + 1].y);
            params[(HALVES + k) * vecs + v] = make_float4(b[2 * k].x, b[2 * k].y, b[2 * k + 1].x, b[2 * k + 1].y);
        }
    }
    if (t == 0) {
        for (int k = 0; k < ring.stages; ++k) mbar_init(full + k, 1);
        mbar_fence_init();
    }
    __syncthreads();

    const long long step = (long long)gridDim.x * groups;
    const T *x0 = static_cast<const T*>(p.x), *r0 = static_cast<const T*>(p.residual);
    const unsigned row_bytes = (unsigned)width * sizeof(T);
    auto misfit = [](const T* q) { return MODE == RAGGED ? (unsigned)(reinterpret_cast<uintptr_t>(q) & 15u) : 0u; };
    auto edge = [&](long long row) { return MODE == RAGGED && (row == 0 || row == p.rows - 1); };
    auto send = [&](long long row, int stage) {
        if (row >= p.rows) return;
        if (edge(row)) {
            mbar_arrive(full + stage);
            return;
        }
        unsigned char* to = mine + (size_t)stage * TENSORS * ring.slot_bytes;
        const T *px = x0 + row * p.x_pitch, *pr = r0 + row * p.res_pitch;
        const unsigned bx = MODE == RAGGED ? (misfit(px) + row_bytes + 15u) & ~15u : row_bytes;
        const unsigned br = !ADD ? 0u : MODE == RAGGED ? (misfit(pr) + row_bytes + 15u) & ~15u : row_bytes;
        mbar_expect_tx(full + stage, bx + br);
        bulk_load(to, reinterpret_cast<const unsigned char*>(px) - misfit(px), bx, full + stage);
        if (ADD) bulk_load(to + ring.slot_bytes, reinterpret_cast<const unsigned char*>(pr) - misfit(pr), br, full + stage);
    };
    long long row = (long long)blockIdx.x * groups + g;
    if (t == 0)
        for (int k = 0; k < ring.stages; ++k) send(row + k * step, k);
    auto meet = [&]() {
        if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "r"(group) : "memory");
        else __syncwarp();
    };
    long long at = row * p.width;
    const long long at_step = step * p.width;
    const unsigned long long seed = ADD && p.drop.on ? p.drop.seed_now() : 0;
    const unsigned long long drop_step = (unsigned long long)(at_step >> 1) * MAM_DROP_STEP;
    unsigned long long start = mam_drop_start(seed, at + vec0 * V);
    uint4 carry = make_uint4(0u, 0u, 0u, 0u);
    int stage = 0;
    unsigned phase = 0;
    bool lost = ring.late;
    if (lost) ring_late_call(p.wait, full, ring.stages, 0, 0, t == 0 ? ring.stages : 0, row, step, p.rows);
    for (; row < p.rows; row += step, at += at_step, start += drop_step) {
        unsigned char* from = mine + (size_t)stage * TENSORS * ring.slot_bytes;
        if (!lost && !mbar_wait_bounded(full + stage, phase, RING_POLLS)) {
            lost = true;
            ring_late_call(p.wait, full, ring.stages, stage, phase, t == 0 ? ring.stages : 0, row, step, p.rows);
        }
        unsigned skip_x = 0, skip_r = 0;
        if constexpr (MODE == RAGGED) {
            const T *px = x0 + row * p.x_pitch, *pr = r0 + row * p.res_pitch;
            skip_x = misfit(px);
            skip_r = misfit(pr);
            if (edge(row)) {
                T *dx = reinterpret_cast<T*>(from + skip_x), *dr = reinterpret_cast<T*>(from + ring.slot_bytes + skip_r);
                for (int c = t; c < width; c += group) {
                    dx[c] = px[c];
                    if (ADD) dr[c] = pr[c];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // before a later copy into this stage
                meet();
            }
            start = mam_drop_start(seed, at + vec0 * V);
        }
        const bool odd = MODE == RAGGED && ((at + vec0 * V) & 1);
        float2 v[NV][V / 2], s = splat2(0.f), d1 = s, d2 = s;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint4* q = reinterpret_cast<const uint4*>(from) + vec0 + i * 32;
            uint4 qx = make_uint4(0u, 0u, 0u, 0u);
            if (count(i) > 0) {
                if constexpr (MODE == RAGGED) qx = cut<T>(q[0], q[1], skip_x);
                else qx = *q;
                if constexpr (ADD) {
                    const uint4* k = reinterpret_cast<const uint4*>(from + ring.slot_bytes) + vec0 + i * 32;
                    uint4 qr;
                    if constexpr (MODE == RAGGED) qr = cut<T>(k[0], k[1], skip_r);
                    else qr = *k;
                    qx = add_residual<T>(qx, qr, p.drop, start + (unsigned long long)(i * 32 * (V / 2)) * MAM_DROP_STEP, odd);
                }
                unpack<T>(qx, v[i]);
                if (MODE == RAGGED && count(i) < V) keep_first<T>(v[i], count(i));
                s = add2(s, total<T>(v[i]));
            }
            if constexpr (ADD)
                store_vec<T, MODE>(static_cast<T*>(p.sum) + at + col(i), qx, MODE == FULL ? V : width - col(i), lane, 32, i == 0,
                                   i == NV - 1, carry);
        }
        float mu = lane_sum<32>(sum2(s));
        if (warps > 1 && lane == 0) slot[0][threadIdx.x >> 5].x = mu;
        meet();
        // all have this row in their registers
        if (t == 0 && !lost) send(row + ring.stages * step, stage);
        if (warps > 1) mu = lane_sum<MOST>(lane < warps ? slot[0][slot0 + lane].x : 0.f);
        mu *= p.inv_width;
        const float2 minus = splat2(-mu);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (count(i) > 0) {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) v[i][j] = add2(v[i][j], minus);
                if (MODE == RAGGED && count(i) < V) keep_first<T>(v[i], count(i));
#pragma unroll
                for (int j = 0; j < V / 2; ++j) d2 = fma2(v[i][j], v[i][j], d2);
                d1 = add2(d1, total<T>(v[i]));
            }
        float2 d = lane_sum2<32>(sum2(d1), sum2(d2));
        if (warps > 1) {
            if (lane == 0) slot[1][threadIdx.x >> 5] = d;
            meet();
            d = lane < warps ? slot[1][slot0 + lane] : make_float2(0.f, 0.f);
            d = lane_sum2<MOST>(d.x, d.y);
        }
        float off;
        const float2 st = row_stats(mu, d.x, d.y, p.inv_width, p.eps, off);
        if (p.stats && t == 0) p.stats[row] = st;
        const float2 r2 = splat2(st.y), o2 = splat2(-off);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (count(i) > 0) {
                Vals<T> y;
#pragma unroll
                for (int k = 0; k < HALVES; ++k) {
                    const float4 w = params[k * vecs + vec0 + i * 32], b = params[(HALVES + k) * vecs + vec0 + i * 32];
                    y[2 * k] = fma2(mul2(add2(v[i][2 * k], o2), r2), make_float2(w.x, w.y), make_float2(b.x, b.y));
                    y[2 * k + 1] = fma2(mul2(add2(v[i][2 * k + 1], o2), r2), make_float2(w.z, w.w), make_float2(b.z, b.w));
                }
                q = pack<T>(y);
            }
            store_vec<T, MODE>(static_cast<T*>(p.y) + at + col(i), q, MODE == FULL ? V : width - col(i), lane, 32, i == 0,
                               i == NV - 1, carry);
        }
        if (++stage == ring.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
}

// Rows of any width: one CTA a row, which reads it again for each of its steps (from L2 mostly).
template <typename T, bool ADD, int MODE>
__global__ void __launch_bounds__(1024) mam_norm_fwd_wide_kernel(const __grid_constant__ NormFwdParams p) {
    __shared__ float2 slot[64];
    constexpr int V = VEC<T>;
    const long long row = blockIdx.x, width = p.width, step = (long long)blockDim.x * V;
    const long long first = (long long)(threadIdx.x & ~31) * V;     // the warp's columns begin here: a loop for all its lanes
    const int lane = threadIdx.x & 31;
    const T* x0 = static_cast<const T*>(p.x);
    RowSrc<T, MODE> src(x0, p.x_pitch, p.rows, width, x0 + row * p.x_pitch);
    uint4 none;
    float2 s = splat2(0.f), d1 = s, d2 = s;
    auto count = [&](long long c) { return (int)min((long long)V, width - c); };
    if constexpr (ADD) {
        const T* r0 = static_cast<const T*>(p.residual);
        const RowSrc<T, MODE> r(r0, p.res_pitch, p.rows, width, r0 + row * p.res_pitch);
        const unsigned long long seed = p.drop.on ? p.drop.seed_now() : 0;
        for (long long c0 = first; c0 < width; c0 += step) {
            const long long c = c0 + lane * V, at = row * width + c;
            uint4 qs = make_uint4(0u, 0u, 0u, 0u);
            if (c < width) {
                qs = add_residual<T>(src.template load<false>(c, count(c)), r.load(c, count(c)), p.drop, mam_drop_start(seed, at),
                                     MODE == RAGGED && (at & 1));
                Vals<T> v;
                unpack<T>(qs, v);
                if (MODE == RAGGED && count(c) < V) keep_first<T>(v, count(c));
                s = add2(s, total<T>(v));
            }
            store_vec<T, MODE>(static_cast<T*>(p.sum) + at, qs, (int)min(width - c, (long long)2 * V), lane, 32, true, true,
                               none);
        }
        // read back behind the reduction's barrier
        const T* s0 = static_cast<const T*>(p.sum);
        src = RowSrc<T, MODE>(s0, width, p.rows, width, s0 + row * width);
    } else {
        for (long long c = first + lane * V; c < width; c += step) {
            Vals<T> v;
            unpack<T>(src.template load<false>(c, count(c)), v);
            if (MODE == RAGGED && count(c) < V) keep_first<T>(v, count(c));
            s = add2(s, total<T>(v));
        }
    }
    const float mu = row_sum<true, 32, 32>(sum2(s), reinterpret_cast<float*>(slot)) * p.inv_width;
    const float2 minus = splat2(-mu);
    for (long long c = first + lane * V; c < width; c += step) {
        Vals<T> v;
        unpack<T>(src.template load<false>(c, count(c)), v);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) v[j] = add2(v[j], minus);
        if (MODE == RAGGED && count(c) < V) keep_first<T>(v, count(c));
#pragma unroll
        for (int j = 0; j < V / 2; ++j) d2 = fma2(v[j], v[j], d2);
        d1 = add2(d1, total<T>(v));
    }
    const float2 d = row_sum2<true, 32, 32>(sum2(d1), sum2(d2), slot + 32);
    float off;
    const float2 st = row_stats(mu, d.x, d.y, p.inv_width, p.eps, off);
    if (p.stats && threadIdx.x == 0) p.stats[row] = st;
    const float2 r2 = splat2(st.y), o2 = splat2(-off);
    for (long long c0 = first; c0 < width; c0 += step) {
        const long long c = c0 + lane * V;
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (c < width) {
            Vals<T> v, w, b;
            unpack<T>(src.template load<false>(c, count(c)), v);
            load_param<T, MODE>(p.weight, p.params_f32, (int)c, count(c), 1.f, w);
            load_param<T, MODE>(p.bias, p.params_f32, (int)c, count(c), 0.f, b);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) w[j] = fma2(mul2(add2(add2(v[j], minus), o2), r2), w[j], b[j]);
            q = pack<T>(w);
        }
        store_vec<T, MODE>(static_cast<T*>(p.y) + row * width + c, q, (int)min(width - c, (long long)2 * V), lane, 32, true, true,
                           none);
    }
}

// Backward of narrow rows, of up to LANES (8 or 16) times NV vectors: 512 / LANES rows at a time in a CTA.  A thread keeps its
// columns' sums of gy h and gy in registers over all its rows, and the CTA leaves one partial row of each.  The next row's
// vectors are on their way while a row is reduced.
template <typename T, int NV, bool ADD, int MODE, int LANES>
__global__ void __launch_bounds__(512) mam_norm_bwd_narrow_kernel(const __grid_constant__ NormBwdParams p) {
    extern __shared__ float cols[];    // [warps][2][width] at the end
    constexpr int V = VEC<T>;
    const int g = threadIdx.x / LANES, t = threadIdx.x % LANES, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int width = (int)p.width, first = t * V;
    auto col = [&](int i) { return first + i * LANES * V; };
    auto count = [&](int i) { return min(V, width - col(i)); };
    uint4 carry = make_uint4(0u, 0u, 0u, 0u), carry2 = carry;
    float2 w[NV][V / 2], aw[NV][V / 2], ab[NV][V / 2];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (count(i) > 0) load_param<T, MODE>(p.weight, p.params_f32, col(i), count(i), 1.f, w[i]);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) aw[i][j] = ab[i][j] = splat2(0.f);
    }
    const float inv_n = p.inv_width;
    const int groups = 512 / LANES, g0 = warp * (32 / LANES);      // the rows of a warp keep step
    const long long step = (long long)gridDim.x * groups;
    const bool has_gy = p.gy != nullptr, has_gs = ADD && p.gs != nullptr, has_dx = ADD && p.dx != nullptr;
    const T *s0 = static_cast<const T*>(p.s), *gy0 = static_cast<const T*>(p.gy), *gs0 = static_cast<const T*>(p.gs);
    // the row that is fetched: its pointer into s, its place in the contiguous tensors
    long long base = (long long)blockIdx.x * groups + g0, ahead = base + (g - g0), at = ahead * p.width;
    const T* ps = s0 + ahead * p.s_pitch;
    const long long s_step = step * p.s_pitch, at_step = step * p.width;
    const unsigned long long seed = has_dx ? p.drop.seed_now() : 0, drop_step = (unsigned long long)(at_step >> 1) * MAM_DROP_STEP;
    unsigned long long start = mam_drop_start(seed, at + first);
    uint4 qs[NV], qg[NV];
    float2 st = make_float2(0.f, 0.f);
    auto fetch = [&]() {
        if (ahead >= p.rows) return;
        const RowSrc<T, MODE> s(s0, p.s_pitch, p.rows, p.width, ps), y(gy0, p.width, p.rows, p.width, gy0 + at);
        st = p.stats[ahead];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (count(i) > 0) qs[i] = s.load(col(i), count(i));
        if (has_gy)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (count(i) > 0) qg[i] = y.load(col(i), count(i));
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) qg[i] = make_uint4(0u, 0u, 0u, 0u);
    fetch();
    for (; base < p.rows; base += step) {
        const bool valid = ahead < p.rows;
        const long long row_at = at;
        const float2 minus = splat2(-st.x), r2 = splat2(st.y);    // (s - mu) r in this order: exact where s is near mu
        const float rstd = st.y;
        float2 h[NV][V / 2], a[NV][V / 2];
        uint4 ga[NV];
        float2 s1 = splat2(0.f), s2 = s1;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (valid && count(i) > 0) {
                unpack<T>(qs[i], h[i]);
                unpack<T>(qg[i], a[i]);
            }
        if (has_gs && valid) {
            const RowSrc<T, MODE> z(gs0, p.width, p.rows, p.width, gs0 + row_at);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (count(i) > 0) ga[i] = z.load(col(i), count(i));
        }
        ahead += step;
        at += at_step;
        ps += s_step;
        fetch();
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (valid && count(i) > 0) {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) h[i][j] = mul2(add2(h[i][j], minus), r2);
                if (MODE == RAGGED && count(i) < V) {
                    keep_first<T>(h[i], count(i));
                    keep_first<T>(a[i], count(i));
                }
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    aw[i][j] = fma2(a[i][j], h[i][j], aw[i][j]);
                    ab[i][j] = add2(ab[i][j], a[i][j]);
                    a[i][j] = mul2(a[i][j], w[i][j]);
                    s1 = add2(s1, a[i][j]);
                    s2 = fma2(a[i][j], h[i][j], s2);
                }
            }
        const float2 m = lane_sum2<LANES>(sum2(s1), sum2(s2));
        // ds = r a - (r mean(a) + h r mean(a h))
        const float2 c1 = splat2(-rstd * (m.x * inv_n)), c2 = splat2(-rstd * (m.y * inv_n));
        const bool odd = MODE == RAGGED && ((row_at + first) & 1);
        if (MODE == RAGGED) start = mam_drop_start(seed, row_at + first);
        T *ds = static_cast<T*>(p.ds) + row_at, *dx = static_cast<T*>(p.dx) + row_at;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int rest = valid ? width - col(i) : 0;
            uint4 q = make_uint4(0u, 0u, 0u, 0u), qd = q;
            if (rest > 0) {
                Vals<T> d;
#pragma unroll
                for (int j = 0; j < V / 2; ++j) d[j] = fma2(a[i][j], r2, fma2(h[i][j], c2, c1));
                if constexpr (ADD) {
                    if (has_gs) {
                        Vals<T> f;
                        unpack<T>(ga[i], f);
#pragma unroll
                        for (int j = 0; j < V / 2; ++j) d[j] = add2(d[j], f[j]);
                    }
                }
                q = pack<T>(d);
                if constexpr (ADD) {
                    if (has_dx) {
                        mam_drop_pairs<V / 2>(d, start + (unsigned long long)(i * LANES * (V / 2)) * MAM_DROP_STEP, odd,
                                              p.drop.threshold, p.drop.scale);
                        qd = pack<T>(d);
                    }
                }
            }
            store_vec<T, MODE>(ds + col(i), q, rest, t, LANES, i == 0, i == NV - 1, carry);
            if constexpr (ADD) {
                if (has_dx) store_vec<T, MODE>(dx + col(i), qd, rest, t, LANES, i == 0, i == NV - 1, carry2);
            }
        }
        start += drop_step;
    }
    if (!p.partial) return;
    float* out = p.partial + (long long)blockIdx.x * 2 * p.width;
    // the rows of a warp are added by shuffles, the warps in shared memory: a fixed order
    float* to = cols + (size_t)warp * 2 * width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[2][V];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            split2(aw[i][j], f[0][2 * j], f[0][2 * j + 1]);
            split2(ab[i][j], f[1][2 * j], f[1][2 * j + 1]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (LANES == 8) f[k][j] += __shfl_xor_sync(~0u, f[k][j], 8);
                f[k][j] += __shfl_xor_sync(~0u, f[k][j], 16);
                if (col(i) + j < width && lane < LANES) to[k * width + col(i) + j] = f[k][j];
            }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * width; c += 512) {
        float sum = cols[c];
#pragma unroll
        for (int k = 1; k < 16; ++k) sum += cols[(size_t)k * 2 * width + c];
        out[c] = sum;
    }
}

// The same for rows from a warp's width on, with the rows brought to shared memory by bulk copies: `stages` rows of each group
// of `group` threads (whole warps) are there or on their way, whatever the registers leave room for.  With the next row's
// vectors in registers instead, bf16 [32768, 4096] took 155 us (this: 130) and with dropout 336 (211).
// A row's stage is free when its group has passed the next row's barrier; thread 0 of the group then sends for the row
// `stages - 1` ahead.
template <typename T, int NV, bool ADD, int MODE>
__global__ void __launch_bounds__(NV * VEC<T> == 8 ? 640 : NV * VEC<T> == 24 ? 384 : 512)
mam_norm_bwd_ring_kernel(const __grid_constant__ NormBwdParams p, const __grid_constant__ NormRing ring) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 slot[2][32];
    constexpr int V = VEC<T>, HALVES = V / 4, TENSORS = ADD ? 3 : 2, MOST = NV * V == 8 ? 32 : 16;      // warps a group can have
    const int group = ring.group, groups = ring.groups, g = threadIdx.x / group, t = threadIdx.x - g * group;
    const int lane = threadIdx.x & 31, warps = group >> 5, slot0 = (g * group) >> 5;
    const int width = (int)p.width;
    const int vec0 = (t >> 5) * NV * 32 + lane;     // a warp's vectors follow one another
    auto col = [&](int i) { return (vec0 + i * 32) * V; };
    auto live = [&](int i) { return MODE == FULL || col(i) < width; };
    const bool has_gy = p.gy != nullptr, has_gs = ADD && p.gs != nullptr, has_dx = ADD && p.dx != nullptr;
    const int tensors = 1 + has_gy + has_gs;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring.bars_at) + g * ring.stages;
    unsigned char* mine = smem + (size_t)g * ring.stages * TENSORS * ring.slot_bytes;      // [stage][s, gy, gs][row]
    // the weight in fp32, the halves of a vector of eight apart: a warp's 16-byte reads then meet no bank twice
    float4* weights = reinterpret_cast<float4*>(smem + ring.weights_at);
    const int vecs = (width + V - 1) / V;
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
        float2 w[V / 2];
        load_param<T, ALIGNED>(p.weight, p.params_f32, v * V, V, 1.f, w);
#pragma unroll
        for (int k = 0; k < HALVES; ++k)
            weights[k * vecs + v] = make_float4(w[2 * k].x, w[2 * k].y, w[2 * k + 1].x, w[2 * k + 1].y);
    }
    if (t == 0) {
        for (int k = 0; k < ring.stages; ++k) mbar_init(full + k, 1);
        mbar_fence_init();
    }
    __syncthreads();

    const long long step = (long long)gridDim.x * groups;
    const T *s0 = static_cast<const T*>(p.s), *gy0 = static_cast<const T*>(p.gy), *gs0 = static_cast<const T*>(p.gs);
    auto send = [&](long long row, int stage) {
        if (row >= p.rows) return;
        unsigned char* to = mine + (size_t)stage * TENSORS * ring.slot_bytes;
        mbar_expect_tx(full + stage, tensors * ring.slot_bytes);
        bulk_load(to, s0 + row * p.s_pitch, ring.slot_bytes, full + stage);
        if (has_gy) bulk_load(to + ring.slot_bytes, gy0 + row * p.width, ring.slot_bytes, full + stage);
        if (has_gs) bulk_load(to + 2 * ring.slot_bytes, gs0 + row * p.width, ring.slot_bytes, full + stage);
    };
    long long row = (long long)blockIdx.x * groups + g;
    if (t == 0)
        for (int k = 0; k < ring.stages - 1; ++k) send(row + k * step, k);

    float2 aw[NV][V / 2], ab[NV][V / 2];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V / 2; ++j) aw[i][j] = ab[i][j] = splat2(0.f);
    const float inv_n = p.inv_width;
    long long at = row * p.width;
    const long long at_step = step * p.width;
    const unsigned long long drop_step = (unsigned long long)(at_step >> 1) * MAM_DROP_STEP;
    unsigned long long start = has_dx ? mam_drop_start(p.drop.seed_now(), at + vec0 * V) : 0;
    float2 next = row < p.rows ? p.stats[row] : make_float2(0.f, 0.f);
    int stage = 0;
    unsigned phase = 0, parity = 0;
    bool lost = ring.late;
    if (lost) ring_late(p.wait, full, ring.stages, 0, 0, t == 0 ? ring.stages - 1 : 0, row, step, p.rows);
    for (; row < p.rows; row += step, at += at_step, start += drop_step) {
        const float2 st = next;
        if (row + step < p.rows) next = p.stats[row + step];
        const float2 minus = splat2(-st.x), r2 = splat2(st.y);    // (s - mu) r in this order: exact where s is near mu
        const unsigned char* from = mine + (size_t)stage * TENSORS * ring.slot_bytes;
        if (!lost && !mbar_wait_bounded(full + stage, phase, RING_POLLS)) {
            lost = true;
            ring_late(p.wait, full, ring.stages, stage, phase, t == 0 ? ring.stages - 1 : 0, row, step, p.rows);
        }
        float2 h[NV][V / 2], a[NV][V / 2], s1 = splat2(0.f), s2 = s1;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
                const uint4* q = reinterpret_cast<const uint4*>(from) + vec0 + i * 32;
                unpack<T>(*q, h[i]);
                if (has_gy) {
                    unpack<T>(*reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(q) + ring.slot_bytes), a[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) a[i][j] = splat2(0.f);
                }
                float2 w[V / 2];
#pragma unroll
                for (int k = 0; k < HALVES; ++k) {
                    const float4 f = weights[k * vecs + vec0 + i * 32];
                    w[2 * k] = make_float2(f.x, f.y);
                    w[2 * k + 1] = make_float2(f.z, f.w);
                }
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    h[i][j] = mul2(add2(h[i][j], minus), r2);
                    aw[i][j] = fma2(a[i][j], h[i][j], aw[i][j]);
                    ab[i][j] = add2(ab[i][j], a[i][j]);
                    a[i][j] = mul2(a[i][j], w[j]);
                    s1 = add2(s1, a[i][j]);
                    s2 = fma2(a[i][j], h[i][j], s2);
                }
            }
        float2 m = lane_sum2<32>(sum2(s1), sum2(s2));
        if (warps > 1) {
            // two sets of slots in turn: a set is written again only behind the next row's barrier
            if (lane == 0) slot[parity][threadIdx.x >> 5] = m;
            asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "r"(group) : "memory");
        } else {
            __syncwarp();
        }
        // all have left the row before this one: its stage takes the row stages - 1 ahead
        if (t == 0 && !lost) send(row + (ring.stages - 1) * step, stage == 0 ? ring.stages - 1 : stage - 1);
        if (warps > 1) {
            m = (lane & (MOST - 1)) < warps ? slot[parity][slot0 + (lane & (MOST - 1))] : make_float2(0.f, 0.f);
            m = lane_sum2<MOST>(m.x, m.y);
            parity ^= 1;
        }
        // ds = r a - (r mean(a) + h r mean(a h))
        const float2 c1 = splat2(-st.y * (m.x * inv_n)), c2 = splat2(-st.y * (m.y * inv_n));
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live(i)) {
                Vals<T> d;
#pragma unroll
                for (int j = 0; j < V / 2; ++j) d[j] = fma2(a[i][j], r2, fma2(h[i][j], c2, c1));
                if constexpr (ADD) {
                    if (has_gs) {
                        Vals<T> f;
                        unpack<T>(*(reinterpret_cast<const uint4*>(from + 2 * ring.slot_bytes) + vec0 + i * 32), f);
#pragma unroll
                        for (int j = 0; j < V / 2; ++j) d[j] = add2(d[j], f[j]);
                    }
                }
                *reinterpret_cast<uint4*>(static_cast<T*>(p.ds) + at + col(i)) = pack<T>(d);
                if constexpr (ADD) {
                    if (has_dx) {
                        mam_drop_pairs<V / 2>(d, start + (unsigned long long)(i * 32 * (V / 2)) * MAM_DROP_STEP, false,
                                              p.drop.threshold, p.drop.scale);
                        *reinterpret_cast<uint4*>(static_cast<T*>(p.dx) + at + col(i)) = pack<T>(d);
                    }
                }
            }
        if (++stage == ring.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (!p.partial) return;
    float* out = p.partial + (long long)blockIdx.x * 2 * p.width;
    // the groups' sums meet in the ring's memory, where no copy is on its way any more (unless a wait ran out): a fixed order
    if (__syncthreads_or(lost)) return;
    float* cols = reinterpret_cast<float*>(smem);
    float* to = groups > 1 ? cols + (size_t)g * 2 * width : out;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (live(i)) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                *reinterpret_cast<float2*>(to + col(i) + 2 * j) = aw[i][j];
                *reinterpret_cast<float2*>(to + width + col(i) + 2 * j) = ab[i][j];
            }
        }
    if (groups == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * width; c += blockDim.x) {
        float sum = cols[c];
        for (int k = 1; k < groups; ++k) sum += cols[(size_t)k * 2 * width + c];
        out[c] = sum;
    }
}

// The ring for rows that are not 16-byte aligned.  They are copied with the aligned 16 bytes at either end, which belong to
// the rows beside them; the first and the last row have no such neighbours and are brought element by element.  A thread
// shifts its vectors out of two aligned ones, and the stores take the way of ragged rows.  (A kernel of its own: as one
// template the aligned form lost 3 to 8 %.)  bf16 [5003, 1283] 25 us, with the next row's vectors in registers instead 40.
template <typename T, int NV, bool ADD>
__global__ void __launch_bounds__(NV * VEC<T> == 8 ? 640 : NV * VEC<T> == 24 ? 384 : 512)
mam_norm_bwd_ragged_kernel(const __grid_constant__ NormBwdParams p, const __grid_constant__ NormRing ring) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 slot[2][32];
    constexpr int V = VEC<T>, HALVES = V / 4, TENSORS = ADD ? 3 : 2, MOST = NV * V == 8 ? 32 : 16;      // warps a group can have
    const int group = ring.group, groups = ring.groups, g = threadIdx.x / group, t = threadIdx.x - g * group;
    const int lane = threadIdx.x & 31, warps = group >> 5, slot0 = (g * group) >> 5;
    const int width = (int)p.width;
    const int vec0 = (t >> 5) * NV * 32 + lane;     // a warp's vectors follow one another
    auto col = [&](int i) { return (vec0 + i * 32) * V; };
    auto count = [&](int i) { return min(V, width - col(i)); };
    const bool has_gy = p.gy != nullptr, has_gs = ADD && p.gs != nullptr, has_dx = ADD && p.dx != nullptr;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring.bars_at) + g * ring.stages;
    unsigned char* mine = smem + (size_t)g * ring.stages * TENSORS * ring.slot_bytes;      // [stage][s, gy, gs][row]
    // the weight in fp32, the halves of a vector of eight apart: a warp's 16-byte reads then meet no bank twice
    float4* weights = reinterpret_cast<float4*>(smem + ring.weights_at);
    const int vecs = (width + V - 1) / V;
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
        float2 w[V / 2];
        load_param<T, RAGGED>(p.weight, p.params_f32, v * V, min(V, width - v * V), 1.f, w);
#pragma unroll
        for (int k = 0; k < HALVES; ++k)
            weights[k * vecs + v] = make_float4(w[2 * k].x, w[2 * k].y, w[2 * k + 1].x, w[2 * k + 1].y);
    }
    if (t == 0) {
        for (int k = 0; k < ring.stages; ++k) mbar_init(full + k, 1);
        mbar_fence_init();
    }
    __syncthreads();

    const long long step = (long long)gridDim.x * groups;
    const T *s0 = static_cast<const T*>(p.s), *gy0 = static_cast<const T*>(p.gy), *gs0 = static_cast<const T*>(p.gs);
    const unsigned row_bytes = (unsigned)width * sizeof(T);
    auto misfit = [](const T* q) { return (unsigned)(reinterpret_cast<uintptr_t>(q) & 15u); };
    auto edge = [&](long long row) { return row == 0 || row == p.rows - 1; };
    auto send = [&](long long row, int stage) {
        if (row >= p.rows) return;
        if (edge(row)) {
            mbar_arrive(full + stage);
            return;
        }
        unsigned char* to = mine + (size_t)stage * TENSORS * ring.slot_bytes;
        const T* from[3] = {s0 + row * p.s_pitch, gy0 + row * p.width, gs0 + row * p.width};
        const bool has[3] = {true, has_gy, has_gs};
        unsigned bytes[3], all = 0;
#pragma unroll
        for (int k = 0; k < TENSORS; ++k) {
            bytes[k] = (misfit(from[k]) + row_bytes + 15u) & ~15u;
            if (has[k]) all += bytes[k];
        }
        mbar_expect_tx(full + stage, all);
#pragma unroll
        for (int k = 0; k < TENSORS; ++k)
            if (has[k])
                bulk_load(to + k * ring.slot_bytes, reinterpret_cast<const unsigned char*>(from[k]) - misfit(from[k]), bytes[k],
                          full + stage);
    };
    long long row = (long long)blockIdx.x * groups + g;
    if (t == 0)
        for (int k = 0; k < ring.stages - 1; ++k) send(row + k * step, k);

    float2 aw[NV][V / 2], ab[NV][V / 2];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V / 2; ++j) aw[i][j] = ab[i][j] = splat2(0.f);
    const float inv_n = p.inv_width;
    long long at = row * p.width;
    const long long at_step = step * p.width;
    const unsigned long long seed = has_dx ? p.drop.seed_now() : 0;
    float2 next = row < p.rows ? p.stats[row] : make_float2(0.f, 0.f);
    uint4 carry = make_uint4(0u, 0u, 0u, 0u), carry2 = carry;
    int stage = 0;
    unsigned phase = 0, parity = 0;
    bool lost = ring.late;
    if (lost) ring_late(p.wait, full, ring.stages, 0, 0, t == 0 ? ring.stages - 1 : 0, row, step, p.rows);
    auto meet = [&]() {
        if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "r"(group) : "memory");
        else __syncwarp();
    };
    for (; row < p.rows; row += step, at += at_step) {
        const float2 st = next;
        if (row + step < p.rows) next = p.stats[row + step];
        const float2 minus = splat2(-st.x), r2 = splat2(st.y);    // (s - mu) r in this order: exact where s is near mu
        unsigned char* from = mine + (size_t)stage * TENSORS * ring.slot_bytes;
        if (!lost && !mbar_wait_bounded(full + stage, phase, RING_POLLS)) {
            lost = true;
            ring_late(p.wait, full, ring.stages, stage, phase, t == 0 ? ring.stages - 1 : 0, row, step, p.rows);
        }
        const T *ps = s0 + row * p.s_pitch, *py = gy0 + at, *pz = gs0 + at;
        if (edge(row)) {
            T *ds = reinterpret_cast<T*>(from + misfit(ps)), *dy = reinterpret_cast<T*>(from + ring.slot_bytes + misfit(py)),
              *dz = reinterpret_cast<T*>(from + 2 * ring.slot_bytes + misfit(pz));
            for (int c = t; c < width; c += group) {
                ds[c] = ps[c];
                if (has_gy) dy[c] = py[c];
                if (has_gs) dz[c] = pz[c];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // before a later copy into this stage
            meet();
        }
        auto vector = [&](int tensor, const T* src, int i) {
            const uint4* q = reinterpret_cast<const uint4*>(from + tensor * ring.slot_bytes) + vec0 + i * 32;
            return cut<T>(q[0], q[1], misfit(src));
        };
        float2 h[NV][V / 2], a[NV][V / 2], s1 = splat2(0.f), s2 = s1;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (count(i) > 0) {
                unpack<T>(vector(0, ps, i), h[i]);
                if (has_gy) {
                    unpack<T>(vector(1, py, i), a[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) a[i][j] = splat2(0.f);
                }
                float2 w[V / 2];
#pragma unroll
                for (int k = 0; k < HALVES; ++k) {
                    const float4 f = weights[k * vecs + vec0 + i * 32];
                    w[2 * k] = make_float2(f.x, f.y);
                    w[2 * k + 1] = make_float2(f.z, f.w);
                }
                if (count(i) < V) {
                    keep_first<T>(h[i], count(i));
                    keep_first<T>(a[i], count(i));
                }
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    h[i][j] = mul2(add2(h[i][j], minus), r2);
                    aw[i][j] = fma2(a[i][j], h[i][j], aw[i][j]);
                    ab[i][j] = add2(ab[i][j], a[i][j]);
                    a[i][j] = mul2(a[i][j], w[j]);
                    s1 = add2(s1, a[i][j]);
                    s2 = fma2(a[i][j], h[i][j], s2);
                }
            }
        float2 m = lane_sum2<32>(sum2(s1), sum2(s2));
        // two sets of slots in turn: a set is written again only behind the next row's barrier
        if (warps > 1 && lane == 0) slot[parity][threadIdx.x >> 5] = m;
        meet();
        // all have left the row before this one: its stage takes the row stages - 1 ahead
        if (t == 0 && !lost) send(row + (ring.stages - 1) * step, stage == 0 ? ring.stages - 1 : stage - 1);
        if (warps > 1) {
            m = (lane & (MOST - 1)) < warps ? slot[parity][slot0 + (lane & (MOST - 1))] : make_float2(0.f, 0.f);
            m = lane_sum2<MOST>(m.x, m.y);
            parity ^= 1;
        }
        // ds = r a - (r mean(a) + h r mean(a h))
        const float2 c1 = splat2(-st.y * (m.x * inv_n)), c2 = splat2(-st.y * (m.y * inv_n));
        const unsigned long long start = mam_drop_start(seed, at + vec0 * V);
        const bool odd = (at + vec0 * V) & 1;
        T *ds = static_cast<T*>(p.ds) + at, *dx = static_cast<T*>(p.dx) + at;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint4 q = make_uint4(0u, 0u, 0u, 0u), qd = q;
            if (count(i) > 0) {
                Vals<T> d;
#pragma unroll
                for (int j = 0; j < V / 2; ++j) d[j] = fma2(a[i][j], r2, fma2(h[i][j], c2, c1));
                if constexpr (ADD) {
                    if (has_gs) {
                        Vals<T> f;
                        unpack<T>(vector(2, pz, i), f);
#pragma unroll
                        for (int j = 0; j < V / 2; ++j) d[j] = add2(d[j], f[j]);
                    }
                }
                q = pack<T>(d);
                if constexpr (ADD) {
                    if (has_dx) {
                        mam_drop_pairs<V / 2>(d, start + (unsigned long long)(i * 32 * (V / 2)) * MAM_DROP_STEP, odd,
                                              p.drop.threshold, p.drop.scale);
                        qd = pack<T>(d);
                    }
                }
            }
            const int rest = width - col(i);
            store_vec<T, RAGGED>(ds + col(i), q, rest, lane, 32, i == 0, i == NV - 1, carry);
            if constexpr (ADD) {
                if (has_dx) store_vec<T, RAGGED>(dx + col(i), qd, rest, lane, 32, i == 0, i == NV - 1, carry2);
            }
        }
        if (++stage == ring.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (!p.partial) return;
    float* out = p.partial + (long long)blockIdx.x * 2 * p.width;
    // the groups' sums meet in the ring's memory, where no copy is on its way any more (unless a wait ran out): a fixed order
    if (__syncthreads_or(lost)) return;
    float* cols = reinterpret_cast<float*>(smem);
    float* to = groups > 1 ? cols + (size_t)g * 2 * width : out;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (col(i) + j < width) {
                to[col(i) + j] = j & 1 ? aw[i][j / 2].y : aw[i][j / 2].x;
                to[width + col(i) + j] = j & 1 ? ab[i][j / 2].y : ab[i][j / 2].x;
            }
    if (groups == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * width; c += blockDim.x) {
        float sum = cols[c];
        for (int k = 1; k < groups; ++k) sum += cols[(size_t)k * 2 * width + c];
        out[c] = sum;
    }
}

// Backward of rows of any width: gradients of the rows, one CTA a row, without the columns' sums.  NV > 0: the row's vectors,
// NV a thread, stay in registers as they were read; 0: they are read again.
template <typename T, int NV, bool ADD, int MODE>
__global__ void __launch_bounds__(1024) mam_norm_bwd_wide_kernel(const __grid_constant__ NormBwdParams p) {
    __shared__ float2 slot[32];
    constexpr int V = VEC<T>, KEPT = NV > 0 ? NV : 1;
    const long long row = blockIdx.x, width = p.width, step = (long long)blockDim.x * V;
    const long long first = (long long)(threadIdx.x & ~31) * V;
    const int lane = threadIdx.x & 31;
    const T *s0 = static_cast<const T*>(p.s), *gy0 = static_cast<const T*>(p.gy), *gs0 = static_cast<const T*>(p.gs);
    const RowSrc<T, MODE> s(s0, p.s_pitch, p.rows, width, s0 + row * p.s_pitch),
        gy(gy0, width, p.rows, width, gy0 + row * width), gs(gs0, width, p.rows, width, gs0 + row * width);
    uint4 none, qs[KEPT], qg[KEPT];
    const float2 st = p.stats[row];
    const float2 minus = splat2(-st.x), r2 = splat2(st.y);    // (s - mu) r in this order: exact where s is near mu
    const unsigned long long seed = ADD && p.drop.on ? p.drop.seed_now() : 0;
    auto count = [&](long long c) { return (int)min((long long)V, width - c); };
    auto get = [&](long long c, int i) {
        qs[i] = s.load(c, count(c));
        qg[i] = p.gy ? gy.load(c, count(c)) : make_uint4(0u, 0u, 0u, 0u);
    };
    // normalised values and weighted gradients of the vector at c
    auto values = [&](long long c, int i, Vals<T>& h, Vals<T>& a) {
        Vals<T> w;
        unpack<T>(qs[i], h);
        unpack<T>(qg[i], a);
        load_param<T, MODE>(p.weight, p.params_f32, (int)c, count(c), 1.f, w);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            h[j] = mul2(add2(h[j], minus), r2);
            a[j] = mul2(a[j], w[j]);
        }
        if (MODE == RAGGED && count(c) < V) {
            keep_first<T>(h, count(c));
            keep_first<T>(a, count(c));
        }
    };
    float2 s1 = splat2(0.f), s2 = s1;
    auto add = [&](long long c, int i) {
        Vals<T> h, a;
        values(c, i, h, a);
        s1 = add2(s1, total<T>(a));
#pragma unroll
        for (int j = 0; j < V / 2; ++j) s2 = fma2(a[j], h[j], s2);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + lane * V + i * step < width) get(first + lane * V + i * step, i);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + lane * V + i * step < width) add(first + lane * V + i * step, i);
    } else if (p.gy) {
        for (long long c = first + lane * V; c < width; c += step) {
            get(c, 0);
            add(c, 0);
        }
    }
    const float2 m = row_sum2<true, 32, 32>(sum2(s1), sum2(s2), slot);
    const float2 c1 = splat2(-st.y * (m.x * p.inv_width)), c2 = splat2(-st.y * (m.y * p.inv_width));
    auto finish = [&](long long c, int i) {
        const long long at = row * width + c;
        const int rest = (int)min(width - c, (long long)2 * V);
        uint4 q = make_uint4(0u, 0u, 0u, 0u), qd = q;
        if (rest > 0) {
            Vals<T> h, a;
            values(c, i, h, a);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) a[j] = fma2(a[j], r2, fma2(h[j], c2, c1));
            if constexpr (ADD) {
                if (p.gs) {
                    unpack<T>(gs.load(c, count(c)), h);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) a[j] = add2(a[j], h[j]);
                }
            }
            q = pack<T>(a);
            if constexpr (ADD) {
                if (p.dx) {
                    mam_drop_pairs<V / 2>(a, mam_drop_start(seed, at), MODE == RAGGED && (at & 1), p.drop.threshold,
                                          p.drop.scale);
                    qd = pack<T>(a);
                }
            }
        }
        store_vec<T, MODE>(static_cast<T*>(p.ds) + at, q, rest, lane, 32, true, true, none);
        if constexpr (ADD) {
            if (p.dx) store_vec<T, MODE>(static_cast<T*>(p.dx) + at, qd, rest, lane, 32, true, true, none);
        }
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + i * step < width) finish(first + lane * V + i * step, i);
    } else {
        for (long long c0 = first; c0 < width; c0 += step) {
            const long long c = c0 + lane * V;
            if (c < width) get(c, 0);
            finish(c, 0);
        }
    }
}

constexpr int NORM_COLS = 32, NORM_LANES = 8;

// The columns' sums of gy h and gy over slabs of rows, for rows wider than a CTA's registers hold: grid (groups of 32
// vectors, slabs), into partial[slab][2][width].  Column by column it read 64 bytes of a row at a time and took longer than
// the rows' own kernel.
template <typename T, int MODE>
__global__ void __launch_bounds__(NORM_COLS * NORM_LANES, 4)
mam_norm_bwd_cols_kernel(const __grid_constant__ NormBwdParams p, long long rows_per) {
    constexpr int V = VEC<T>;
    __shared__ float part[NORM_LANES][2][NORM_COLS * V];
    const int lane = threadIdx.x % NORM_COLS, l = threadIdx.x / NORM_COLS;
    const long long c = ((long long)blockIdx.x * NORM_COLS + lane) * V;
    const long long m0 = (long long)blockIdx.y * rows_per, m1 = min(m0 + rows_per, p.rows);
    const int n = (int)min((long long)V, p.width - c);
    const T *s0 = static_cast<const T*>(p.s), *gy0 = static_cast<const T*>(p.gy);
    float2 aw[V / 2], ab[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) aw[j] = ab[j] = splat2(0.f);
    if (n > 0 && gy0)
#pragma unroll 4
        for (long long m = m0 + l; m < m1; m += NORM_LANES) {
            const RowSrc<T, MODE> s(s0, p.s_pitch, p.rows, p.width, s0 + m * p.s_pitch),
                gy(gy0, p.width, p.rows, p.width, gy0 + m * p.width);
            const uint4 qs = s.load(c, n), qg = gy.load(c, n);
            const float2 st = p.stats[m];
            Vals<T> h, a;
            unpack<T>(qs, h);
            unpack<T>(qg, a);
            const float2 minus = splat2(-st.x), r2 = splat2(st.y);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                aw[j] = fma2(a[j], mul2(add2(h[j], minus), r2), aw[j]);
                ab[j] = add2(ab[j], a[j]);
            }
        }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
        *reinterpret_cast<float2*>(&part[l][0][lane * V + 2 * j]) = aw[j];
        *reinterpret_cast<float2*>(&part[l][1][lane * V + 2 * j]) = ab[j];
    }
    __syncthreads();
    float* out = p.partial + (long long)blockIdx.y * 2 * p.width;
    for (int k = threadIdx.x; k < 2 * NORM_COLS * V; k += NORM_COLS * NORM_LANES) {
        const int which = k / (NORM_COLS * V), at = k % (NORM_COLS * V);
        const long long to = (long long)blockIdx.x * NORM_COLS * V + at;
        if (to >= p.width) continue;      // what lies behind a row's end is not a number to be had
        float sum = part[0][which][at];
#pragma unroll
        for (int i = 1; i < NORM_LANES; ++i) sum += part[i][which][at];
        out[which * p.width + to] = sum;
    }
}

// dw and db: the partial rows added in a fixed order, rounded once to the parameters' type.  Bound by the latency of its
// loads: eight rows at a time in a CTA, eight of them in flight a thread.  Its launch depends programmatically on the kernel
// before it, which has no early trigger: it starts when that kernel's last CTA has ended and waits here for its partial
// rows.  What that saves is a part of the gap between two launches: [12608, 768] fp32 25.5 us for 26.2, [8192, 2048] bf16 nothing.
template <typename T>
__global__ void __launch_bounds__(NORM_COLS * NORM_LANES)
mam_norm_params_kernel(const float* partial, void* dweight, void* dbias, long long parts, long long width,
                       bool params_f32) {
    __shared__ float part[NORM_LANES][NORM_COLS];
    const int c = threadIdx.x % NORM_COLS, l = threadIdx.x / NORM_COLS;
    const long long n = (long long)blockIdx.x * NORM_COLS + c;      // 0 .. 2 * width - 1: weight, then bias
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < 2 * width)
        for (long long m = l; m < parts; m += 8 * NORM_LANES)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (m + i * NORM_LANES < parts) s[i] += __ldcg(partial + (m + i * NORM_LANES) * 2 * width + n);
    part[l][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (l != 0 || n >= 2 * width) return;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < NORM_LANES; ++i) v += part[i][c];
    void* out = n < width ? dweight : dbias;
    if (!out) return;
    const long long k = n < width ? n : n - width;
    if (params_f32) static_cast<float*>(out)[k] = v;
    else static_cast<T*>(out)[k] = from_f32<T>(v);
}

}  // namespace mamb200
