// C ABI of the operators between the MAM layers of a transformer block: layer norm, dropout with residual addition, GELU.
// Declarations are in include/mam_b200.h.
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/mam_b200.h"
#include "mam_host.cuh"
#include "mam_norm.cuh"
#include "mam_pointwise.cuh"

using namespace mamb200;

namespace {

bool dtype_ok(int dtype) { return dtype == MAM_F32 || dtype == MAM_F16 || dtype == MAM_BF16; }
int dtype_size(int dtype) { return dtype == MAM_F32 ? 4 : 2; }
bool natural(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (unsigned)(dtype_size(dtype) - 1)) == 0; }

int drop_args(float rate, uint64_t seed, const int64_t* seed_at, DropArgs* d) {
    *d = DropArgs{};
    d->scale = 1.f;      // nothing dropped leaves the values as they are
    unsigned thr = 0;
    if (!drop_threshold(rate, &thr) || (reinterpret_cast<uintptr_t>(seed_at) & 7u)) return MAM_ERR_INVALID_ARGUMENT;
    if (rate == 0.f) return MAM_OK;
    d->on = 1;
    d->seed = seed;
    d->seed_at = reinterpret_cast<const long long*>(seed_at);
    d->threshold = thr;
    d->scale = (float)(1.0 / (1.0 - (double)rate));
    return MAM_OK;
}

// ---- rows through shared memory ----
// A row of the ring in shared memory; ragged ones have up to 15 bytes in front, and are read 16 bytes beyond their end.
size_t ring_slot(int64_t width, int size, bool aligned) {
    return aligned ? (size_t)width * size : ((size_t)width * size + 15) / 16 * 16 + 32;
}
// shared memory beside the rows: the parameters, the barriers, their alignment
size_t ring_rest(int64_t width, int params) { return params * (size_t)(width + 8) * 4 + 32 * 4 * 8 + 256; }
int ring_stages(int64_t width, int groups, int size, int tensors, int params, bool aligned, const DevInfo& d) {
    const size_t row = tensors * ring_slot(width, size, aligned) * groups, rest = ring_rest(width, params) + 1024;
    const long long n = (long long)d.max_smem > (long long)rest ? (long long)((d.max_smem - rest) / row) : 0;
    return (int)(n < 4 ? n : 4);
}

// Lets a kernel have all the dynamic shared memory that ring_stages counts with: asked of the runtime once for each device,
// and always the same, so that calls from several threads cannot take it from one another.
template <auto KERNEL>
int allow_smem(const DevInfo& d) {
    static std::atomic<bool> allowed[64];
    int dev = 0;
    MAM_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return MAM_ERR_UNSUPPORTED;
    if (allowed[dev].load(std::memory_order_acquire)) return MAM_OK;
    MAM_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, d.max_smem - 1024));
    allowed[dev].store(true, std::memory_order_release);
    return MAM_OK;
}

template <auto KERNEL, class Params>
int ring_run(const Params& p, unsigned ctas, const NormRing& r, const DevInfo& d, cudaStream_t st) {
    const int e = allow_smem<KERNEL>(d);
    if (e != MAM_OK) return e;
    KERNEL<<<ctas, r.group * r.groups, r.bytes, st>>>(p, r);
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}
NormRing ring_of(int64_t width, int group, int groups, int stages, int size, int tensors, int params, bool aligned) {
    NormRing r{};
    r.group = group;
    r.groups = groups;
    r.stages = stages;
    r.slot_bytes = (unsigned)ring_slot(width, size, aligned);
    r.weights_at = (unsigned)(((size_t)tensors * r.slot_bytes * groups * stages + 127) / 128 * 128);
    r.bars_at = (unsigned)(r.weights_at + params * ((width + 7) / 8 * 8 * 4));
    r.bytes = r.bars_at + groups * stages * 8;
    r.late = g_norm_late;
    return r;
}

// ---- forward of the norm ----
template <typename T, int NV, bool ADD, int MODE>
void fwd_launch(const NormFwdParams& p, int lanes, int threads, cudaStream_t st) {
    const auto grid = [&](int per) { return (unsigned)((p.rows + per - 1) / per); };
    if (lanes == 32) {
        mam_norm_fwd_kernel<T, NV, ADD, MODE, false, 32><<<grid(4), 128, 0, st>>>(p);
    } else if (lanes) {
        if constexpr (NV == 1) {
            if (lanes == 8) mam_norm_fwd_kernel<T, 1, ADD, MODE, false, 8><<<grid(16), 128, 0, st>>>(p);
            else mam_norm_fwd_kernel<T, 1, ADD, MODE, false, 16><<<grid(8), 128, 0, st>>>(p);
        }
    } else if constexpr (NV != 3 && NV != 6) {
        mam_norm_fwd_kernel<T, NV, ADD, MODE, true, 32><<<(unsigned)p.rows, threads, 0, st>>>(p);
    }
}
template <typename T, int NV, bool ADD>
void fwd_mode(const NormFwdParams& p, bool aligned, int lanes, int threads, cudaStream_t st) {
    const bool full = p.width == (long long)(lanes ? lanes : threads) * NV * VEC<T>;
    if (!aligned) fwd_launch<T, NV, ADD, RAGGED>(p, lanes, threads, st);
    else if (full) fwd_launch<T, NV, ADD, FULL>(p, lanes, threads, st);
    else fwd_launch<T, NV, ADD, ALIGNED>(p, lanes, threads, st);
}

// Threads a row and rows at a time for the forward's ring: the form that leaves the fewest threads without values.
struct FwdPlan {
    int per, group, groups;
};
FwdPlan fwd_plan(int64_t width, int size, bool add, bool aligned, const DevInfo& d) {
    FwdPlan b{};
    const int tensors = add ? 2 : 1;
    double best = 0;
    for (int per : {16, 24, 8}) {
        const int group = (int)(((width + per - 1) / per + 31) / 32 * 32), most = per == 8 ? 1024 : per == 16 ? 768 : 640;
        int groups = most / group;
        if (group > 32 && groups > 15) groups = 15;      // named barriers
        while (groups > 1 && ring_stages(width, groups, size, tensors, 2, aligned, d) < 3) --groups;
        if (groups == 0 || ring_stages(width, groups, size, tensors, 2, aligned, d) < 2) continue;
        const double score = (double)width * groups / ((double)per * most) * (per == 8 ? 0.85 : 1.0) * (groups > 1 ? 1.0 : 0.8);
        if (score <= best) continue;
        best = score;
        b = FwdPlan{per, group, groups};
    }
    return b;
}

template <typename T, int NV, bool ADD>
int fwd_ring(const NormFwdParams& p, const FwdPlan& b, bool aligned, const DevInfo& d, cudaStream_t st) {
    const int tensors = ADD ? 2 : 1, stages = ring_stages(p.width, b.groups, sizeof(T), tensors, 2, aligned, d);
    const NormRing r = ring_of(p.width, b.group, b.groups, stages, sizeof(T), tensors, 2, aligned);
    const long long ctas = (p.rows + b.groups - 1) / b.groups;
    const unsigned grid = (unsigned)(ctas < d.sms ? ctas : d.sms);
    if (!aligned) return ring_run<mam_norm_fwd_ring_kernel<T, NV, ADD, RAGGED>>(p, grid, r, d, st);
    if (p.width == (long long)b.group * NV * VEC<T>) return ring_run<mam_norm_fwd_ring_kernel<T, NV, ADD, FULL>>(p, grid, r, d, st);
    return ring_run<mam_norm_fwd_ring_kernel<T, NV, ADD, ALIGNED>>(p, grid, r, d, st);
}

template <typename T, bool ADD>
int fwd_pick(NormFwdParams& p, bool aligned, const DevInfo& d, cudaStream_t st) {
    const long long vecs = (p.width + VEC<T> - 1) / VEC<T>;
    // few rows: as many threads a row as it has vectors; many: a warp or less a row while it fits, else eight or four
    // vectors a thread
    const bool few = p.rows < 4 * (long long)d.sms;
    // Through shared memory: ragged rows (bf16 [5003, 1283] 18.5 -> 16.5 us, with dropout and residual 45 -> 30), and 16-bit rows
    // behind a residual that would take eight vectors a thread ([32768, 4096] 277 -> 179 us).  The others keep more
    // threads on an SM without it: [32768, 4096] bf16 97 us against 118, [12608, 768] fp32 with residual 27 against 29; 16-bit
    // with residual, without / through shared memory: [16384, 5120] 124 / 132, [32768, 2560] 114 / 123, 1280 63 / 74, 1024 47 / 51.
    const bool eight = vecs > 192 && (vecs <= 256 || vecs % 256 == 0 || vecs > 2048);
    if ((!aligned || (ADD && eight && sizeof(T) == 2)) && p.rows >= 16LL * d.sms && p.width > 128) {
        const FwdPlan b = fwd_plan(p.width, sizeof(T), ADD, aligned, d);
        if (b.per) {
            const int e = wait_words(&p.wait);
            if (e != MAM_OK) return e;
            if (b.per == 8) return fwd_ring<T, 8 / VEC<T>, ADD>(p, b, aligned, d, st);
            if (b.per == 16) return fwd_ring<T, 16 / VEC<T>, ADD>(p, b, aligned, d, st);
            return fwd_ring<T, 24 / VEC<T>, ADD>(p, b, aligned, d, st);
        }
    }
    if (vecs <= 32) {
        fwd_mode<T, 1, ADD>(p, aligned, vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32, 0, st);
    } else if (!few && vecs <= 256) {
        if (vecs <= 64) fwd_mode<T, 2, ADD>(p, aligned, 32, 0, st);
        else if (vecs <= 96) fwd_mode<T, 3, ADD>(p, aligned, 32, 0, st);
        else if (vecs <= 128) fwd_mode<T, 4, ADD>(p, aligned, 32, 0, st);
        else if (vecs <= 192) fwd_mode<T, 6, ADD>(p, aligned, 32, 0, st);
        else fwd_mode<T, 8, ADD>(p, aligned, 32, 0, st);
    } else if (vecs <= 4096) {
        const int nv = few ? (vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : 8) : vecs % 256 == 0 || vecs > 2048 ? 8 : 4;
        const int threads = (int)(((vecs + nv - 1) / nv + 31) / 32 * 32);
        if (nv == 1) fwd_mode<T, 1, ADD>(p, aligned, 0, threads, st);
        else if (nv == 2) fwd_mode<T, 2, ADD>(p, aligned, 0, threads, st);
        else if (nv == 4) fwd_mode<T, 4, ADD>(p, aligned, 0, threads, st);
        else fwd_mode<T, 8, ADD>(p, aligned, 0, threads, st);
    } else if (aligned) {
        mam_norm_fwd_wide_kernel<T, ADD, ALIGNED><<<(unsigned)p.rows, 1024, 0, st>>>(p);
    } else {
        mam_norm_fwd_wide_kernel<T, ADD, RAGGED><<<(unsigned)p.rows, 1024, 0, st>>>(p);
    }
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}

// ---- backward of the norm ----
struct BwdPlan {
    enum { WIDE, NARROW, RING } kind;      // rows beyond a CTA's registers; less than a warp a row; rows in shared memory
    int per;                               // values a thread
    int group, groups;                     // threads a row, rows at a time in a CTA
    long long parts;                       // partial rows
};

// Most partial rows of a backward: a CTA an SM, or the slabs of the wide form.
long long bwd_parts(int64_t rows, int64_t width, int sms) {
    if (width <= 8192) return rows < sms ? rows : sms;
    const long long groups = (width + 127) / 128;      // a CTA's columns in fp32; 16-bit types have half as many CTAs
    const long long slabs = 8LL * sms / groups, most = (rows + 31) / 32;
    return slabs < 1 ? 1 : slabs < most ? slabs : most;
}

BwdPlan bwd_plan(int64_t rows, int64_t width, int size, bool add, bool aligned, const DevInfo& d) {
    BwdPlan b{};
    if (width > 8192) {
        b.kind = BwdPlan::WIDE;
        b.parts = bwd_parts(rows, width, d.sms);
        return b;
    }
    const auto threads = [&](int per) { return (int)(((width + per - 1) / per + 31) / 32 * 32); };
    const int tensors = add ? 3 : 2;
    if (width > 128) {
        // The form that leaves the fewest threads without values: 8, 16 or 24 values a thread, of which an SM's registers
        // hold 640, 512 and 384 threads.  Fewer values a thread cost more for what each row takes beside them, and a row at
        // a time leaves its reduction uncovered.  bf16, GB/s by values a thread, 8 / 16 / 24: width 512 4000 / 5170 / 4560,
        // 768 2790 / 2900 / 3060, 2048 3170 / 4000 / 3910, 5120 4370 / 4580 / 3960 (with dropout 5100 / 4650 / 3940).
        b.kind = BwdPlan::RING;
        double best = 0;
        for (int per : {16, 24, 8}) {
            const int group = threads(per), most = per == 24 ? 384 : per == 8 ? 640 : 512;
            int groups = most / group < 15 ? most / group : 15;      // named barriers
            while (groups > 1 && ring_stages(width, groups, size, tensors, 1, aligned, d) < 3) --groups;
            if (groups == 0 || ring_stages(width, groups, size, tensors, 1, aligned, d) < 2) continue;
            const double score = (double)width * groups / ((double)per * most) * (per == 8 ? 0.85 : 1.0) * (groups > 1 ? 1.0 : 0.8);
            if (score <= best) continue;
            best = score;
            b.per = per;
            b.group = group;
            b.groups = groups;
        }
    }
    if (width > 128 && b.per == 0) {      // shared memory for less than two rows (not on a B200)
        b.kind = BwdPlan::WIDE;
        b.parts = bwd_parts(rows, width, d.sms);
        return b;
    }
    if (width <= 128) {
        b.kind = BwdPlan::NARROW;
        b.per = 8;
        b.group = width <= 64 ? 8 : 16;
        b.groups = 512 / b.group;
    }
    if (b.group >= 32) {
        // few rows: over all SMs first
        const long long fair = (rows + d.sms - 1) / d.sms;
        if (fair < b.groups) b.groups = (int)fair;
    }
    const long long ctas = (rows + b.groups - 1) / b.groups;
    b.parts = ctas < d.sms ? ctas : d.sms;
    return b;
}

template <typename T, int NV, bool ADD>
int ring_launch(const NormBwdParams& p, const BwdPlan& b, bool aligned, const DevInfo& d, cudaStream_t st) {
    const int tensors = ADD ? 3 : 2, stages = ring_stages(p.width, b.groups, sizeof(T), tensors, 1, aligned, d);
    if (stages < 2) return MAM_ERR_UNSUPPORTED;
    const NormRing r = ring_of(p.width, b.group, b.groups, stages, sizeof(T), tensors, 1, aligned);
    const unsigned ctas = (unsigned)b.parts;
    if (!aligned) return ring_run<mam_norm_bwd_ragged_kernel<T, NV, ADD>>(p, ctas, r, d, st);
    if (p.width == (long long)b.group * NV * VEC<T>) return ring_run<mam_norm_bwd_ring_kernel<T, NV, ADD, FULL>>(p, ctas, r, d, st);
    return ring_run<mam_norm_bwd_ring_kernel<T, NV, ADD, ALIGNED>>(p, ctas, r, d, st);
}

template <typename T, bool ADD, int MODE>
void narrow_launch(const NormBwdParams& p, const BwdPlan& b, cudaStream_t st) {
    const size_t smem = 16 * 2 * (size_t)p.width * 4;      // at most 16 KB
    if (b.group == 8) mam_norm_bwd_narrow_kernel<T, 8 / VEC<T>, ADD, MODE, 8><<<(unsigned)b.parts, 512, smem, st>>>(p);
    else mam_norm_bwd_narrow_kernel<T, 8 / VEC<T>, ADD, MODE, 16><<<(unsigned)b.parts, 512, smem, st>>>(p);
}

template <typename T, bool ADD, int MODE>
void wide_launch(const NormBwdParams& p, cudaStream_t st) {
    const unsigned rows = (unsigned)p.rows;
    // CTAs of half the size where they suffice: two rows at a time on an SM
    if (p.width <= 4096 * VEC<T>)
        mam_norm_bwd_wide_kernel<T, 4, ADD, MODE><<<rows, p.width <= 2048 * VEC<T> ? 512 : 1024, 0, st>>>(p);
    else mam_norm_bwd_wide_kernel<T, 0, ADD, MODE><<<rows, 1024, 0, st>>>(p);
}

template <typename T, bool ADD>
int bwd_pick(const NormBwdParams& p, const BwdPlan& b, bool aligned, const DevInfo& d, cudaStream_t st) {
    if (b.kind == BwdPlan::RING) {
        if (b.per == 8) return ring_launch<T, 8 / VEC<T>, ADD>(p, b, aligned, d, st);
        if (b.per == 16) return ring_launch<T, 16 / VEC<T>, ADD>(p, b, aligned, d, st);
        return ring_launch<T, 24 / VEC<T>, ADD>(p, b, aligned, d, st);
    }
    if (b.kind == BwdPlan::NARROW) {
        if (aligned) narrow_launch<T, ADD, ALIGNED>(p, b, st);
        else narrow_launch<T, ADD, RAGGED>(p, b, st);
        MAM_CUDA(cudaGetLastError());
        return MAM_OK;
    }
    if (aligned) wide_launch<T, ADD, ALIGNED>(p, st);
    else wide_launch<T, ADD, RAGGED>(p, st);
    if (p.partial) {
        const long long per = (p.rows + b.parts - 1) / b.parts;
        const dim3 grid((unsigned)((p.width + NORM_COLS * VEC<T> - 1) / (NORM_COLS * VEC<T>)), (unsigned)b.parts);
        if (aligned) mam_norm_bwd_cols_kernel<T, ALIGNED><<<grid, NORM_COLS * NORM_LANES, 0, st>>>(p, per);
        else mam_norm_bwd_cols_kernel<T, RAGGED><<<grid, NORM_COLS * NORM_LANES, 0, st>>>(p, per);
    }
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}

template <typename T>
int bwd_type(const NormBwdParams& p, const BwdPlan& b, bool vec, bool add, void* dweight, void* dbias, const DevInfo& d,
             cudaStream_t st) {
    int e;
    if (add) e = bwd_pick<T, true>(p, b, vec, d, st);
    else e = bwd_pick<T, false>(p, b, vec, d, st);
    if (e != MAM_OK || !p.partial) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((2 * p.width + NORM_COLS - 1) / NORM_COLS));
    cfg.blockDim = dim3(NORM_COLS * NORM_LANES);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MAM_CUDA(cudaLaunchKernelEx(&cfg, mam_norm_params_kernel<T>, (const float*)p.partial, dweight, dbias, (long long)b.parts,
                                p.width, p.params_f32));
    return MAM_OK;
}

// ---- pointwise ----
template <typename T, int NV, int OP>
int point_run(PointParams p, bool aligned, cudaStream_t st) {
    const long long per = (long long)POINT_THREADS * VEC<T> * NV;
    const int tail = aligned ? (int)(p.n % VEC<T>) : 0;
    p.n -= tail;
    p.tail = tail;
    const long long blocks = (p.n + per - 1) / per + (tail ? 1 : 0);
    if (blocks > 2147483647LL) return MAM_ERR_UNSUPPORTED;
    if (tail) mam_point_kernel<T, NV, OP, ALIGNED, true><<<(unsigned)blocks, POINT_THREADS, 0, st>>>(p);
    else if (aligned) mam_point_kernel<T, NV, OP, ALIGNED, false><<<(unsigned)blocks, POINT_THREADS, 0, st>>>(p);
    else mam_point_kernel<T, NV, OP, RAGGED, false><<<(unsigned)blocks, POINT_THREADS, 0, st>>>(p);
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}
template <typename T, int OP>
int point_launch(const PointParams& p, bool aligned, const DevInfo& d, cudaStream_t st) {
    // four vectors a thread, or one where that leaves SMs without work
    if (p.n > 4LL * POINT_THREADS * VEC<T> * 2 * d.sms) return point_run<T, 4, OP>(p, aligned, st);
    return point_run<T, 1, OP>(p, aligned, st);
}
template <int OP>
int point(const void* x, const void* other, void* out, int64_t n, int dtype, float rate, uint64_t seed,
          const int64_t* seed_at, void* stream) {
    if (bad_ptr(x) || bad_ptr(out) || n <= 0 || !dtype_ok(dtype)) return MAM_ERR_INVALID_ARGUMENT;
    if (!natural(x, dtype) || !natural(other, dtype) || !natural(out, dtype)) return MAM_ERR_INVALID_ARGUMENT;
    PointParams p{x, other, out, n, 0, {}};
    int st = drop_args(rate, seed, seed_at, &p.drop);
    if (st != MAM_OK) return st;
    const DevInfo* d = nullptr;
    st = device_info(&d);
    if (st != MAM_OK) return st;
    const bool aligned = aligned16(x) && aligned16(other) && aligned16(out);
    cudaStream_t cs = (cudaStream_t)stream;
    switch (dtype) {
        case MAM_F32: return point_launch<float, OP>(p, aligned, *d, cs);
        case MAM_F16: return point_launch<__half, OP>(p, aligned, *d, cs);
        default: return point_launch<__nv_bfloat16, OP>(p, aligned, *d, cs);
    }
}

constexpr int64_t MOST_ROWS = 2147483647LL, MOST_WIDTH = 1LL << 30;

}  // namespace

extern "C" {

int mam_layer_norm_fwd(const void* x, int64_t x_pitch, const void* residual, int64_t residual_pitch, const void* weight,
                       const void* bias, int param_dtype, float eps, float drop_rate, uint64_t drop_seed,
                       const int64_t* drop_seed_at, void* y, void* sum, float* stats, int64_t rows, int64_t width,
                       int dtype, void* stream) {
    if (bad_ptr(x) || bad_ptr(y) || rows <= 0 || width <= 0 || !dtype_ok(dtype)) return MAM_ERR_INVALID_ARGUMENT;
    if ((param_dtype != MAM_F32 && param_dtype != dtype) || !(eps >= 0.f)) return MAM_ERR_INVALID_ARGUMENT;
    if ((residual == nullptr) != (sum == nullptr) || (residual == nullptr && drop_rate != 0.f))
        return MAM_ERR_INVALID_ARGUMENT;
    if (x_pitch < width || (residual && residual_pitch < width)) return MAM_ERR_INVALID_ARGUMENT;
    for (const void* q : {x, residual, (const void*)y, (const void*)sum})
        if (!natural(q, dtype)) return MAM_ERR_INVALID_ARGUMENT;
    if (!natural(weight, param_dtype) || !natural(bias, param_dtype) || (reinterpret_cast<uintptr_t>(stats) & 7u))
        return MAM_ERR_INVALID_ARGUMENT;
    if (rows > MOST_ROWS || width > MOST_WIDTH) return MAM_ERR_UNSUPPORTED;
    NormFwdParams p{x, residual, weight, bias, y, sum, reinterpret_cast<float2*>(stats), rows, width, x_pitch,
                    residual_pitch, eps, 1.0f / (float)width, param_dtype == MAM_F32, {}, {}};
    int st = drop_args(drop_rate, drop_seed, drop_seed_at, &p.drop);
    if (st != MAM_OK) return st;
    const DevInfo* d = nullptr;
    st = device_info(&d);
    if (st == MAM_OK) st = report_wait((cudaStream_t)stream);      // of an earlier call
    if (st != MAM_OK) return st;
    const int per = 16 / dtype_size(dtype);
    const bool vec = width % per == 0 && x_pitch % per == 0 && (!residual || residual_pitch % per == 0) && aligned16(x) &&
                     aligned16(residual) && aligned16(y) && aligned16(sum) && aligned16(weight) && aligned16(bias);
    cudaStream_t cs = (cudaStream_t)stream;
    switch (dtype) {
        case MAM_F32: return residual ? fwd_pick<float, true>(p, vec, *d, cs) : fwd_pick<float, false>(p, vec, *d, cs);
        case MAM_F16: return residual ? fwd_pick<__half, true>(p, vec, *d, cs) : fwd_pick<__half, false>(p, vec, *d, cs);
        default:
            return residual ? fwd_pick<__nv_bfloat16, true>(p, vec, *d, cs) : fwd_pick<__nv_bfloat16, false>(p, vec, *d, cs);
    }
}

size_t mam_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const DevInfo* d = nullptr;
    const int sms = device_info(&d) == MAM_OK ? d->sms : 148;
    return (size_t)bwd_parts(rows, width, sms) * 2 * (size_t)width * 4;
}

int mam_layer_norm_bwd(const void* gy, const void* gsum, const void* s, int64_t s_pitch, const float* stats,
                       const void* weight, int param_dtype, float drop_rate, uint64_t drop_seed,
                       const int64_t* drop_seed_at, void* ds, void* dx, void* dweight, void* dbias, int64_t rows,
                       int64_t width, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (bad_ptr(s) || bad_ptr(stats) || bad_ptr(ds) || rows <= 0 || width <= 0 || !dtype_ok(dtype) || s_pitch < width)
        return MAM_ERR_INVALID_ARGUMENT;
    if (param_dtype != MAM_F32 && param_dtype != dtype) return MAM_ERR_INVALID_ARGUMENT;
    if (dx == nullptr && drop_rate != 0.f) return MAM_ERR_INVALID_ARGUMENT;
    for (const void* q : {gy, gsum, s, (const void*)ds, (const void*)dx})
        if (!natural(q, dtype)) return MAM_ERR_INVALID_ARGUMENT;
    for (const void* q : {weight, (const void*)dweight, (const void*)dbias})
        if (!natural(q, param_dtype)) return MAM_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(stats) & 7u) return MAM_ERR_INVALID_ARGUMENT;
    if (rows > MOST_ROWS || width > MOST_WIDTH) return MAM_ERR_UNSUPPORTED;
    const bool want_params = dweight || dbias;
    NormBwdParams p{gy, gsum, s, reinterpret_cast<const float2*>(stats), weight, ds, dx, nullptr, rows, width, s_pitch,
                    1.0f / (float)width, param_dtype == MAM_F32, {}, {}};
    int st = drop_args(drop_rate, drop_seed, drop_seed_at, &p.drop);
    if (st != MAM_OK) return st;
    const DevInfo* d = nullptr;
    st = device_info(&d);
    if (st == MAM_OK) st = report_wait((cudaStream_t)stream);      // of an earlier call
    if (st != MAM_OK) return st;
    const int per = 16 / dtype_size(dtype);
    const bool vec = width % per == 0 && s_pitch % per == 0 && aligned16(gy) && aligned16(gsum) && aligned16(s) &&
                     aligned16(ds) && aligned16(dx) && aligned16(weight);
    const bool add = gsum || dx;
    const BwdPlan b = bwd_plan(rows, width, dtype_size(dtype), add, vec, *d);
    if (b.kind == BwdPlan::RING) {
        st = wait_words(&p.wait);
        if (st != MAM_OK) return st;
    }
    if (want_params) {
        if (bad_ptr(workspace) || workspace_bytes < (size_t)b.parts * 2 * (size_t)width * 4 ||
            (reinterpret_cast<uintptr_t>(workspace) & 255u))
            return MAM_ERR_WORKSPACE;
        p.partial = static_cast<float*>(workspace);
    }
    cudaStream_t cs = (cudaStream_t)stream;
    switch (dtype) {
        case MAM_F32: return bwd_type<float>(p, b, vec, add, dweight, dbias, *d, cs);
        case MAM_F16: return bwd_type<__half>(p, b, vec, add, dweight, dbias, *d, cs);
        default: return bwd_type<__nv_bfloat16>(p, b, vec, add, dweight, dbias, *d, cs);
    }
}

int mam_dropout_add(const void* x, const void* residual, void* y, int64_t n, int dtype, float drop_rate,
                    uint64_t drop_seed, const int64_t* drop_seed_at, void* stream) {
    return point<POINT_DROPOUT>(x, residual, y, n, dtype, drop_rate, drop_seed, drop_seed_at, stream);
}

int mam_gelu_fwd(const void* x, void* y, int64_t n, int dtype, float drop_rate, uint64_t drop_seed,
                 const int64_t* drop_seed_at, void* stream) {
    return point<POINT_GELU>(x, nullptr, y, n, dtype, drop_rate, drop_seed, drop_seed_at, stream);
}

int mam_gelu_bwd(const void* gy, const void* x, void* dx, int64_t n, int dtype, float drop_rate, uint64_t drop_seed,
                 const int64_t* drop_seed_at, void* stream) {
    if (bad_ptr(gy)) return MAM_ERR_INVALID_ARGUMENT;
    return point<POINT_GELU_BWD>(x, gy, dx, n, dtype, drop_rate, drop_seed, drop_seed_at, stream);
}

}  // extern "C"
