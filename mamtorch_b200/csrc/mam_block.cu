// C ABI of the operators between the MAM layers of a transformer block: layer norm, dropout with residual addition, GELU.
// Declarations are in include/mam_b200.h.
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

// ---- forward of the norm ----
template <typename T, int VEC, int NV, bool ADD>
void fwd_launch(const NormFwdParams& p, bool warp, int threads, cudaStream_t st) {
    if (warp) mam_norm_fwd_kernel<T, VEC, NV, ADD, true><<<(unsigned)((p.rows + 3) / 4), 128, 0, st>>>(p);
    else mam_norm_fwd_kernel<T, VEC, NV, ADD, false><<<(unsigned)p.rows, threads, 0, st>>>(p);
}

template <typename T, int VEC, bool ADD>
void fwd_pick(const NormFwdParams& p, const DevInfo& d, cudaStream_t st) {
    constexpr int E = VEC == 1 ? 4 : 1;            // vectors a thread: E, 2E, 4E, 8E
    const long long vecs = (p.width + VEC - 1) / VEC;
    // few rows: as many threads a row as it has vectors; many: a warp a row while it fits, else 4E vectors a thread
    const bool few = p.rows < 4 * (long long)d.sms;
    const bool warp = vecs <= 32 * E || (!few && vecs <= 32 * 8 * E);
    long long per = warp ? (vecs + 31) / 32 : few ? (vecs + 1023) / 1024 : 4 * E;
    if (!warp && vecs > 1024 * per) per = (vecs + 1023) / 1024;
    if (per > 8 * E) {
        mam_norm_fwd_wide_kernel<T, VEC, ADD><<<(unsigned)p.rows, 1024, 0, st>>>(p);
        return;
    }
    const int nv = per <= E ? E : per <= 2 * E ? 2 * E : per <= 4 * E ? 4 * E : 8 * E;
    const int threads = (int)(((vecs + nv - 1) / nv + 31) / 32 * 32);
    if (nv == E) fwd_launch<T, VEC, E, ADD>(p, warp, threads, st);
    else if (nv == 2 * E) fwd_launch<T, VEC, 2 * E, ADD>(p, warp, threads, st);
    else if (nv == 4 * E) fwd_launch<T, VEC, 4 * E, ADD>(p, warp, threads, st);
    else fwd_launch<T, VEC, 8 * E, ADD>(p, warp, threads, st);
}

template <typename T>
void fwd_type(const NormFwdParams& p, bool vec, const DevInfo& d, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (p.residual) {
        if (vec) fwd_pick<T, V, true>(p, d, st);
        else fwd_pick<T, 1, true>(p, d, st);
    } else {
        if (vec) fwd_pick<T, V, false>(p, d, st);
        else fwd_pick<T, 1, false>(p, d, st);
    }
}

// ---- backward of the norm ----
struct BwdPlan {
    bool wide;          // rows beyond what a CTA's registers hold: rows and columns in kernels of their own
    int per;            // values a thread
    int group, groups;  // threads a row, rows at a time in a CTA
    long long parts;    // partial rows
};

BwdPlan bwd_plan(int64_t rows, int64_t width, int sms) {
    BwdPlan b{};
    b.wide = width > 8192;
    if (b.wide) {
        const long long groups = (width + NORM_COLS - 1) / NORM_COLS;
        long long slabs = (8LL * sms + groups - 1) / groups;
        const long long most = (rows + 63) / 64;
        b.parts = slabs < most ? slabs : most;
        return b;
    }
    b.per = width <= 4096 ? 8 : 16;
    b.group = (int)(((width + b.per - 1) / b.per + 31) / 32 * 32);
    b.groups = 512 / b.group > 0 ? 512 / b.group : 1;
    if (b.groups > 8) b.groups = 8;
    const long long ctas = (rows + b.groups - 1) / b.groups, most = 2LL * sms;
    b.parts = ctas < most ? ctas : most;
    return b;
}

template <typename T, int VEC, int NV, bool ADD>
int bwd_launch(const NormBwdParams& p, const BwdPlan& b, cudaStream_t st) {
    const size_t smem = b.groups > 1 ? (size_t)p.width * 8 : 0;   // at most 16 KB: several groups share a CTA up to width 2048
    mam_norm_bwd_kernel<T, VEC, NV, ADD><<<(unsigned)b.parts, b.group * b.groups, smem, st>>>(p, b.group);
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}

template <typename T, int VEC, bool ADD>
int bwd_pick(const NormBwdParams& p, const BwdPlan& b, cudaStream_t st) {
    if (!b.wide) {
        if (b.per == 8) return bwd_launch<T, VEC, 8 / VEC, ADD>(p, b, st);
        return bwd_launch<T, VEC, 16 / VEC, ADD>(p, b, st);
    }
    mam_norm_bwd_wide_kernel<T, VEC, ADD><<<(unsigned)p.rows, 1024, 0, st>>>(p);
    if (p.partial) {
        const long long per = (p.rows + b.parts - 1) / b.parts;
        mam_norm_bwd_cols_kernel<T><<<dim3((unsigned)((p.width + NORM_COLS - 1) / NORM_COLS), (unsigned)b.parts),
                                      NORM_COLS * NORM_LANES, 0, st>>>(p, per);
    }
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}

template <typename T>
int bwd_type(const NormBwdParams& p, const BwdPlan& b, bool vec, bool add, void* dweight, void* dbias, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    int e;
    if (add) e = vec ? bwd_pick<T, V, true>(p, b, st) : bwd_pick<T, 1, true>(p, b, st);
    else e = vec ? bwd_pick<T, V, false>(p, b, st) : bwd_pick<T, 1, false>(p, b, st);
    if (e != MAM_OK || !p.partial) return e;
    mam_norm_params_kernel<T><<<(unsigned)((2 * p.width + NORM_COLS - 1) / NORM_COLS), NORM_COLS * NORM_LANES, 0, st>>>(
        p.partial, dweight, dbias, b.parts, p.width, p.params_f32);
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}

// ---- pointwise ----
template <typename T, int VEC, int OP>
int point_launch(const PointParams& p, cudaStream_t st) {
    constexpr int NV = VEC == 1 ? 4 : 2;
    const long long blocks = (p.n + 256LL * VEC * NV - 1) / (256LL * VEC * NV);
    if (blocks > 2147483647LL) return MAM_ERR_UNSUPPORTED;
    mam_point_kernel<T, VEC, NV, OP><<<(unsigned)blocks, 256, 0, st>>>(p);
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}
template <int OP>
int point(const void* x, const void* other, void* out, int64_t n, int dtype, float rate, uint64_t seed,
          const int64_t* seed_at, void* stream) {
    if (bad_ptr(x) || bad_ptr(out) || n <= 0 || !dtype_ok(dtype)) return MAM_ERR_INVALID_ARGUMENT;
    if (!natural(x, dtype) || !natural(other, dtype) || !natural(out, dtype)) return MAM_ERR_INVALID_ARGUMENT;
    PointParams p{x, other, out, n, {}};
    int st = drop_args(rate, seed, seed_at, &p.drop);
    if (st != MAM_OK) return st;
    const DevInfo* d = nullptr;
    st = device_info(&d);
    if (st != MAM_OK) return st;
    const bool vec = aligned16(x) && aligned16(other) && aligned16(out);
    cudaStream_t cs = (cudaStream_t)stream;
    switch (dtype) {
        case MAM_F32: return vec ? point_launch<float, 4, OP>(p, cs) : point_launch<float, 1, OP>(p, cs);
        case MAM_F16: return vec ? point_launch<__half, 8, OP>(p, cs) : point_launch<__half, 1, OP>(p, cs);
        default: return vec ? point_launch<__nv_bfloat16, 8, OP>(p, cs) : point_launch<__nv_bfloat16, 1, OP>(p, cs);
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
                    residual_pitch, eps, param_dtype == MAM_F32, {}};
    int st = drop_args(drop_rate, drop_seed, drop_seed_at, &p.drop);
    if (st != MAM_OK) return st;
    const DevInfo* d = nullptr;
    st = device_info(&d);
    if (st != MAM_OK) return st;
    const int per = 16 / dtype_size(dtype);
    const bool vec = width % per == 0 && x_pitch % per == 0 && (!residual || residual_pitch % per == 0) && aligned16(x) &&
                     aligned16(residual) && aligned16(y) && aligned16(sum) && aligned16(weight) && aligned16(bias);
    cudaStream_t cs = (cudaStream_t)stream;
    switch (dtype) {
        case MAM_F32: fwd_type<float>(p, vec, *d, cs); break;
        case MAM_F16: fwd_type<__half>(p, vec, *d, cs); break;
        default: fwd_type<__nv_bfloat16>(p, vec, *d, cs);
    }
    MAM_CUDA(cudaGetLastError());
    return MAM_OK;
}

size_t mam_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const DevInfo* d = nullptr;
    const int sms = device_info(&d) == MAM_OK ? d->sms : 148;
    return (size_t)bwd_plan(rows, width, sms).parts * 2 * (size_t)width * 4;
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
                    param_dtype == MAM_F32, {}};
    int st = drop_args(drop_rate, drop_seed, drop_seed_at, &p.drop);
    if (st != MAM_OK) return st;
    const DevInfo* d = nullptr;
    st = device_info(&d);
    if (st != MAM_OK) return st;
    const BwdPlan b = bwd_plan(rows, width, d->sms);
    if (want_params) {
        if (bad_ptr(workspace) || workspace_bytes < (size_t)b.parts * 2 * (size_t)width * 4 ||
            (reinterpret_cast<uintptr_t>(workspace) & 255u))
            return MAM_ERR_WORKSPACE;
        p.partial = static_cast<float*>(workspace);
    }
    const int per = 16 / dtype_size(dtype);
    const bool vec = width % per == 0 && s_pitch % per == 0 && aligned16(gy) && aligned16(gsum) && aligned16(s) &&
                     aligned16(ds) && aligned16(dx) && aligned16(weight);
    const bool add = gsum || dx;
    cudaStream_t cs = (cudaStream_t)stream;
    switch (dtype) {
        case MAM_F32: return bwd_type<float>(p, b, vec, add, dweight, dbias, cs);
        case MAM_F16: return bwd_type<__half>(p, b, vec, add, dweight, dbias, cs);
        default: return bwd_type<__nv_bfloat16>(p, b, vec, add, dweight, dbias, cs);
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
