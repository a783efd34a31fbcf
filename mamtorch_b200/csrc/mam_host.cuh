// Host-side helpers shared by the translation units of libmam_b200.so: error recording and device attributes.
#pragma once
#include <atomic>
#include <cuda_runtime.h>
#include <mutex>

#include "../../include/mam_b200.h"

namespace mamb200 {

inline thread_local cudaError_t t_last_cuda = cudaSuccess;

inline int cuda_fail(cudaError_t e) {
    t_last_cuda = e;
    return MAM_ERR_CUDA;
}
#define MAM_CUDA(x)                                  \
    do {                                             \
        cudaError_t e_ = (x);                        \
        if (e_ != cudaSuccess) return cuda_fail(e_); \
    } while (0)

struct DevInfo {
    int sms = 0, major = 0, minor = 0, max_smem = 0;
};
inline DevInfo g_dev[64];
inline std::atomic<bool> g_dev_known[64];     // written behind the mutex: calls come from any thread
inline std::mutex g_dev_mutex;

inline int device_info(const DevInfo** out) {
    int dev = 0;
    MAM_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return MAM_ERR_UNSUPPORTED;
    DevInfo& d = g_dev[dev];
    if (!g_dev_known[dev].load(std::memory_order_acquire)) {
        std::lock_guard<std::mutex> lock(g_dev_mutex);
        DevInfo n;
        MAM_CUDA(cudaDeviceGetAttribute(&n.sms, cudaDevAttrMultiProcessorCount, dev));
        MAM_CUDA(cudaDeviceGetAttribute(&n.major, cudaDevAttrComputeCapabilityMajor, dev));
        MAM_CUDA(cudaDeviceGetAttribute(&n.minor, cudaDevAttrComputeCapabilityMinor, dev));
        MAM_CUDA(cudaDeviceGetAttribute(&n.max_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
        if (!g_dev_known[dev].load(std::memory_order_relaxed)) {
            d = n;
            g_dev_known[dev].store(true, std::memory_order_release);
        }
    }
    *out = &d;
    return d.major == 10 ? MAM_OK : MAM_ERR_NOT_SM100;
}

inline int g_norm_late = 0;   // 1: the first wait of the norm's ring counts as run out (MAM_TUNE_NORM_LATE)

// Where kernels say that a bounded wait ran out (mam_capi.cu): a flag of the device, and its image in pinned host memory, which
// kernels that are given its address write too, so that the host sees it without a copy.
struct WaitWords {
    int *flag, *image;
};
int wait_words(WaitWords* w);
// MAM_ERR_DEVICE_TIMEOUT, once, where the image of the current device says so and `stream` is not being captured
int report_wait(cudaStream_t stream);

inline int bad_ptr(const void* p) { return p == nullptr; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// rate in [0, 1) -> threshold on a 32-bit draw; false if the rate is out of range
inline bool drop_threshold(float rate, unsigned* thr) {
    if (!(rate >= 0.f && rate < 1.f)) return false;
    const double t = (double)rate * 4294967296.0;
    *thr = t >= 4294967295.0 ? 4294967295u : (unsigned)t;
    return true;
}

}  // namespace mamb200
