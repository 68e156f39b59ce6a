// What the operators on device tensors (rms_norm.cu, linear.cu, sample.cu) share: element types and
// the guards of their C entries.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <string>

#include "../../include/lokiscan.h"
#include "lk_common.cuh"

namespace lk {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// One value of a type known at run time (LK_F32 / LK_F16 / LK_BF16).
__device__ __forceinline__ float load_as(int dtype, const void *p, long long i) {
    if (dtype == LK_F32) return static_cast<const float *>(p)[i];
    if (dtype == LK_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

inline bool float_type(int t) { return t == LK_F32 || t == LK_F16 || t == LK_BF16; }
inline int type_bytes(int t) { return t == LK_F32 ? 4 : (t == LK_I8 ? 1 : 2); }
// Base and row stride both on `to`-byte boundaries.
inline bool aligned_rows(const void *p, long long ld, int elem, int to) {
    return reinterpret_cast<uintptr_t>(p) % to == 0 && (ld * elem) % to == 0;
}

constexpr int kMaxDevices = 64;

// Makes `device` current for the call and puts the caller's device back.
class DeviceScope {
  public:
    // 0, or the status the entry returns
    int enter(int device, const char *who) {
        static const int count = lk_device_count();
        if (device < 0 || device >= count || device >= kMaxDevices)
            return fail(LK_ECUDA, std::string(who) + ": no such CUDA device (this library has no CPU path)");
        int now = -1;
        LK_CUDA(cudaGetDevice(&now));
        if (now == device) return 0;
        LK_CUDA(cudaSetDevice(device));
        prev_ = now;
        return 0;
    }
    ~DeviceScope() {
        if (prev_ >= 0) cudaSetDevice(prev_);
    }

  private:
    int prev_ = -1;
};

// rms_norm.cu: whether one of its bounded waits ran out on the current device since the last call; waits for the device.
int norm_failed(int *out);

// What a device is asked, or told, once: the first call on it does so, and calls that come meanwhile wait until it is done.  What
// went wrong is tried again by the next call.
class OncePerDevice {
  public:
    template <typename F>
    int run(int device, F ask) {
        if (done_[device].load(std::memory_order_acquire)) return 0;
        std::lock_guard<std::mutex> lock(mutex_);
        if (done_[device].load(std::memory_order_relaxed)) return 0;
        LK_TRY(ask());
        done_[device].store(true, std::memory_order_release);
        return 0;
    }

  private:
    std::mutex mutex_;
    std::atomic<bool> done_[kMaxDevices] = {};
};

// SMs of a device, asked once.
inline int sm_count(int device) {
    static OncePerDevice once;
    static int known[kMaxDevices];
    once.run(device, [&] {
        if (cudaDeviceGetAttribute(&known[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
            cudaGetLastError();
            known[device] = 148;
        }
        return 0;
    });
    return known[device];
}

// Launches through the call that returns this launch's own error: nothing another library left pending is
// taken for it.
template <typename... P, typename... A>
inline int launch_cfg(const char *who, void (*kernel)(P...), const cudaLaunchConfig_t &cfg, const A &...args) {
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
    if (e == cudaSuccess) return 0;
    cudaGetLastError();
    return fail(LK_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
}
template <typename... P, typename... A>
inline int launch(const char *who, void (*kernel)(P...), unsigned grid, unsigned threads, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    return launch_cfg(who, kernel, cfg, args...);
}

}  // namespace lk
