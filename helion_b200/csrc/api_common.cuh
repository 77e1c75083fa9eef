// Host-side helpers shared by the files that hold the extern "C" entry points: the per-device facts, the launch
// counter, the last CUDA error of a thread, and small arithmetic.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>
#include <mutex>

#include "../../include/helion_lce.h"

namespace lce {

constexpr int kMaxDevices = 64;

struct DeviceInfo {
    std::atomic<bool> known{false};  // sm_count and cc_major hold
    std::atomic<bool> ready{false};  // status_ptr and done_counters hold, and the tensor-map encoder
    int index = 0;
    int sm_count = 0;
    int cc_major = 0;
    int* status_ptr = nullptr;
    unsigned* done_counters = nullptr;  // kDoneSlots of them, zero when idle
    mutable std::atomic<unsigned> next_done_slot{0};
};

inline DeviceInfo g_dev[kMaxDevices];
inline std::mutex g_mutex;
inline std::atomic<unsigned long long> g_launches{0};  // kernels this library has launched (all devices)
#define LCE_COUNT_LAUNCH() g_launches.fetch_add(1, std::memory_order_relaxed)

// The CUDA error behind the last LCE_ERR_CUDA of this thread (lce_last_cuda_error reports its name).
inline thread_local cudaError_t t_last_cuda_error = cudaSuccess;
inline bool cuda_failed(cudaError_t e) {
    if (e == cudaSuccess) return false;
    t_last_cuda_error = e;
    return true;
}

// The current device, which has to be compute capability 10.x.
inline int device_basics(DeviceInfo** out) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return LCE_ERR_CUDA;
    if (dev < 0 || dev >= kMaxDevices) return LCE_ERR_ARG;
    DeviceInfo& d = g_dev[dev];
    if (!d.known.load(std::memory_order_acquire)) {
        std::lock_guard<std::mutex> lock(g_mutex);
        d.index = dev;
        if (cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return LCE_ERR_CUDA;
        if (cudaDeviceGetAttribute(&d.cc_major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return LCE_ERR_CUDA;
        d.known.store(true, std::memory_order_release);
    }
    *out = &d;
    return d.cc_major == 10 ? LCE_OK : LCE_ERR_ARCH;
}

inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
inline size_t align_up(size_t a, size_t b) { return (a + b - 1) / b * b; }
inline size_t elem_size(int dtype) { return dtype == LCE_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == LCE_DTYPE_BF16 || dtype == LCE_DTYPE_F16 || dtype == LCE_DTYPE_F32; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Programmatic dependent launch (HELION_B200_PDL=0 switches it off): kernels that call ptx::grid_dep_wait()
// before they read anything their predecessor in the stream wrote may be launched while that predecessor is
// still running; their launch latency and set-up then hide under its tail.
inline bool pdl_enabled() {
    static const bool kEnabled = [] { const char* e = getenv("HELION_B200_PDL"); return e ? atoi(e) != 0 : true; }();
    return kEnabled;
}

// Launches such a kernel (no dynamic shared memory). Only for kernels that contain the wait.
template <class... KArgs, class... Args>
cudaError_t launch_dependent(void (*kern)(KArgs...), int grid, int block, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = 0;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace lce
