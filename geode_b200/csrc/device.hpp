// device.hpp - what every translation unit of the library shares on the host: the process-wide launch counter, the
// per-device set-up state with the operators' status word, and the launch with or without programmatic overlap.
// What depends on the GPU (its SM count, the kernels' shared-memory opt-in, the status word) is kept per device and
// set up the first time a launch on that device (the current one) needs it, so handles on several GPUs of one
// process each get their own.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>

#include "../../include/geode_cuda.h"

namespace gcu {

inline std::atomic<uint64_t> &launch_counter() {
    static std::atomic<uint64_t> n{0};
    return n;
}
inline void count_launch(uint64_t k = 1) { launch_counter().fetch_add(k, std::memory_order_relaxed); }

// Per-device set-up state, filled lazily under one mutex. gemv_rc / bf16_rc: 0 = not tried yet, else the outcome
// (GCUDA_OK or GCUDA_E_CUDA) of the shared-memory opt-in on that device.
constexpr int kMaxDevices = 64;
struct DeviceState {
    std::mutex mu;
    int sms[kMaxDevices] = {};
    int gemv_rc[kMaxDevices] = {};
    int bf16_rc[kMaxDevices] = {};
    int umma_rc[kMaxDevices] = {};
    int lane_rc[kMaxDevices] = {};
    size_t lane_avail[kMaxDevices] = {};   // the expert lane kernels' dynamic shared memory limit
    uint32_t *status[kMaxDevices] = {};
};
inline DeviceState &device_state() {
    static DeviceState d;
    return d;
}
inline int current_device() {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
    return dev;
}

inline int sm_count() {
    const int dev = current_device();
    if (dev < 0) return 148;
    DeviceState &d = device_state();
    std::lock_guard<std::mutex> lock(d.mu);
    if (!d.sms[dev]) {
        int c = 0;
        if (cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || c <= 0) c = 148;
        d.sms[dev] = c;
    }
    return d.sms[dev];
}

// GCUDA_OK where the pointers (NULL: passed over) can be followed on the current device - its own memory, page-locked host
// memory, managed memory - else GCUDA_E_ARG (a kernel that follows memory of another device, or an ordinary host address,
// faults); GCUDA_E_CUDA without a device. The driver's single attribute, 29 ns a pointer: the runtime's query of all of them
// takes 2.5 us. The driver's function comes through the runtime, so the library loads where no driver is installed.
inline decltype(&cuPointerGetAttribute) pointer_attribute() {
    static const auto fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuPointerGetAttribute", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<decltype(&cuPointerGetAttribute)>(f);
    }();
    return fn;
}
template <typename... P>
inline int on_current_device(const P *...p) {
    const int dev = current_device();
    if (dev < 0 || !pointer_attribute()) return GCUDA_E_CUDA;
    auto ask = [](const void *q, CUpointer_attribute what) {   // (-1: unknown to the driver)
        int v = 0;
        return pointer_attribute()(&v, what, reinterpret_cast<CUdeviceptr>(q)) == CUDA_SUCCESS ? v : -1;
    };
    auto here = [&](const void *q) {
        return !q || ask(q, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL) == dev || ask(q, CU_POINTER_ATTRIBUTE_MEMORY_TYPE) == CU_MEMORYTYPE_HOST ||
               ask(q, CU_POINTER_ATTRIBUTE_IS_MANAGED) == 1;
    };
    return (here(p) && ...) ? GCUDA_OK : GCUDA_E_ARG;
}

// The operators' status word on the current device (device memory, zeroed once): kernels OR error flags into it.
// The first call on a device may come while the caller captures a stream, so the word is made outside any capture:
// the thread's capture mode relaxed for the allocation, the zeroing on a stream of its own.
inline uint32_t *device_status() {
    const int dev = current_device();
    if (dev < 0) return nullptr;
    DeviceState &d = device_state();
    std::lock_guard<std::mutex> lock(d.mu);
    if (!d.status[dev]) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
        void *q = nullptr;
        cudaStream_t st = nullptr;
        const bool ok = cudaMalloc(&q, 4) == cudaSuccess &&
                        cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) == cudaSuccess &&
                        cudaMemsetAsync(q, 0, 4, st) == cudaSuccess && cudaStreamSynchronize(st) == cudaSuccess;
        if (st) cudaStreamDestroy(st);
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (!ok) {
            if (q) cudaFree(q);
            return nullptr;
        }
        d.status[dev] = static_cast<uint32_t *>(q);
    }
    return d.status[dev];
}

// A kernel's shared-memory opt-in on the current device, once per device (bytes: the largest any of its launches takes).
template <auto kern>
inline bool shared_opt_in(int bytes) {
    static std::atomic<uint64_t> done{0};
    const int dev = current_device();
    if (dev < 0) return false;
    if (done.load(std::memory_order_acquire) >> dev & 1) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done.fetch_or(1ull << dev, std::memory_order_release);
    return true;
}

// Launch with the programmatic-stream-serialization attribute when pdl: the kernel may begin (its prologue, the
// weight stream) before the previous kernel on the stream ends; it waits for it at griddepcontrol.wait.
template <typename Kern, typename... Args>
inline cudaError_t launch_ex(Kern kern, dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    int na = 0;
    if (pdl) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        na = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    count_launch();
    return e;
}

}  // namespace gcu
