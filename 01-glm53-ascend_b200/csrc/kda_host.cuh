// Host helpers of the layer's norm and projection launchers.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <map>
#include <mutex>

namespace kda {

// What is remembered per device has a slot for each of the first 64 (-1: none).
constexpr int kDeviceSlots = 64;

inline int device_slot(int dev) { return dev >= 0 && dev < kDeviceSlots ? dev : -1; }

inline int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess ? dev : 0;
}

inline int sm_count() {
    static std::atomic<int> count[kDeviceSlots];
    const int dev = current_device(), slot = device_slot(dev);
    int c = slot >= 0 ? count[slot].load(std::memory_order_relaxed) : 0;
    if (c == 0) {
        cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
        c = c > 0 ? c : 1;
        if (slot >= 0) count[slot].store(c, std::memory_order_relaxed);
    }
    return c;
}

// The dynamic shared memory that a kernel has been let have on each device.
struct OptIn {
    std::atomic<int> bytes[kDeviceSlots];
    std::mutex growing;
    std::map<int, int> beyond;   // devices without a slot
};

// Lets a kernel have `bytes` of dynamic shared memory; asked once per device
// and growth (`done` is the kernel's own). Threads grow it in turn: the attribute
// is the last value set, so a smaller one must never follow a larger one.
template <typename K>
inline bool opt_in(K kernel, OptIn &done, int bytes) {
    const int dev = current_device(), slot = device_slot(dev);
    if (slot >= 0 && done.bytes[slot].load(std::memory_order_acquire) >= bytes) return true;
    const std::lock_guard<std::mutex> lock(done.growing);
    if ((slot >= 0 ? done.bytes[slot].load(std::memory_order_relaxed) : done.beyond[dev]) >= bytes) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    if (slot >= 0)
        done.bytes[slot].store(bytes, std::memory_order_release);
    else
        done.beyond[dev] = bytes;
    return true;
}

// A launch that may begin while the kernel before it in the stream ends (see
// wait_for_previous), over clusters of `cluster` CTAs along x.
template <typename... P, typename... A>
inline cudaError_t launch_overlapped(void (*kernel)(P...), dim3 grid, int threads, int bytes, int cluster, cudaStream_t st,
                                     const A &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = static_cast<size_t>(bytes);
    config.stream = st;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    config.attrs = attrs;
    config.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
    if (e != cudaSuccess) cudaGetLastError();   // reported by the return value; an earlier call's error is left for its owner
    return e;
}

}  // namespace kda
