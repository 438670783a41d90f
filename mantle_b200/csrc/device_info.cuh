// A device's figures, asked once, and the shared-memory limits of kernels: for the host side of every
// translation unit that launches kernels (each keeps a record of its own).
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

namespace {

// What the library asks a device once and then remembers: the driver calls behind these
// figures cost microseconds, which shows on a single-row launch of under twenty.
constexpr int kMaxDevices = 64;
struct DeviceInfo {
    int per_sm;     // shared memory of one SM
    int per_block;  // largest opt-in dynamic shared memory of one CTA
    int sms;
};
DeviceInfo g_device_info[kMaxDevices];
std::atomic<int> g_device_known[kMaxDevices];
std::mutex g_device_mutex;

// Current device ordinal and its figures.  Without a usable device (argument checks run on
// hosts that have none) the B200's own figures stand in and the ordinal is -1.
DeviceInfo device_info(int* dev_out = nullptr) {
    const DeviceInfo b200 = {233472, 232448, 148};
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
        (void)cudaGetLastError();
        if (dev_out) *dev_out = -1;
        return b200;
    }
    if (dev_out) *dev_out = dev;
    if (g_device_known[dev].load(std::memory_order_acquire)) return g_device_info[dev];
    std::lock_guard<std::mutex> lock(g_device_mutex);
    DeviceInfo d = b200;
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMaxSharedMemoryPerMultiprocessor, dev) == cudaSuccess && v > 0) d.per_sm = v;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) == cudaSuccess && v > 0) d.per_block = v;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0) d.sms = v;
    g_device_info[dev] = d;
    g_device_known[dev].store(1, std::memory_order_release);
    return d;
}

// Raises a kernel's dynamic shared-memory limit on the current device when `smem` exceeds what
// an earlier launch already asked for; `granted` is the kernel's own per-device record.  Setting and recording are one
// step to other threads: the limit is the last size set, so that a smaller one set in between would leave the record above it.
template <class K>
int ensure_smem(K kern, size_t smem, std::atomic<int>* granted) {
    int dev = -1;
    (void)device_info(&dev);
    if (dev >= 0 && (size_t)granted[dev].load(std::memory_order_relaxed) >= smem) return 0;
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (dev >= 0 && (size_t)granted[dev].load(std::memory_order_relaxed) >= smem) return 0;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0) granted[dev].store((int)smem, std::memory_order_relaxed);
    return 0;
}

}  // namespace
