// What the launchers of the caches' calls share on the host: a device's facts, the current device, launches, alignment.  Every source
// file that includes this has its own.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "fa_b200.h"

namespace {

constexpr int kMaxDevices = 64;

// What is asked of a device once.
struct Device {
    std::atomic<int> sms{0};   // 0: not asked yet
    std::atomic<uint64_t> attr_done{0};   // bit per kernel instance whose shared-memory attribute is set
};
Device g_device[kMaxDevices];

int device_of(int device, Device** out) {
    if (device < 0 || device >= kMaxDevices) return static_cast<int>(cudaErrorInvalidDevice);
    Device& d = g_device[device];
    if (d.sms.load(std::memory_order_acquire) == 0) {
        int major = 0, sms = 0;
        cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return static_cast<int>(e);
        if (major != 10) return FA_B200_ERR_ARCH;
        d.sms.store(sms, std::memory_order_release);
    }
    *out = &d;
    return FA_B200_OK;
}

// Makes `device` current for a call and puts the old one back.
struct OnDevice {
    int before = -1, rc = 0;
    bool changed = false;
    explicit OnDevice(int device) {
        cudaError_t e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) {
            e = cudaSetDevice(device);
            changed = e == cudaSuccess;
        }
        rc = static_cast<int>(e);
    }
    ~OnDevice() {
        if (changed) (void)cudaSetDevice(before);
    }
};

// (the kernels wait for the one before them on the stream before they touch memory)
template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), uint32_t grid, uint32_t block, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <typename Kernel>
int allow_smem(Device& d, uint32_t bit, Kernel* kernel, int bytes) {
    if (d.attr_done.load(std::memory_order_acquire) & (1ull << bit)) return FA_B200_OK;   // (setting it twice is harmless)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    d.attr_done.fetch_or(1ull << bit, std::memory_order_release);
    return FA_B200_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool multiple16(int64_t x) { return (x & 15) == 0; }

}  // namespace
