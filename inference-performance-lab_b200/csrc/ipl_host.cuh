// Host helpers of the C ABI: last-error message, device limits and kernel launches. Included once,
// by the library's single translation unit.
#pragma once

#include "ipl_b200.h"

#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstring>

namespace ipl {
namespace {

thread_local char t_last_error[512] = "";

ipl_status fail(ipl_status status, const char* fmt, ...) {
    va_list args;
    va_start(args, fmt);
    std::vsnprintf(t_last_error, sizeof(t_last_error), fmt, args);
    va_end(args);
    return status;
}

constexpr int kMaxDevices = 64;

struct DeviceInfo {
    std::atomic<int> sm_count{0};
    std::atomic<int> max_smem_optin{0};
    std::atomic<uint32_t> smem_configured{0};  // bit per kernel instance given the shared-memory (or cluster-size) opt-in
};
DeviceInfo g_devices[kMaxDevices];

// SM count and opt-in shared memory of the current device, queried once per device.
ipl_status current_device(int* device, DeviceInfo** info) {
    cudaError_t err = cudaGetDevice(device);
    if (err != cudaSuccess) {
        return fail(IPL_ERROR_CUDA, "failed to query the current CUDA device: %s", cudaGetErrorString(err));
    }
    if (*device < 0 || *device >= kMaxDevices) {
        return fail(IPL_ERROR_CUDA, "CUDA device index %d is out of range", *device);
    }
    DeviceInfo& d = g_devices[*device];
    if (d.sm_count.load(std::memory_order_acquire) == 0) {
        int sms = 0, smem = 0;
        err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, *device);
        if (err == cudaSuccess) {
            err = cudaDeviceGetAttribute(&smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, *device);
        }
        if (err != cudaSuccess) {
            return fail(IPL_ERROR_CUDA, "failed to read CUDA device properties: %s", cudaGetErrorString(err));
        }
        d.max_smem_optin.store(smem, std::memory_order_relaxed);
        d.sm_count.store(sms, std::memory_order_release);
    }
    *info = &d;
    return IPL_SUCCESS;
}

// Limits the plan queries plan with: the current device's, as the launch path reads them, so a
// query names the kernel a call on this device launches. Where no device can be queried (a host
// without a GPU), a B200's: 148 SMs, 232448 bytes of opt-in shared memory per block. Leaves
// neither this thread's last-error message nor CUDA's last error changed.
void plan_limits(int* sm_count, int* smem_limit) {
    char saved[sizeof(t_last_error)];
    std::memcpy(saved, t_last_error, sizeof(saved));
    int device = 0;
    DeviceInfo* info = nullptr;
    if (current_device(&device, &info) == IPL_SUCCESS) {
        *sm_count = info->sm_count.load(std::memory_order_relaxed);
        *smem_limit = info->max_smem_optin.load(std::memory_order_relaxed);
        return;
    }
    std::memcpy(t_last_error, saved, sizeof(saved));
    (void)cudaGetLastError();
    *sm_count = 148;
    *smem_limit = 232448;
}

template <typename Kernel, typename... Args>
cudaError_t launch_2d(Kernel kernel, unsigned grid_x, unsigned grid_y, unsigned block, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid_x, grid_y);
    config.blockDim = dim3(block);
    config.stream = stream;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                   Args... args) {
    // Programmatic stream serialisation: the kernel may be scheduled while the previous kernel
    // in the stream drains; it orders its own global reads with griddepcontrol.wait.
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// The same with the grid in thread-block clusters of `cluster` CTAs along x (grid a multiple of it).
template <typename Kernel, typename... Args>
cudaError_t launch_clustered(Kernel kernel, unsigned grid, unsigned cluster, unsigned block, size_t smem,
                             cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = cluster;
    attribute[1].val.clusterDim.y = 1;
    attribute[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = attribute;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

}  // namespace
}  // namespace ipl
