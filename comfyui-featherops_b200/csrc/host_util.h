// Host-side helpers shared by the translation units of libfeather_b200: the thread-local error text
// behind feather_last_error_string(), what is known once for each device, and launches beside the kernel before.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include <mutex>

namespace feather {

char* error_buffer();   // 512 bytes, thread-local (defined in quant.cu)

inline int set_error(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

constexpr int kMaxDevices = 64;

// SMs of the current device, 0 if that cannot be read.
inline int sm_count() {
    static std::mutex mu;
    static int cached[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    std::lock_guard<std::mutex> lock(mu);
    if (cached[dev] == 0 && cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return cached[dev];
}

// Opt-in shared memory of a kernel, once for each device; one of these belongs to each kernel.
struct SmemOptIn {
    std::mutex mu;
    bool done[kMaxDevices] = {};
    template <typename Kernel>
    cudaError_t operator()(Kernel kernel, int smem) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
        std::lock_guard<std::mutex> lock(mu);
        if (done[dev]) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        done[dev] = e == cudaSuccess;
        return e;
    }
};

// A launch that may become resident and set up while the previous kernel on the stream drains (pdl_wait_for_previous_kernel in ptx.cuh);
// cluster: CTAs of a cluster along x, 0 for a launch without clusters.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, int cluster, int smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace feather
