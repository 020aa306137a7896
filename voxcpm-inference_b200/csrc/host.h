// Host helpers shared by the translation units of libvxb: error reporting,
// the tensor-map encoder, device figures and the programmatic launch.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <string>
#include <utility>

#include "vxb.h"

namespace vxb {

// Records the calling thread's last error message and returns `code`
// (vxb_last_error reads it).
int fail(int code, const std::string& msg);

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, or null if the driver has none.
EncodeTiledFn encode_fn();

// Streaming multiprocessors of device `dev`.
int num_sms(int dev);

// Waits for a stream's work up to timeout_ms (VXB_ERR_TIMEOUT).
int wait_stream(cudaStream_t s, int timeout_ms);

#define CUDA_TRY(expr)                                                                              \
    do {                                                                                            \
        cudaError_t e_ = (expr);                                                                    \
        if (e_ != cudaSuccess)                                                                      \
            return fail(e_ == cudaErrorMemoryAllocation ? VXB_ERR_OUT_OF_MEMORY : VXB_ERR_BACKEND, \
                        std::string(#expr) + ": " + cudaGetErrorString(e_));                       \
    } while (0)

// Launches a kernel with programmatic stream serialisation (the kernel calls
// grid_dep_sync before it touches activations), so its launch and setup
// overlap the previous kernel; captured into graphs as programmatic edges.
// cluster > 1: clusters of that many blocks along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, int cluster, size_t smem,
                               cudaStream_t s, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                       Args&&... args) {
    return launch_pdl_cluster(kernel, grid, block, 1, smem, s, std::forward<Args>(args)...);
}

// Raises a kernel's dynamic shared-memory limit, once per device.
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<bool>* done /* [64] */, int dev) {
    if (dev < 0 || dev >= 64) return fail(VXB_ERR_BACKEND, "device index out of range");
    if (!done[dev].load(std::memory_order_acquire)) {
        CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done[dev].store(true, std::memory_order_release);
    }
    return VXB_OK;
}

}  // namespace vxb
