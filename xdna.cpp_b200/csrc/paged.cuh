// Internal launcher interface of the paged KV cache operators.  The argument
// records are those of the public header; the entry points (paged_api.cpp)
// have checked them and filled in the strides.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/ggml-b200.h"

namespace xb {

// Streaming multiprocessors of the current device (0 without one).
int sm_count();

constexpr int kMaxSeqs = 16384;  // requests of a plan
cudaError_t kv_plan_launch(const struct b200_kv_plan_args& p, cudaStream_t stream);

cudaError_t qk_norm_rope_launch(const struct b200_qk_norm_rope_args& p, const struct b200_kv_cache& kv,
                                cudaStream_t stream);

size_t paged_attention_workspace(const struct b200_paged_attention_args& p, const struct b200_kv_cache& kv);
cudaError_t paged_attention_launch(const struct b200_paged_attention_args& p, const struct b200_kv_cache& kv,
                                   cudaStream_t stream);
// Reads and clears the current device's error word of the attention kernels'
// bounded waits.
cudaError_t paged_error_status(int* out);

// Lets a kernel have `bytes` of dynamic shared memory; asked of the runtime once
// per device.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
    static std::atomic<uint64_t> done{0};  // a bit for each device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
    e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    return e;
}

// Launch with programmatic stream serialization: the kernel may start while
// the one before it on the stream drains.  Every thread of every kernel
// launched so executes griddepcontrol.wait before its first access to global
// memory (and before it returns), so stream order holds as without it.
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                       int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    cfg.attrs = attr;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

#ifdef __CUDACC__
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

}  // namespace xb
