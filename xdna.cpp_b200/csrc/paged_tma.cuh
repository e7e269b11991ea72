// Barriers with bounded waits and TMA loads of cache blocks, for the attention
// kernels.
#pragma once
#include <cuda.h>

#include <mutex>

#include "paged_attn.cuh"

namespace xb {
namespace {

constexpr unsigned long long kWaitNs = 2000000000ull;  // of %globaltimer

// Set when a wait in one of this file's kernels has run out.
__device__ int g_wait_error, g_wait_taken;

__global__ void take_error_kernel() { g_wait_taken = atomicExch(&g_wait_error, 0); }

// Reads and clears the word in one step, so that none is lost that a kernel of
// another thread sets meanwhile.  The caller has waited for the device.
inline cudaError_t take_wait_error(int* out) {
    static std::mutex one;  // at a time: g_wait_taken is shared
    std::lock_guard<std::mutex> lock(one);
    const cudaError_t e = cudaLaunchKernel(take_error_kernel, dim3(1), dim3(1), nullptr, 0, nullptr);
    return e != cudaSuccess ? e : cudaMemcpyFromSymbol(out, g_wait_taken, sizeof(int));
}

__device__ __forceinline__ void bar_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_addr(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase; false when 2 s have passed or another wait has given up.
__device__ __forceinline__ bool bar_wait_slow(uint64_t* b, uint32_t parity, volatile int* dead) {
    const unsigned long long t0 = now_ns();
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (bar_try(b, parity)) return true;
        if (dead && *dead) return false;
        if (now_ns() - t0 > kWaitNs) {
            if (dead) *dead = 1;
            atomicExch(&g_wait_error, 1);
            return false;
        }
    }
}
// For one thread.
__device__ __forceinline__ bool bar_wait_one(uint64_t* b, uint32_t parity, volatile int* dead) {
    return bar_try(b, parity) || bar_try(b, parity) || bar_wait_slow(b, parity, dead);
}
// For a warp: it goes on, or gives up, as one.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* dead) {
    return __all_sync(0xffffffffu, bar_wait_one(b, parity, dead));
}

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                        int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Map of K or V with boxes of 64 values by box_tokens tokens, 128-byte swizzled in
// shared memory; what lies outside the cache reads as zeros.
inline bool cache_map(CUtensorMap* map, const struct b200_kv_cache& kv, void* data, int box_tokens) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.head_dim), static_cast<cuuint64_t>(kv.block_size),
                                static_cast<cuuint64_t>(kv.kv_heads), static_cast<cuuint64_t>(kv.num_blocks)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(kv.nb_token), static_cast<cuuint64_t>(kv.nb_head),
                                   static_cast<cuuint64_t>(kv.nb_block)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_tokens), 1, 1}, ones[4] = {1, 1, 1, 1};
    const EncodeFn encode = encode_fn();
    return encode &&
           encode(map,
                       kv.type == GGML_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                       data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace xb
