// What the operator kernels (kv_cache.cu, q4_matmul.cu, logprobs.cu) share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../internal.hpp"

namespace csdr {

// Lets the kernel behind on the stream start its own prologue, then waits until everything before on the
// stream has completed and is visible: no global memory is touched before.
__device__ __forceinline__ void op_enter() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The kernel must begin with op_enter(), or have its two halves in an order of its own. cluster: CTAs of a cluster along x (1: none).
template <typename... KArgs, typename... Args>
void launch_op(csdr_context* ctx, void (*kern)(KArgs...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ctx->pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CSDR_CUDA(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"      // once: mbar_wait has the limit
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0u;
}
// How long a kernel that has given up waits for its own copies, which write into its shared memory until they are done.
constexpr uint32_t kDrainRounds = 4000000u;
// The whole warp waits, and gives up as one.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t limit) {
    if (__all_sync(0xFFFFFFFFu, mbar_try(bar, parity))) return true;
    for (uint32_t spin = 0; spin < limit; ++spin)
        if (__all_sync(0xFFFFFFFFu, mbar_try(bar, parity))) return true;
    return false;
}
// Where a kernel's first wait is: without a limit it is given up whatever it finds (CSDR_WAIT_GIVE_UP).
__device__ __forceinline__ bool mbar_wait_first(uint32_t bar, uint32_t parity, uint32_t limit) {
    return mbar_wait(bar, parity, limit) && limit != 0u;
}

__device__ __forceinline__ float op_widen(float v) { return v; }
__device__ __forceinline__ float op_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float op_widen(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T op_narrow(float v);
template <>
__device__ __forceinline__ float op_narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 op_narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half op_narrow<__half>(float v) { return __float2half_rn(v); }

// Eight elements that leave in 128-bit pieces.
template <typename T>
struct alignas(16) Eight128 {
    T v[8];
    __device__ __forceinline__ void store(T* to) const {
        static_assert(sizeof(*this) % sizeof(uint4) == 0 && alignof(Eight128) >= alignof(uint4), "whole pieces");
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2u; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(v)[i];
    }
};

// Calls f with a null pointer of the element type that a CSDR_DTYPE_* stands for.
template <typename F>
void with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case CSDR_DTYPE_F32: f(static_cast<float*>(nullptr)); break;
        case CSDR_DTYPE_BF16: f(static_cast<__nv_bfloat16*>(nullptr)); break;
        case CSDR_DTYPE_F16: f(static_cast<__half*>(nullptr)); break;
        default: throw Error(CSDR_ERR_INVALID_ARG, "unknown dtype");
    }
}

}  // namespace csdr
