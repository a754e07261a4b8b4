// What the kernels of the language-model operators share: element types, vectors, notification, launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <llis/job/finished_block_notifier.h>

#include <cstring>
#include <type_traits>

#include "launch_slot.cuh"
#include "ops.h"
#include "pb_common.h"

namespace pb {

using llis::job::FinishedBlockNotifier;

// Codes of the error flag.
constexpr uint32_t kFlagLmPosition = 0x301, kFlagLmSlot = 0x302, kFlagLmLength = 0x303, kFlagLmPage = 0x304, kFlagLmToken = 0x305, kFlagLmWait = 0x310;

inline size_t dtype_bytes(int dtype) { return dtype == PB_F32 ? 4 : 2; }
inline bool is_float_dtype(int dtype) { return dtype == PB_F32 || dtype == PB_BF16 || dtype == PB_F16; }
inline bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }
// Rows of `length` elements, `stride` apart in either direction, do not lie over their neighbours.
inline bool rows_apart(int64_t count, int64_t stride, int64_t length) { return count <= 1 || stride >= length || stride <= -length; }

template <typename F>
uint32_t lm_regs(F fn) {
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, fn) != cudaSuccess) { cudaGetLastError(); return 0; }
    return (uint32_t)a.numRegs;
}

// Launches `kern` as a programmatic dependent of what precedes it in the stream: its blocks may come in, and set themselves up, while a
// predecessor that lets them still runs; all of them wait for its end (griddep_wait) before they touch memory.
template <typename... KArgs, typename... Args>
int lm_launch(const char* what, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("launch of %s failed: %s", what, cudaGetErrorString(e));
        return PB_ERR_CUDA;
    }
    return PB_OK;
}

#ifdef __CUDACC__
template <typename T> __device__ __forceinline__ float lm_to_f(T x);
template <> __device__ __forceinline__ float lm_to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float lm_to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float lm_to_f<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T lm_from_f(float x);
template <> __device__ __forceinline__ float lm_from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 lm_from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half lm_from_f<__half>(float x) { return __float2half_rn(x); }
template <typename T> __device__ __forceinline__ uint32_t lm_pack2(float lo, float hi);   // lo in the lower half
template <> __device__ __forceinline__ uint32_t lm_pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t lm_pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// N values as one access of N * sizeof(T) bytes (a power of two, at most 16), aligned to it.
template <typename T, int N> struct alignas(sizeof(T) * N) LmVec {
    T v[N];
};
#endif

}  // namespace pb
