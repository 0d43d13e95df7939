// adapter_common.cuh -- element types and small reductions shared by the query
// adapter's kernels (norm.cu, linear.cu, preference.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fg_common.cuh"

namespace fg {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(uint8_t v) { return (float)v; }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

inline bool float_dtype(int t) { return t == FG_DTYPE_F32 || t == FG_DTYPE_F16 || t == FG_DTYPE_BF16; }
inline int dtype_size(int t) { return t == FG_DTYPE_F32 ? 4 : t == FG_DTYPE_U8 ? 1 : 2; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over a block of NT threads, in every thread.  `s`: NT / 32 floats.
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* s) {
    v = warp_sum(v);
    __syncthreads();  // the previous call's readers are done with s
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) t += s[w];
    return t;
}

inline int adapter_ws(void* ws, size_t have, size_t need) {
    if (need == 0) return FG_OK;
    if (!ws) return fail(FG_ERR_WORKSPACE, "workspace is NULL (%zu bytes needed)", need);
    if (!aligned(ws, 256)) return fail(FG_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    if (have < need) return fail(FG_ERR_WORKSPACE, "workspace of %zu bytes < %zu needed", have, need);
    return FG_OK;
}

// Runs an entry point's body; no C++ exception leaves the C ABI.
template <class F>
int c_entry(F&& body) noexcept {
    try {
        return body();
    } catch (...) {
        return FG_ERR_CUDA;
    }
}

}  // namespace fg
