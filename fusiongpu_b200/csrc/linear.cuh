// linear.cuh -- what the linear layer's kernels share: shapes, activations and the
// epilogue (linear.cu, linear_tc.cu).
#pragma once

#include "adapter_common.cuh"

namespace fg {

struct Epilogue {
    const void *bias, *residual;
    void *pre, *y;
    long long ldr, ldp, ldy;
    int act;
};

// C(m, n) = sum over k of A(m, k) B(n, k); strides per index.
struct GemmShape {
    long long m, n, k;
    long long am, ak, bn, bk;
};

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case FG_ACT_RELU: return z > 0.0f ? z : (z == z ? 0.0f : z);
        case FG_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678f));
        case FG_ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}

__device__ __forceinline__ float activate_grad(float z, int act) {
    switch (act) {
        case FG_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case FG_ACT_GELU:
            return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * expf(-0.5f * z * z) * 0.39894228f;
        case FG_ACT_SILU: {
            const float s = 1.0f / (1.0f + expf(-z));
            return s * (1.0f + z * (1.0f - s));
        }
        default: return 1.0f;
    }
}

template <class T>
__device__ __forceinline__ void epilogue_store(const Epilogue& e, long long m, long long n, float z) {
    if (e.bias) z += to_f32(static_cast<const T*>(e.bias)[n]);
    if (e.pre) static_cast<T*>(e.pre)[m * e.ldp + n] = from_f32<T>(z);
    float y = activate(z, e.act);
    if (e.residual) y += to_f32(static_cast<const T*>(e.residual)[m * e.ldr + n]);
    static_cast<T*>(e.y)[m * e.ldy + n] = from_f32<T>(y);
}

// Tensor-core product of 16-bit operands (linear_tc.cu).  tc_gemm_fits: the
// operands' rows start on 16-byte boundaries, as their TMA loads need.
bool tc_gemm_fits(const void* a, const void* b, const GemmShape& g);
int tc_gemm(int dtype, const void* a, const void* b, const GemmShape& g, const Epilogue& e, cudaStream_t s);

}  // namespace fg
