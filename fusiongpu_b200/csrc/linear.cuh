// linear.cuh -- what the linear layer's kernels share: shapes, activations and the
// epilogue (linear.cu, linear_tc.cu).
#pragma once

#include "adapter_common.cuh"
#include "packed.cuh"

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

// GELU = z Phi(z).  float32 results: CUDA's erfc, which keeps the small tail.
// Results rounded to 16 bits (FAST): with a = |z| / sqrt(2), t = 1 / (1 + 0.3275911 a)
// and e = exp(-a^2), erfc(a) = e t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) + 1.5e-7
// (Abramowitz and Stegun 7.1.26): two special-function and a dozen other
// operations, where erff would bound the epilogue.  e also serves the
// derivative Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi).
__device__ __forceinline__ float upper_tail(float z, float& e) {  // Phi(-|z|)
    const float t = __fdividef(1.0f, fmaf(fabsf(z), 0.3275911f * 0.70710678f, 1.0f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * z * (-0.5f * 1.44269504f)));
    float p = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    p = fmaf(t, p, 0.5f * 1.421413741f);
    p = fmaf(t, p, 0.5f * -0.284496736f);
    p = fmaf(t, p, 0.5f * 0.254829592f);
    return p * t * e;
}

// GELU of two values for results of 16 bits: max(z, 0) - a Phi(-a), a = min(|z|, 30)
// (Phi(-30) is 0 in float32), the formula of upper_tail in 9 issues a value.
__device__ __forceinline__ void gelu2(float& z0, float& z1) {
    const float a0 = fminf(fabsf(z0), 30.0f), a1 = fminf(fabsf(z1), 30.0f);
    const uint64_t a = pair2(a0, a1);
    float d0, d1, m0, m1;
    unpair2(fma2(a, pair2(0.3275911f * 0.70710678f, 0.3275911f * 0.70710678f), pair2(1.0f, 1.0f)), d0, d1);
    unpair2(mul2(mul2(a, a), pair2(-0.5f * 1.44269504f, -0.5f * 1.44269504f)), m0, m1);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d1));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(m0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(m1));
    const uint64_t t = pair2(d0, d1);
    uint64_t p = fma2(t, pair2(-0.5f * 1.061405429f, -0.5f * 1.061405429f), pair2(0.5f * 1.453152027f, 0.5f * 1.453152027f));
    p = fma2(t, p, pair2(-0.5f * 1.421413741f, -0.5f * 1.421413741f));
    p = fma2(t, p, pair2(0.5f * 0.284496736f, 0.5f * 0.284496736f));
    p = fma2(t, p, pair2(-0.5f * 0.254829592f, -0.5f * 0.254829592f));
    p = mul2(mul2(p, t), pair2(m0, m1));
    float r0, r1;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r0) : "f"(z0));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r1) : "f"(z1));
    unpair2(fma2(a, p, pair2(r0, r1)), z0, z1);
}

template <bool FAST>
__device__ __forceinline__ float sigmoid(float z) {  // z >= -100
    // below -87 the quotient's divisor would pass 2^126, where __fdividef is 0
    if (FAST) return __fdividef(z < -87.0f ? 0.0f : 1.0f, 1.0f + __expf(z < -87.0f ? 87.0f : -z));
    return 1.0f / (1.0f + expf(-z));
}

template <bool FAST>
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case FG_ACT_RELU: return z > 0.0f ? z : (z == z ? 0.0f : z);
        case FG_ACT_GELU: {
            if (!FAST) return fmaxf(z, -100.0f) * (0.5f * erfcf(z * -0.70710678f));
            float other = z;
            gelu2(z, other);
            return z;
        }
        case FG_ACT_SILU:
            z = z < -100.0f ? -100.0f : z;  // a NaN stays
            return z * sigmoid<FAST>(z);
        default: return z;
    }
}

template <bool FAST>
__device__ __forceinline__ float activate_grad(float z, int act) {
    switch (act) {
        case FG_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case FG_ACT_GELU: {
            const float zc = fminf(fmaxf(z, -100.0f), 100.0f);
            if (!FAST) return fmaf(zc, expf(-0.5f * z * z) * 0.39894228f, 0.5f * erfcf(z * -0.70710678f));
            float e;
            const float q = upper_tail(z, e);
            return fmaf(zc * 0.39894228f, e, z >= 0.0f ? 1.0f - q : q);
        }
        case FG_ACT_SILU: {
            z = z < -100.0f ? -100.0f : z > 100.0f ? 100.0f : z;
            const float s = sigmoid<FAST>(z);
            return s * fmaf(z, 1.0f - s, 1.0f);
        }
        default: return 1.0f;
    }
}

template <class T>
__device__ __forceinline__ void epilogue_store(const Epilogue& e, long long m, long long n, float z) {
    if (e.bias) z += to_f32(static_cast<const T*>(e.bias)[n]);
    if (e.pre) static_cast<T*>(e.pre)[m * e.ldp + n] = from_f32<T>(z);
    float y = activate<sizeof(T) == 2>(z, e.act);
    if (e.residual) y += to_f32(static_cast<const T*>(e.residual)[m * e.ldr + n]);
    static_cast<T*>(e.y)[m * e.ldy + n] = from_f32<T>(y);
}

// Tensor-core product of 16-bit operands (linear_tc.cu).  tc_gemm_fits: the
// operands' rows start on 16-byte boundaries, as their TMA loads need.
bool tc_gemm_fits(const void* a, const void* b, const GemmShape& g);
int tc_gemm(int dtype, const void* a, const void* b, const GemmShape& g, const Epilogue& e, cudaStream_t s);

}  // namespace fg
