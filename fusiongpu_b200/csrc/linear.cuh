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
    bool any_parts = false;  // k may be split among pairs into 3, 5, ... parts as well as powers of two
};

// GELU = z Phi(z).  float32 results: CUDA's erfc.  Results of 16 bits (FAST): fits of our
// own, least in their largest weighted error over 0 <= a <= 14, that keep the relative
// accuracy of the tail Phi(-a), as such results show it.
//   value:      max(z, 0) - a Phi(-a), a = |z|.  Phi(-a) = 2^P(a), P of degree 9: off by
//               2^-16.7 of the value down to z = -6 (float16's last results) and 2^-12.8
//               to -13 (bfloat16's).  One special-function operation a value, which with
//               the other issues balances the epilogue (two are 4,096 cycles of a tile's
//               6,144 of products)
//   derivative: T for z < 0, 1 - T otherwise, T = Phi(-a) - a phi(a) = exp(-a^2 / 2) (M -
//               a / sqrt(2 pi)), M(a) = t Q(t), t = 1 / (1 + 0.26 a), Q of degree 6: off by
//               2^-22 near 0 and 2^-19 of the value from -1 to -8
// GELU of two values; 2^24 in P's constant and back keeps Phi(-13) off exp2's underflow.
__device__ __forceinline__ void gelu2(float& z0, float& z1) {
    const uint64_t a = pair2(fminf(fabsf(z0), 14.0f), fminf(fabsf(z1), 14.0f));
    auto both = [](float c) { return pair2(c, c); };
    uint64_t p = fma2(a, both(-2.12431917e-09f), both(1.53519707e-07f));
    p = fma2(a, p, both(-4.85575265e-06f));
    p = fma2(a, p, both(8.9097688e-05f));
    p = fma2(a, p, both(-0.00106443313f));
    p = fma2(a, p, both(0.00886763725f));
    p = fma2(a, p, both(-0.054471042f));
    p = fma2(a, p, both(-0.458130389f));
    p = fma2(a, p, both(-1.15131855f));
    p = fma2(a, p, both(23.0000038f));
    float q0, q1, r0, r1;
    unpair2(p, q0, q1);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(q0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(q1));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r0) : "f"(z0));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r1) : "f"(z1));
    unpair2(fma2(mul2(a, both(-5.9604645e-08f)), pair2(q0, q1), pair2(r0, r1)), z0, z1);
}

// GELU's derivative of two values; z held to [-30, 30], a NaN stays.
__device__ __forceinline__ void gelu_grad2(float& z0, float& z1) {
    float c0, c1, d0, d1, m0, m1, t0, t1;
    asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC1F00000;\n\tmin.NaN.f32 %0, t, 0f41F00000;\n\t}" : "=f"(c0) : "f"(z0));
    asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC1F00000;\n\tmin.NaN.f32 %0, t, 0f41F00000;\n\t}" : "=f"(c1) : "f"(z1));
    auto both = [](float c) { return pair2(c, c); };
    const uint64_t a = pair2(fabsf(c0), fabsf(c1));
    unpair2(fma2(a, both(0.26f), both(1.0f)), d0, d1);
    unpair2(mul2(mul2(a, a), both(-0.5f * 1.44269504f)), m0, m1);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d1));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(m0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(m1));
    const uint64_t t = pair2(d0, d1);
    uint64_t p = fma2(t, both(-0.0721131678f), both(0.225167564f));
    p = fma2(t, p, both(-0.0996524985f));
    p = fma2(t, p, both(0.160275265f));
    p = fma2(t, p, both(0.0762695383f));
    p = fma2(t, p, both(0.106471479f));
    p = fma2(t, p, both(0.10358178f));
    unpair2(mul2(pair2(m0, m1), fma2(a, both(-0.39894228f), mul2(p, t))), t0, t1);
    z0 = c0 < 0.0f ? t0 : 1.0f - t0;
    z1 = c1 < 0.0f ? t1 : 1.0f - t1;
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
            if (FAST) {
                float other = z;
                gelu_grad2(z, other);
                return z;
            }
            const float zc = fminf(fmaxf(z, -100.0f), 100.0f);
            return fmaf(zc, expf(-0.5f * z * z) * 0.39894228f, 0.5f * erfcf(z * -0.70710678f));
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

// Gated layer: a gate's z and its partner's, columns n and up + n.
template <class T>
__device__ __forceinline__ void gated_store(const Epilogue& e, int up, long long m, long long n, float z, float p) {
    if (e.bias) {
        z += to_f32(static_cast<const T*>(e.bias)[n]);
        p += to_f32(static_cast<const T*>(e.bias)[up + n]);
    }
    if (e.pre) {
        static_cast<T*>(e.pre)[m * e.ldp + n] = from_f32<T>(z);
        static_cast<T*>(e.pre)[m * e.ldp + up + n] = from_f32<T>(p);
    }
    static_cast<T*>(e.y)[m * e.ldy + n] = from_f32<T>(activate<sizeof(T) == 2>(z, e.act) * p);
}

// A 32-bit value as two of 16 bits, for an operand that is worked out in 32: the
// rounding to the type, and the rounding of what that leaves.  bf16: v = p0 + p1, to 16
// bits of the significand.  f16: v = 2 (p0 + 2^-12 p1), to 22 bits, or 2^-36 where that is
// more: a gradient may lie below f16's 2^-24 and up to 1.13 times its largest value.  An
// infinity or NaN has 0 behind it.
//
// A gated layer's dz = dy p act'(z) may pass that range as well, up to 2^32.2.  Such an f16
// value is a NaN, whose payload and lower part hold its bits from F16_FAR on, rounded to
// 2^-21 of it; the results that it enters come out as NaN and are taken again one product
// at a time, from of_parts.
constexpr int F16_PART_SHIFT = 12;
constexpr uint32_t F16_FAR = 0x47800000u;  // 2^16
template <class T>
struct PartsOf {  // v = hi p0 + lo p1
    static constexpr float hi = 1.0f, lo = 1.0f;
};
template <>
struct PartsOf<__half> {
    static constexpr float hi = 2.0f, lo = 2.0f / (1 << F16_PART_SHIFT);
};
__device__ __forceinline__ void split2(float v, __nv_bfloat16& p0, __nv_bfloat16& p1) {
    p0 = from_f32<__nv_bfloat16>(v);
    const bool finite = fabsf(v) <= FLT_MAX;
    if (finite && !(fabsf(to_f32(p0)) <= FLT_MAX)) p0 = from_f32<__nv_bfloat16>(__uint_as_float(__float_as_uint(v) & 0xffff0000u));
    p1 = from_f32<__nv_bfloat16>(finite ? v - to_f32(p0) : 0.0f);
}
__device__ __forceinline__ void split2(float v, __half& p0, __half& p1) {
    const float h = v * 0.5f;
    p0 = from_f32<__half>(h);
    if (fabsf(v) <= FLT_MAX && fabsf(to_f32(p0)) > 65504.0f) {
        const uint32_t u = ((__float_as_uint(v) & 0x7fffffffu) - F16_FAR + 4) >> 3;  // below 2^25 - 2^16, a plain NaN's
        p0 = __ushort_as_half((unsigned short)(0x7e00u | (u >> 16) | (v < 0.0f ? 0x8000u : 0u)));
        p1 = __ushort_as_half((unsigned short)u);
        return;
    }
    const float r = (h - to_f32(p0)) * (float)(1 << F16_PART_SHIFT);
    p1 = from_f32<__half>(fabsf(v) <= FLT_MAX ? fminf(fmaxf(r, -65504.0f), 65504.0f) : 0.0f);
}

// What the parts stand for.
template <class T>
__device__ __forceinline__ float of_parts(T p0, T p1) {
    return PartsOf<T>::hi * to_f32(p0) + PartsOf<T>::lo * to_f32(p1);
}
template <>
__device__ __forceinline__ float of_parts<__half>(__half p0, __half p1) {
    const uint32_t b = __half_as_ushort(p0);
    if ((b & 0x7e00u) == 0x7e00u && (b & 0x7fffu) != 0x7fffu) {
        const float v = __uint_as_float(F16_FAR + (((b & 0x1ffu) << 16 | __half_as_ushort(p1)) << 3));
        return b & 0x8000u ? -v : v;
    }
    return PartsOf<__half>::hi * to_f32(p0) + PartsOf<__half>::lo * to_f32(p1);
}

// The same of two values at once, which are ordinary ones: neither cut nor past the range.
__device__ __forceinline__ void split2(float v0, float v1, __nv_bfloat162& p0, __nv_bfloat162& p1) {
    if (!(fabsf(v0) < 3.3e38f && fabsf(v1) < 3.3e38f)) {
        split2(v0, p0.x, p1.x);
        split2(v1, p0.y, p1.y);
        return;
    }
    p0 = __floats2bfloat162_rn(v0, v1);
    const float2 f = __bfloat1622float2(p0);
    p1 = __floats2bfloat162_rn(v0 - f.x, v1 - f.y);
}
__device__ __forceinline__ void split2(float v0, float v1, __half2& p0, __half2& p1) {
    if (!(fabsf(v0) < 65000.0f && fabsf(v1) < 65000.0f)) {
        split2(v0, p0.x, p1.x);
        split2(v1, p0.y, p1.y);
        return;
    }
    constexpr float up = 1 << F16_PART_SHIFT;
    p0 = __floats2half2_rn(v0 * 0.5f, v1 * 0.5f);
    const float2 f = __half22float2(p0);  // up (v / 2 - f), exact but for its rounding
    p1 = __floats2half2_rn(fmaf(v0, 0.5f * up, f.x * -up), fmaf(v1, 0.5f * up, f.y * -up));
}

// Tensor-core product (linear_tc.cu) of 16-bit operands, A possibly in the two parts
// above, a_plane elements apart (0: as it is), or for F32 of three bf16 planes of each,
// a_plane and b_plane apart.  tc_gemm_fits: the operands' rows start on 16-byte
// boundaries, as their TMA loads need.  The workspace (256-byte aligned) holds the
// partial tiles of a split product; its size goes by the number of plane products.
inline int tc_products(int dtype, bool parts) { return dtype == FG_DTYPE_F32 ? 6 : parts ? 2 : 1; }
bool tc_gemm_fits(const void* a, const void* b, const GemmShape& g);
size_t tc_gemm_workspace(int products, const GemmShape& g);
// Gated layer: g.n = 2 up rows of B, up outputs.  Operands as tc_gemm takes them, B K-major,
// both of at most 32,768 k.
int tc_gated(int dtype, const void* a, long long a_plane, const void* b, long long b_plane, const GemmShape& g,
             const Epilogue& e, cudaStream_t s);
// Codes of 8 bits, both K-major, rows on 16-byte boundaries, at most 131,071 k.  dtype: of the
// epilogue's matrices.
int tc_int8(int dtype, const void* a, const float* xs, const void* b, const float* ws, const GemmShape& g, const Epilogue& e,
            cudaStream_t s);
int tc_gemm(int dtype, const void* a, long long a_plane, const void* b, long long b_plane, const GemmShape& g,
            const Epilogue& e, void* ws, cudaStream_t s);

// ---- the layer's host side (linear.cu), shared with the gated layer (gated.cu) --------

struct PackJob {
    const void* in;
    void* out;
    long long rows, ld, plane;
    int cols;
};
struct PackArgs {
    PackJob job[2];
    int jobs;
};

__host__ __device__ inline long long pack_stride(long long cols) { return (cols + 7) / 8 * 8; }

__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
    p[0] = from_f32<__nv_bfloat16>(x);
    const bool finite = fabsf(x) <= FLT_MAX;
    if (finite && !(fabsf(to_f32(p[0])) <= FLT_MAX)) p[0] = from_f32<__nv_bfloat16>(__uint_as_float(__float_as_uint(x) & 0xffff0000u));
    const float r = x - to_f32(p[0]);
    p[1] = from_f32<__nv_bfloat16>(finite ? r : 0.0f);
    p[2] = from_f32<__nv_bfloat16>(finite ? r - to_f32(p[1]) : 0.0f);
}

// An operand on its way to a product: as it lies, or packed into the workspace.
struct Operand {
    const void* p;
    long long ld, plane;  // elements
};

// `off`: it does not start on a 16-byte boundary either (10,000 x 768 -> 1536 f16: 43 us
// with x packed, 27 as it lies on one, 1,247 on the CUDA cores).
inline bool needs_pack(int dtype, long long ld, bool off) { return dtype == FG_DTYPE_F32 || ld % 8 != 0 || off; }
inline size_t pack_bytes(int dtype, long long rows, long long cols) {
    return (size_t)rows * pack_stride(cols) * 2 * (dtype == FG_DTYPE_F32 ? 3 : 1);
}

Operand operand(int dtype, const void* p, long long rows, int cols, long long ld, bool off, void* room, PackArgs& a);

constexpr int GEMV_ROWS = 8;  // rows that go without tensor cores

struct FewArgs {
    const void *dy, *x, *w, *pre;
    void *dx, *dw, *db;
    long long lddy, ldx, ldw, ldp;
    int rows, in_dim, out_dim, act, dx_blocks;
    int up;  // gated layer: out_dim / 2, pre [rows][out_dim], dy [rows][up]; else 0
};

struct Strides {
    long long x, w, r, p, y;
};

constexpr long long LINEAR_MAX = (1ll << 31) - 1024;  // tensor coordinates are 32 bits

int linear_check(const fg_linear_params* p, Strides& t);
bool few(const fg_linear_params* p);
int linear_pack(int dtype, const PackArgs& a, cudaStream_t s);
int linear_gemm(int dtype, const Operand& a, const Operand& b, const GemmShape& g, const Epilogue& e, void* ws, cudaStream_t s);
int linear_gemv_gated(int dtype, const void* x, const void* w, const GemmShape& g, const Epilogue& e, int up, cudaStream_t s);
int linear_few_rows(int dtype, const FewArgs& g, cudaStream_t s);
int linear_column_sums(int dtype, const float* part, int parts, int dim, void* out, cudaStream_t s);

}  // namespace fg
