// linear.cu -- linear layer with bias, activation and residual in its epilogue,
// and its gradients.
//
//   z = x w^T + bias,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  dbias = sum over rows of dz
#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace fg {

constexpr int SG_T = 64, SG_K = 16;

// 64 x 64 tile per block of 256 threads, 4 x 4 outputs each, fp32 FMA.
template <class T>
__global__ void __launch_bounds__(256) gemm_simt_kernel(const T* a, const T* b, const GemmShape g, const Epilogue e) {
    __shared__ float sa[SG_K][SG_T + 1], sb[SG_K][SG_T + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long nt = (g.n + SG_T - 1) / SG_T;
    const long long m0 = blockIdx.x / nt * SG_T, n0 = blockIdx.x % nt * SG_T;
    float acc[4][4] = {};
    for (long long k0 = 0; k0 < g.k; k0 += SG_K) {
        for (int i = threadIdx.x; i < SG_T * SG_K; i += 256) {
            // the fast index follows the unit stride of the operand
            const int ra = g.ak == 1 ? i / SG_K : i % SG_T, ka = g.ak == 1 ? i % SG_K : i / SG_T;
            const int rb = g.bk == 1 ? i / SG_K : i % SG_T, kb = g.bk == 1 ? i % SG_K : i / SG_T;
            sa[ka][ra] = (m0 + ra < g.m && k0 + ka < g.k) ? to_f32(a[(m0 + ra) * g.am + (k0 + ka) * g.ak]) : 0.0f;
            sb[kb][rb] = (n0 + rb < g.n && k0 + kb < g.k) ? to_f32(b[(n0 + rb) * g.bn + (k0 + kb) * g.bk]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < SG_K; ++k) {
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = sa[k][ty + 16 * i];
                y[i] = sb[k][tx + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < g.m && n < g.n) epilogue_store<T>(e, m, n, acc[i][j]);
        }
}

template <class T>
static int gemm(const void* a, const void* b, const GemmShape& g, const Epilogue& e, void* ws, cudaStream_t s) {
    const long long tiles = ((g.m + SG_T - 1) / SG_T) * ((g.n + SG_T - 1) / SG_T);
    FG_REQUIRE(tiles <= 0x7fffffffll, "%lld x %lld outputs: too many tiles", g.m, g.n);
    if (tiles == 0) return FG_OK;
    if (sizeof(T) == 2 && tc_gemm_fits(a, b, g))
        return tc_gemm(std::is_same<T, __half>::value ? FG_DTYPE_F16 : FG_DTYPE_BF16, a, b, g, e, ws, s);
    gemm_simt_kernel<T><<<(unsigned)tiles, 256, 0, s>>>(static_cast<const T*>(a), static_cast<const T*>(b), g, e);
    return check_launch("gemm_simt_kernel");
}

// dz = dy act'(pre) and the column sums of dz, in one pass over dy and pre: a warp
// takes 32 x VEC columns of every eighth row of its block's range, two rows at a
// time, sums them in registers, and the block writes one partial row.  Memory-bound;
// DZFIG
constexpr int DZ_WARPS = 8;

struct DzArgs {
    const void *dy, *pre;
    void* dz;     // NULL: not stored
    float* part;  // NULL: no sums
    long long lddy, ldp, rows, per;
    int dim, act, wide;
};

template <class T, int VEC>
__device__ __forceinline__ void dz_load(T (&v)[VEC], const T* p, int left, int wide) {
    if (wide && left >= VEC) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < left) v[i] = p[i];
    }
}

// dy act'(pre) of two columns.
template <int ACT, bool FAST>
__device__ __forceinline__ void dz_pair(float& d0, float& d1, float p0, float p1) {
    if (ACT == FG_ACT_NONE) return;
    if (ACT == FG_ACT_GELU && FAST) {
        gelu_grad2(p0, p1);
    } else {
        p0 = activate_grad<FAST>(p0, ACT);
        p1 = activate_grad<FAST>(p1, ACT);
    }
    unpair2(mul2(pair2(d0, d1), pair2(p0, p1)), d0, d1);
}

template <class T, int ACT>
__global__ void __launch_bounds__(DZ_WARPS * 32) dz_kernel(const DzArgs g) {
    constexpr int VEC = 16 / sizeof(T), U = 2;
    __shared__ float s[DZ_WARPS][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = (blockIdx.x * 32 + lane) * VEC, left = g.dim - j;
    const long long r0 = blockIdx.y * g.per, r1 = min(r0 + g.per, g.rows);
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
    if (left > 0)
        for (long long r = r0 + warp; r < r1; r += U * DZ_WARPS) {
            alignas(16) T d[U][VEC], p[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long q = r + u * DZ_WARPS;
                if (q < r1) {
                    dz_load<T, VEC>(d[u], static_cast<const T*>(g.dy) + q * g.lddy + j, left, g.wide);
                    if (ACT != FG_ACT_NONE) dz_load<T, VEC>(p[u], static_cast<const T*>(g.pre) + q * g.ldp + j, left, g.wide);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long q = r + u * DZ_WARPS;
                if (q >= r1) break;
                alignas(16) T o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i += 2) {
                    float v0 = to_f32(d[u][i]), v1 = to_f32(d[u][i + 1]);
                    dz_pair<ACT, sizeof(T) == 2>(v0, v1, to_f32(p[u][i]), to_f32(p[u][i + 1]));
                    v0 = i < left ? v0 : 0.0f;  // columns past the last
                    v1 = i + 1 < left ? v1 : 0.0f;
                    sum[i] += v0;
                    sum[i + 1] += v1;
                    o[i] = from_f32<T>(v0);
                    o[i + 1] = from_f32<T>(v1);
                }
                if (g.dz) {  // rows of dz are padded to 16 bytes
                    T* out = static_cast<T*>(g.dz) + q * ((g.dim + VEC - 1) / VEC * VEC) + j;
                    *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(o);
                }
            }
        }
    if (!g.part) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[warp][lane * VEC + i] = sum[i];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * VEC; c += DZ_WARPS * 32) {
        const int col = blockIdx.x * 32 * VEC + c;
        if (col >= g.dim) break;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < DZ_WARPS; ++w) v += s[w][c];
        g.part[(size_t)blockIdx.y * g.dim + col] = v;
    }
}

// Adds the partial rows: 32 columns per block, warp w the rows w, w + 32, ... in
// order, then the warps in order.
template <class T>
__global__ void __launch_bounds__(1024) dz_reduce_kernel(const float* part, int parts, int dim, T* dbias) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (j < dim) {
#pragma unroll 4
        for (int p = warp; p < parts; p += 32) v += part[(size_t)p * dim + j];
    }
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && j < dim) {
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) v += s[w][lane];
        dbias[j] = from_f32<T>(v);
    }
}

// Row ranges: four blocks to an SM over the column tiles, 16 rows at least to a range.
static int dz_split(long long rows, int dim, int elem) {
    const int cols = 32 * (16 / elem), tiles = (dim + cols - 1) / cols;
    const long long fill = std::max(1ll, 4ll * std::max(1, device_attr(cudaDevAttrMultiProcessorCount)) / tiles);
    return (int)std::max(1ll, std::min(fill, (rows + 15) / 16));
}

template <class T>
static int launch_dz(DzArgs g, int split, cudaStream_t s) {
    constexpr int cols = 32 * (16 / (int)sizeof(T));
    g.per = (g.rows + split - 1) / split;
    auto lies = [&](const void* p, long long ld) { return !p || (aligned(p, 16) && ld * (int)sizeof(T) % 16 == 0); };
    g.wide = lies(g.dy, g.lddy) && lies(g.pre, g.ldp);
    const dim3 grid((g.dim + cols - 1) / cols, split);
    switch (g.act) {
        case FG_ACT_RELU: dz_kernel<T, FG_ACT_RELU><<<grid, DZ_WARPS * 32, 0, s>>>(g); break;
        case FG_ACT_GELU: dz_kernel<T, FG_ACT_GELU><<<grid, DZ_WARPS * 32, 0, s>>>(g); break;
        case FG_ACT_SILU: dz_kernel<T, FG_ACT_SILU><<<grid, DZ_WARPS * 32, 0, s>>>(g); break;
        default: dz_kernel<T, FG_ACT_NONE><<<grid, DZ_WARPS * 32, 0, s>>>(g);
    }
    return check_launch("dz_kernel");
}

struct Strides {
    long long x, w, r, p, y;
};

static int linear_check(const fg_linear_params* p, Strides& t) {
    FG_REQUIRE(p, "null params");
    FG_REQUIRE(p->rows >= 0 && p->in_dim >= 1 && p->out_dim >= 1, "bad linear shape");
    FG_REQUIRE(float_dtype(p->dtype), "unknown dtype %d", p->dtype);
    FG_REQUIRE(p->activation >= FG_ACT_NONE && p->activation <= FG_ACT_SILU, "unknown activation %d", p->activation);
    t.x = p->x_stride ? p->x_stride : p->in_dim;
    t.w = p->w_stride ? p->w_stride : p->in_dim;
    t.r = p->residual_stride ? p->residual_stride : p->out_dim;
    t.p = p->pre_stride ? p->pre_stride : p->out_dim;
    t.y = p->y_stride ? p->y_stride : p->out_dim;
    FG_REQUIRE(t.x >= p->in_dim && t.w >= p->in_dim && t.r >= p->out_dim && t.p >= p->out_dim && t.y >= p->out_dim,
               "row stride below the row length");
    return FG_OK;
}

// Products of a layer: z = x w^T, dx = dz w, dw = dz^T x.
static GemmShape forward_shape(const fg_linear_params* p, const Strides& t) {
    return {p->rows, p->out_dim, p->in_dim, t.x, 1, t.w, 1};
}
static GemmShape dx_shape(const fg_linear_params* p, const Strides& t, long long ldz) {
    return {p->rows, p->in_dim, p->out_dim, ldz, 1, 1, t.w};
}
static GemmShape dw_shape(const fg_linear_params* p, const Strides& t, long long ldz) {
    return {p->out_dim, p->in_dim, p->rows, 1, ldz, 1, t.x};
}

struct BackwardWs {
    void *dz, *product;
    float* part;
};

static long long dz_stride(const fg_linear_params* p) {
    const int vec = 16 / dtype_size(p->dtype);
    return (long long)(p->out_dim + vec - 1) / vec * vec;
}

static size_t backward_carve(const fg_linear_params* p, const Strides& t, void* ws, size_t bytes, BackwardWs& w) {
    Carve c(ws, bytes);
    const size_t n = p->dtype == FG_DTYPE_F32 ? 0
                                              : std::max(tc_gemm_workspace(dx_shape(p, t, t.y)),
                                                         tc_gemm_workspace(dw_shape(p, t, t.y)));
    w.product = n ? c.take<char>(n) : nullptr;
    w.dz = p->activation == FG_ACT_NONE ? nullptr : c.take<char>((size_t)p->rows * dz_stride(p) * dtype_size(p->dtype));
    w.part = c.take<float>((size_t)dz_split(p->rows, p->out_dim, dtype_size(p->dtype)) * p->out_dim);
    return c.used;
}

template <class T>
static int linear_backward(const fg_linear_params* p, const Strides& t, const void* dy, const void* x, const void* w,
                           const void* pre, void* dx, void* dw, void* dbias, const BackwardWs& ws, cudaStream_t s) {
    const bool act = p->activation != FG_ACT_NONE, store = act && (dx || dw);
    const int split = p->rows ? dz_split(p->rows, p->out_dim, sizeof(T)) : 0;
    int rc;
    if (split && (store || dbias)) {
        const DzArgs g{dy, act ? pre : nullptr, store ? ws.dz : nullptr, dbias ? ws.part : nullptr, t.y, t.p, p->rows, 0,
                       p->out_dim, p->activation, 0};
        if ((rc = launch_dz<T>(g, split, s))) return rc;
    }
    if (dbias) {
        dz_reduce_kernel<T><<<(p->out_dim + 31) / 32, 1024, 0, s>>>(ws.part, split, p->out_dim, (T*)dbias);
        if ((rc = check_launch("dz_reduce_kernel"))) return rc;
    }
    const void* dz = act ? ws.dz : dy;
    const long long ldz = act ? dz_stride(p) : t.y;
    Epilogue e{};
    if (dx && p->rows) {
        e.y = dx;
        e.ldy = p->in_dim;
        rc = gemm<T>(dz, w, dx_shape(p, t, ldz), e, ws.product, s);
        if (rc) return rc;
    }
    if (dw) {
        e.y = dw;
        e.ldy = p->in_dim;
        rc = gemm<T>(dz, x, dw_shape(p, t, ldz), e, ws.product, s);
        if (rc) return rc;
    }
    return FG_OK;
}

}  // namespace fg

using namespace fg;

extern "C" {

int fg_linear_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        Strides t;
        const int rc = linear_check(params, t);
        if (rc) return rc;
        *bytes = params->dtype == FG_DTYPE_F32 || params->rows == 0 ? 0 : tc_gemm_workspace(forward_shape(params, t));
        return FG_OK;
    });
}

int fg_linear(const fg_linear_params* params, const void* x, const void* w, const void* bias, const void* residual,
              void* pre, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&]() -> int {
        Strides t;
        const int rc = linear_check(params, t);
        if (rc) return rc;
        if (params->rows == 0) return FG_OK;
        FG_REQUIRE(x && w && y, "null buffer");
        const GemmShape g = forward_shape(params, t);
        if (params->dtype != FG_DTYPE_F32 && tc_gemm_fits(x, w, g)) {
            const int bad = adapter_ws(workspace, workspace_bytes, tc_gemm_workspace(g));
            if (bad) return bad;
        }
        const Epilogue e{bias, residual, pre, y, t.r, t.p, t.y, params->activation};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return params->dtype == FG_DTYPE_F32   ? gemm<float>(x, w, g, e, workspace, s)
               : params->dtype == FG_DTYPE_F16 ? gemm<__half>(x, w, g, e, workspace, s)
                                               : gemm<__nv_bfloat16>(x, w, g, e, workspace, s);
    });
}

int fg_linear_backward_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        Strides t;
        const int rc = linear_check(params, t);
        if (rc) return rc;
        BackwardWs w;
        *bytes = backward_carve(params, t, nullptr, 0, w);
        return FG_OK;
    });
}

int fg_linear_backward(const fg_linear_params* params, const void* dy, const void* x, const void* w, const void* pre,
                       void* dx, void* dw, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&]() -> int {
        Strides t;
        int rc = linear_check(params, t);
        if (rc) return rc;
        if (params->rows) {
            FG_REQUIRE(dy, "null dy");
            FG_REQUIRE(!dx || w, "dx needs w");
            FG_REQUIRE(!dw || x, "dw needs x");
            FG_REQUIRE(params->activation == FG_ACT_NONE || pre, "the activation's gradient needs pre");
        }
        BackwardWs ws;
        rc = adapter_ws(workspace, workspace_bytes, backward_carve(params, t, nullptr, 0, ws));
        if (rc) return rc;
        backward_carve(params, t, workspace, workspace_bytes, ws);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return params->dtype == FG_DTYPE_F32 ? linear_backward<float>(params, t, dy, x, w, pre, dx, dw, dbias, ws, s)
               : params->dtype == FG_DTYPE_F16
                   ? linear_backward<__half>(params, t, dy, x, w, pre, dx, dw, dbias, ws, s)
                   : linear_backward<__nv_bfloat16>(params, t, dy, x, w, pre, dx, dw, dbias, ws, s);
    });
}

}  // extern "C"
