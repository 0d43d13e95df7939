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
static int gemm(const void* a, const void* b, const GemmShape& g, const Epilogue& e, cudaStream_t s) {
    const long long tiles = ((g.m + SG_T - 1) / SG_T) * ((g.n + SG_T - 1) / SG_T);
    FG_REQUIRE(tiles <= 0x7fffffffll, "%lld x %lld outputs: too many tiles", g.m, g.n);
    if (tiles == 0) return FG_OK;
    if (sizeof(T) == 2 && tc_gemm_fits(a, b, g))
        return tc_gemm(std::is_same<T, __half>::value ? FG_DTYPE_F16 : FG_DTYPE_BF16, a, b, g, e, s);
    gemm_simt_kernel<T><<<(unsigned)tiles, 256, 0, s>>>(static_cast<const T*>(a), static_cast<const T*>(b), g, e);
    return check_launch("gemm_simt_kernel");
}

constexpr int DZ_COLS = 32, DZ_SPLIT = 64;

// dz = dy act'(pre) (dz NULL: not stored) and the partial column sums of dz of
// each row range.
template <class T>
__global__ void __launch_bounds__(256) dz_kernel(const T* dy, long long lddy, const T* pre, long long ldp, int act,
                                                 long long rows, int dim, T* dz, float* part) {
    __shared__ float sb[8][DZ_COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * DZ_COLS + lane;
    const long long per = (rows + gridDim.y - 1) / gridDim.y;
    const long long r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float b = 0.0f;
    if (j < dim)
        for (long long r = r0 + warp; r < r1; r += 8) {
            float v = to_f32(dy[r * lddy + j]);
            if (act != FG_ACT_NONE) v *= activate_grad<sizeof(T) == 2>(to_f32(pre[r * ldp + j]), act);
            if (dz) dz[r * dim + j] = from_f32<T>(v);
            b += v;
        }
    if (!part) return;
    sb[warp][lane] = b;
    __syncthreads();
    if (warp == 0 && j < dim) {
        b = 0.0f;
        for (int i = 0; i < 8; ++i) b += sb[i][lane];
        part[(size_t)blockIdx.y * dim + j] = b;
    }
}

template <class T>
__global__ void dz_reduce_kernel(const float* part, int parts, int dim, T* dbias) {
    const int j = blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= dim) return;
    float v = 0.0f;
    for (int p = 0; p < parts; ++p) v += part[(size_t)p * dim + j];
    dbias[j] = from_f32<T>(v);
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

struct BackwardWs {
    void* dz;
    float* part;
};

static size_t backward_carve(const fg_linear_params* p, void* ws, size_t bytes, BackwardWs& w) {
    Carve c(ws, bytes);
    w.dz = p->activation == FG_ACT_NONE
               ? nullptr
               : c.take<char>((size_t)p->rows * p->out_dim * dtype_size(p->dtype));
    w.part = c.take<float>((size_t)DZ_SPLIT * p->out_dim);
    return c.used;
}

template <class T>
static int linear_backward(const fg_linear_params* p, const Strides& t, const void* dy, const void* x, const void* w,
                           const void* pre, void* dx, void* dw, void* dbias, const BackwardWs& ws, cudaStream_t s) {
    const bool act = p->activation != FG_ACT_NONE;
    const int split = (int)std::min<long long>(DZ_SPLIT, (p->rows + 7) / 8);
    int rc;
    if (split && (act || dbias)) {
        dz_kernel<T><<<dim3((p->out_dim + DZ_COLS - 1) / DZ_COLS, split), 256, 0, s>>>(
            (const T*)dy, t.y, (const T*)pre, t.p, p->activation, p->rows, p->out_dim, act ? (T*)ws.dz : nullptr,
            dbias ? ws.part : nullptr);
        if ((rc = check_launch("dz_kernel"))) return rc;
    }
    if (dbias) {
        dz_reduce_kernel<T><<<(p->out_dim + 255) / 256, 256, 0, s>>>(ws.part, split, p->out_dim, (T*)dbias);
        if ((rc = check_launch("dz_reduce_kernel"))) return rc;
    }
    const void* dz = act ? ws.dz : dy;
    const long long ldz = act ? p->out_dim : t.y;
    Epilogue e{};
    if (dx && p->rows) {
        e.y = dx;
        e.ldy = p->in_dim;
        rc = gemm<T>(dz, w, GemmShape{p->rows, p->in_dim, p->out_dim, ldz, 1, 1, t.w}, e, s);
        if (rc) return rc;
    }
    if (dw) {
        e.y = dw;
        e.ldy = p->in_dim;
        rc = gemm<T>(dz, x, GemmShape{p->out_dim, p->in_dim, p->rows, 1, ldz, 1, t.x}, e, s);
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
        *bytes = 0;
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
        (void)workspace;
        (void)workspace_bytes;
        const GemmShape g{params->rows, params->out_dim, params->in_dim, t.x, 1, t.w, 1};
        const Epilogue e{bias, residual, pre, y, t.r, t.p, t.y, params->activation};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return params->dtype == FG_DTYPE_F32   ? gemm<float>(x, w, g, e, s)
               : params->dtype == FG_DTYPE_F16 ? gemm<__half>(x, w, g, e, s)
                                               : gemm<__nv_bfloat16>(x, w, g, e, s);
    });
}

int fg_linear_backward_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        Strides t;
        const int rc = linear_check(params, t);
        if (rc) return rc;
        BackwardWs w;
        *bytes = backward_carve(params, nullptr, 0, w);
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
        rc = adapter_ws(workspace, workspace_bytes, backward_carve(params, nullptr, 0, ws));
        if (rc) return rc;
        backward_carve(params, workspace, workspace_bytes, ws);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return params->dtype == FG_DTYPE_F32 ? linear_backward<float>(params, t, dy, x, w, pre, dx, dw, dbias, ws, s)
               : params->dtype == FG_DTYPE_F16
                   ? linear_backward<__half>(params, t, dy, x, w, pre, dx, dw, dbias, ws, s)
                   : linear_backward<__nv_bfloat16>(params, t, dy, x, w, pre, dx, dw, dbias, ws, s);
    });
}

}  // extern "C"
