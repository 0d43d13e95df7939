// norm.cu -- layer norm over rows and its gradients.
//
//   y = (x - m) r w + b,   m = avg(x),  r = 1 / sqrt(avg((x - m)^2) + eps)
//   h = (x - m) r,  a = dy w:   dx = r (a - avg(a) - h avg(a h)),
//   dw = sum over rows of dy h,  db = sum over rows of dy
#include <algorithm>

#include "adapter_common.cuh"

namespace fg {

constexpr int LN_MAX_DIM = 16384;
constexpr int LN_NT = 128;
constexpr int LN_COLS = 32;    // columns per block of the column sums
constexpr int LN_SPLIT = 64;   // row ranges of the column sums

struct NormArgs {
    const void *x, *dy, *w, *b;
    const float *mean, *rstd;
    void *y, *dx;
    float *out_mean, *out_rstd, *part;
    long long rows, ldx, ldy, lddx;
    int dim, w_f32;
    float eps;
};

template <class T>
__device__ __forceinline__ float param(const void* p, int f32, int j) {
    return f32 ? static_cast<const float*>(p)[j] : to_f32(static_cast<const T*>(p)[j]);
}

template <class T>
__global__ void __launch_bounds__(LN_NT) ln_forward_kernel(const NormArgs g) {
    __shared__ float s[LN_NT / 32];
    for (long long r = blockIdx.x; r < g.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(g.x) + r * g.ldx;
        T* y = static_cast<T*>(g.y) + r * g.ldy;
        float t = 0.0f;
        for (int j = threadIdx.x; j < g.dim; j += LN_NT) t += to_f32(x[j]);
        const float mean = block_sum<LN_NT>(t, s) / (float)g.dim;
        t = 0.0f;
        for (int j = threadIdx.x; j < g.dim; j += LN_NT) {
            const float c = to_f32(x[j]) - mean;
            t = fmaf(c, c, t);
        }
        const float rstd = rsqrtf(block_sum<LN_NT>(t, s) / (float)g.dim + g.eps);
        for (int j = threadIdx.x; j < g.dim; j += LN_NT) {
            const float h = __fmul_rn(to_f32(x[j]) - mean, rstd);  // an absent weight or bias is 1 or 0, bit for bit
            y[j] = from_f32<T>(fmaf(h, g.w ? param<T>(g.w, g.w_f32, j) : 1.0f, g.b ? param<T>(g.b, g.w_f32, j) : 0.0f));
        }
        if (g.out_mean && threadIdx.x == 0) {
            g.out_mean[r] = mean;
            g.out_rstd[r] = rstd;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(LN_NT) ln_dx_kernel(const NormArgs g) {
    __shared__ float s[LN_NT / 32];
    for (long long r = blockIdx.x; r < g.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(g.x) + r * g.ldx;
        const T* dy = static_cast<const T*>(g.dy) + r * g.ldy;
        T* dx = static_cast<T*>(g.dx) + r * g.lddx;
        const float mean = g.mean[r], rstd = g.rstd[r];
        float sa = 0.0f, sah = 0.0f;
        for (int j = threadIdx.x; j < g.dim; j += LN_NT) {
            const float h = (to_f32(x[j]) - mean) * rstd;
            const float a = to_f32(dy[j]) * (g.w ? param<T>(g.w, g.w_f32, j) : 1.0f);
            sa += a;
            sah = fmaf(a, h, sah);
        }
        sa = block_sum<LN_NT>(sa, s) / (float)g.dim;
        sah = block_sum<LN_NT>(sah, s) / (float)g.dim;
        for (int j = threadIdx.x; j < g.dim; j += LN_NT) {
            const float h = (to_f32(x[j]) - mean) * rstd;
            const float a = to_f32(dy[j]) * (g.w ? param<T>(g.w, g.w_f32, j) : 1.0f);
            dx[j] = from_f32<T>(rstd * (a - sa - h * sah));
        }
    }
}

// Block (c, s): columns [32c, 32c + 32) over the s-th range of rows.
template <class T>
__global__ void __launch_bounds__(256) ln_columns_kernel(const NormArgs g) {
    __shared__ float sw[8][LN_COLS], sb[8][LN_COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * LN_COLS + lane;
    const long long per = (g.rows + gridDim.y - 1) / gridDim.y;
    const long long r0 = blockIdx.y * per, r1 = r0 + per < g.rows ? r0 + per : g.rows;
    float w = 0.0f, b = 0.0f;
    if (j < g.dim)
        for (long long r = r0 + warp; r < r1; r += 8) {
            const float d = to_f32(static_cast<const T*>(g.dy)[r * g.ldy + j]);
            w = fmaf(d, (to_f32(static_cast<const T*>(g.x)[r * g.ldx + j]) - g.mean[r]) * g.rstd[r], w);
            b += d;
        }
    sw[warp][lane] = w;
    sb[warp][lane] = b;
    __syncthreads();
    if (warp == 0 && j < g.dim) {
        w = b = 0.0f;
        for (int i = 0; i < 8; ++i) {
            w += sw[i][lane];
            b += sb[i][lane];
        }
        g.part[(size_t)blockIdx.y * 2 * g.dim + j] = w;
        g.part[((size_t)blockIdx.y * 2 + 1) * g.dim + j] = b;
    }
}

// Adds the partial rows in their order.
template <class P>
__global__ void ln_reduce_kernel(const float* part, int parts, int dim, P* dw, P* db) {
    const int j = blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= 2 * dim) return;
    float v = 0.0f;
    for (int p = 0; p < parts; ++p) v += part[(size_t)p * 2 * dim + j];
    P* out = j < dim ? dw : db;
    if (out) out[j < dim ? j : j - dim] = from_f32<P>(v);
}

static int norm_check(int dtype, int param_dtype, long long rows, int dim) {
    FG_REQUIRE(float_dtype(dtype), "unknown dtype %d", dtype);
    FG_REQUIRE(param_dtype == dtype || param_dtype == FG_DTYPE_F32, "param_dtype %d is neither dtype nor F32",
               param_dtype);
    FG_REQUIRE(rows >= 0, "rows %lld < 0", rows);
    FG_REQUIRE(dim >= 1, "dim %d < 1", dim);
    if (dim > LN_MAX_DIM) return fail(FG_ERR_UNSUPPORTED, "dim %d > %d", dim, LN_MAX_DIM);
    return FG_OK;
}

static size_t norm_ws(int dim) { return (size_t)LN_SPLIT * 2 * dim * sizeof(float); }

template <class T>
static int norm_forward(const NormArgs& g, cudaStream_t s) {
    ln_forward_kernel<T><<<(unsigned)std::min<long long>(g.rows, 1 << 20), LN_NT, 0, s>>>(g);
    return check_launch("ln_forward_kernel");
}

template <class T>
static int norm_backward(const NormArgs& g, void* dw, void* db, cudaStream_t s) {
    if (g.dx && g.rows) {
        ln_dx_kernel<T><<<(unsigned)std::min<long long>(g.rows, 1 << 20), LN_NT, 0, s>>>(g);
        const int rc = check_launch("ln_dx_kernel");
        if (rc) return rc;
    }
    if (!dw && !db) return FG_OK;
    const int split = (int)std::min<long long>(LN_SPLIT, (g.rows + 7) / 8);
    if (split) {
        ln_columns_kernel<T><<<dim3((g.dim + LN_COLS - 1) / LN_COLS, split), 256, 0, s>>>(g);
        const int rc = check_launch("ln_columns_kernel");
        if (rc) return rc;
    }
    const int nb = (2 * g.dim + 255) / 256;
    if (g.w_f32)
        ln_reduce_kernel<float><<<nb, 256, 0, s>>>(g.part, split, g.dim, (float*)dw, (float*)db);
    else
        ln_reduce_kernel<T><<<nb, 256, 0, s>>>(g.part, split, g.dim, (T*)dw, (T*)db);
    return check_launch("ln_reduce_kernel");
}

}  // namespace fg

using namespace fg;

extern "C" {

int fg_layer_norm(const void* x, int32_t dtype, int64_t rows, int32_t dim, int64_t x_stride, const void* weight,
                  const void* bias, int32_t param_dtype, float eps, void* y, int64_t y_stride, float* mean,
                  float* rstd, void* stream) {
    return c_entry([&]() -> int {
        int rc = norm_check(dtype, param_dtype, rows, dim);
        if (rc) return rc;
        FG_REQUIRE(eps >= 0.0f, "eps %g is not >= 0", (double)eps);
        NormArgs g{};
        g.ldx = x_stride ? x_stride : dim;
        g.ldy = y_stride ? y_stride : dim;
        FG_REQUIRE(g.ldx >= dim && g.ldy >= dim, "row stride below dim");
        FG_REQUIRE((mean != nullptr) == (rstd != nullptr), "mean and rstd: both or neither");
        if (rows == 0) return FG_OK;
        FG_REQUIRE(x && y, "null buffer");
        g.x = x;
        g.w = weight;
        g.b = bias;
        g.y = y;
        g.out_mean = mean;
        g.out_rstd = rstd;
        g.rows = rows;
        g.dim = dim;
        g.w_f32 = param_dtype == FG_DTYPE_F32;
        g.eps = eps;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return dtype == FG_DTYPE_F32   ? norm_forward<float>(g, s)
               : dtype == FG_DTYPE_F16 ? norm_forward<__half>(g, s)
                                       : norm_forward<__nv_bfloat16>(g, s);
    });
}

int fg_layer_norm_backward_workspace_size(int64_t rows, int32_t dim, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        const int rc = norm_check(FG_DTYPE_F32, FG_DTYPE_F32, rows, dim);
        if (rc) return rc;
        *bytes = norm_ws(dim);
        return FG_OK;
    });
}

int fg_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int32_t dtype, int64_t rows,
                           int32_t dim, int64_t x_stride, const void* weight, int32_t param_dtype, const float* mean,
                           const float* rstd, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                           void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&]() -> int {
        int rc = norm_check(dtype, param_dtype, rows, dim);
        if (rc) return rc;
        NormArgs g{};
        g.ldx = x_stride ? x_stride : dim;
        g.ldy = dy_stride ? dy_stride : dim;
        g.lddx = dx_stride ? dx_stride : dim;
        FG_REQUIRE(g.ldx >= dim && g.ldy >= dim && g.lddx >= dim, "row stride below dim");
        if (rows) FG_REQUIRE(dy && x && mean && rstd, "null buffer");
        if (dweight || dbias) rc = adapter_ws(workspace, workspace_bytes, norm_ws(dim));
        if (rc) return rc;
        g.x = x;
        g.dy = dy;
        g.w = weight;
        g.mean = mean;
        g.rstd = rstd;
        g.dx = dx;
        g.part = static_cast<float*>(workspace);
        g.rows = rows;
        g.dim = dim;
        g.w_f32 = param_dtype == FG_DTYPE_F32;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return dtype == FG_DTYPE_F32   ? norm_backward<float>(g, dweight, dbias, s)
               : dtype == FG_DTYPE_F16 ? norm_backward<__half>(g, dweight, dbias, s)
                                       : norm_backward<__nv_bfloat16>(g, dweight, dbias, s);
    });
}

}  // extern "C"
