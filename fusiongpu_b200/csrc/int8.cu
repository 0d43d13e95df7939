// int8.cu -- rows as codes of 8 bits with a scale each, and the linear layer of such rows.
//
//   s = max |x| / 127,  q = 127 x / max |x| rounded to nearest, ties to even
//   y = act(xs ws (xq wq^T) + bias) + residual
//
// The sums are 32-bit integers (127^2 or 128^2 times at most 131,071), exact in any
// order; the product with the scales rounds once to 32 bits, the result once to its type.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace fg {

// ---- codes of rows -----------------------------------------------------------------
//
// A group of threads holds its row in registers, so that memory is read once: a warp up
// to 1,024 columns, a block of 256 up to 8,192 (16 bits) or 4,096 (32); longer rows are
// read again from L2.  The largest magnitude is found on the bits, as integers, where a
// NaN is above all numbers.
constexpr int QR_NT = 256;
constexpr int QUANTIZE_DIM = 1 << 30;

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 127 x / top, rounded to nearest, ties to even.  x inv is off by at most 2^-23 of it
// (1.6e-5 at 127); next to a half, or where inv is not finite, the quotient in 64 bits,
// whose distance from a half, if not 0, is at least 2^-25 of it.
__device__ __forceinline__ int code_of(float x, float top, float inv) {
    const float t = x * inv, r = rintf(t);
    if (fabsf(fabsf(t - r) - 0.5f) > 2e-5f && inv <= FLT_MAX) return (int)r;
    return top > 0.0f ? (int)rint(127.0 * (double)x / (double)top) : 0;
}

struct QuantArgs {
    const void* x;
    signed char* q;
    float* scale;
    long long rows, ldx, ldq;
    int dim, wide;  // wide: rows of x and q start on 16 bytes
};

template <class T, int VEC>
__device__ __forceinline__ void qr_store(signed char* p, const T (&v)[VEC], float top, float inv, bool finite, int left, int wide) {
    alignas(8) signed char c[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = finite ? (signed char)code_of(to_f32(v[i]), top, inv) : (signed char)0;
    if (wide && left >= VEC) {
        if constexpr (VEC == 8)
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(c);
        else
            *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(c);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < left) p[i] = c[i];
    }
}

template <class T, int VEC>
__device__ __forceinline__ void qr_load(T (&v)[VEC], const T* p, int left, int wide) {
    if (wide && left >= VEC) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = i < left ? p[i] : from_f32<T>(0.0f);
    }
}

// L threads a row (32, or the block), PER pieces of 16 bytes each; PER 0: rows of any
// length, read twice.
template <class T, int L, int PER>
__global__ void __launch_bounds__(QR_NT) quantize_kernel(const QuantArgs g) {
    constexpr int VEC = 16 / sizeof(T), HELD = PER ? PER : 1;
    __shared__ uint32_t s[QR_NT / 32];
    const int lane = threadIdx.x % L;
    const long long row = blockIdx.x * (long long)(QR_NT / L) + threadIdx.x / L;
    if (row >= g.rows) return;  // L == 32: whole warps; L == QR_NT: none
    const T* x = static_cast<const T*>(g.x) + row * g.ldx;
    signed char* q = g.q + row * g.ldq;
    alignas(16) T v[HELD][VEC];
    uint32_t top = 0;
    auto more = [&](const T (&v)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, magnitude(to_f32(v[i])));
    };
    if (PER) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int c = (k * L + lane) * VEC;
            qr_load<T, VEC>(v[k], x + c, g.dim - c, g.wide);
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) more(v[k]);
    } else {
        for (int c = lane * VEC; c < g.dim; c += L * VEC) {
            qr_load<T, VEC>(v[0], x + c, g.dim - c, g.wide);
            more(v[0]);
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (L > 32) {
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < QR_NT / 32; ++w) top = max(top, s[w]);
    }
    const bool finite = top < 0x7f800000u;
    const float most = __uint_as_float(top), inv = 127.0f / most;
    if (lane == 0) g.scale[row] = finite ? most / 127.0f : NAN;
    if (PER) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int c = (k * L + lane) * VEC;
            qr_store<T, VEC>(q + c, v[k], most, inv, finite, g.dim - c, g.wide);
        }
    } else {
        for (int c = lane * VEC; c < g.dim; c += L * VEC) {
            qr_load<T, VEC>(v[0], x + c, g.dim - c, g.wide);
            qr_store<T, VEC>(q + c, v[0], most, inv, finite, g.dim - c, g.wide);
        }
    }
}

template <class T>
static int launch_quantize(QuantArgs g, cudaStream_t s) {
    constexpr int VEC = 16 / (int)sizeof(T);
    g.wide = aligned(g.x, 16) && g.ldx * (int)sizeof(T) % 16 == 0 && aligned(g.q, 16) && g.ldq % 16 == 0;
    const long long pieces = (g.dim + VEC - 1) / VEC;
    const bool warps = pieces <= 32 * (sizeof(T) == 2 ? 4 : 8);
    const long long blocks = warps ? (g.rows + QR_NT / 32 - 1) / (QR_NT / 32) : g.rows;
    FG_REQUIRE(blocks <= 0x7fffffffll, "too many rows");
    const int per = (int)std::min<long long>(8, (pieces + (warps ? 32 : QR_NT) - 1) / (warps ? 32 : QR_NT));
    auto kernel = &quantize_kernel<T, QR_NT, 0>;
    if (warps)
        kernel = per <= 1 ? &quantize_kernel<T, 32, 1> : per <= 2 ? &quantize_kernel<T, 32, 2> : per <= 3 ? &quantize_kernel<T, 32, 3>
                 : per <= 4 ? &quantize_kernel<T, 32, 4> : per <= 6 ? &quantize_kernel<T, 32, 6> : &quantize_kernel<T, 32, 8>;
    else if (pieces <= 4 * QR_NT)
        kernel = per <= 1 ? &quantize_kernel<T, QR_NT, 1> : per <= 2 ? &quantize_kernel<T, QR_NT, 2> : &quantize_kernel<T, QR_NT, 4>;
    kernel<<<(unsigned)blocks, QR_NT, 0, s>>>(g);
    return check_launch("quantize_kernel");
}

// ---- a few rows: a warp a column, four codes at a time -----------------------------
template <class T, int R>
__global__ void __launch_bounds__(128) gemv_int8_kernel(const signed char* __restrict__ x, const signed char* __restrict__ w,
                                                        const GemmShape g, int wide, const float* xs, const float* ws, const Epilogue e) {
    const int lane = threadIdx.x & 31;
    const long long n = blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (n >= g.n) return;
    const signed char* wr = w + n * g.bn;
    const signed char* xr[R];  // rows past the last are the last again: no branch keeps loads apart
    int acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        xr[r] = x + min((long long)r, g.m - 1) * g.am;
        acc[r] = 0;
    }
    long long k0 = 0;
    if (wide) {
#pragma unroll 2
        for (long long k = lane * 16; k + 16 <= g.k; k += 512) {
            const uint4 b = *reinterpret_cast<const uint4*>(wr + k);
            uint4 a[R];
#pragma unroll
            for (int r = 0; r < R; ++r) a[r] = *reinterpret_cast<const uint4*>(xr[r] + k);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                acc[r] = __dp4a((int)a[r].x, (int)b.x, acc[r]);
                acc[r] = __dp4a((int)a[r].y, (int)b.y, acc[r]);
                acc[r] = __dp4a((int)a[r].z, (int)b.z, acc[r]);
                acc[r] = __dp4a((int)a[r].w, (int)b.w, acc[r]);
            }
        }
        k0 = g.k / 16 * 16;
    }
    for (long long k = k0 + lane; k < g.k; k += 32) {
        const int b = wr[k];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] += b * xr[r][k];
    }
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int v = __reduce_add_sync(0xffffffffu, acc[r]);
        if (lane == r) mine = v;
    }
    if (lane < R && lane < g.m) epilogue_store<T>(e, lane, n, (float)mine * (xs[lane] * ws[n]));
}

template <class T>
static int gemv_int8(const void* x, const void* w, const GemmShape& g, const float* xs, const float* ws, const Epilogue& e, cudaStream_t s) {
    const int wide = aligned(x, 16) && g.am % 16 == 0 && aligned(w, 16) && g.bn % 16 == 0;
    auto kernel = g.m == 1 ? &gemv_int8_kernel<T, 1> : g.m == 2 ? &gemv_int8_kernel<T, 2> : g.m <= 4 ? &gemv_int8_kernel<T, 4>
                                                                                          : &gemv_int8_kernel<T, GEMV_ROWS>;
    kernel<<<(unsigned)((g.n + 3) / 4), 128, 0, s>>>(static_cast<const signed char*>(x), static_cast<const signed char*>(w), g, wide,
                                                     xs, ws, e);
    return check_launch("gemv_int8_kernel");
}

// ---- rows off 16 bytes, copied to rows on them --------------------------------------
__global__ void __launch_bounds__(256) pack_int8_kernel(const signed char* in, signed char* out, long long rows, long long ld, int cols,
                                                        long long stride) {
    const long long i = blockIdx.x * 256ll + threadIdx.x, per = stride / 16, row = i / per;
    if (row >= rows) return;
    const int c0 = (int)(i - row * per) * 16;
    alignas(16) signed char v[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) v[c] = c0 + c < cols ? in[row * ld + c0 + c] : (signed char)0;
    *reinterpret_cast<uint4*>(out + row * stride + c0) = *reinterpret_cast<const uint4*>(v);
}

constexpr int INT8_IN = 131071;  // 128^2 times as many stay below 2^31

static int int8_check(const fg_linear_params* p, Strides& t) {
    const int rc = linear_check(p, t);
    if (rc) return rc;
    if (p->in_dim > INT8_IN) return fail(FG_ERR_UNSUPPORTED, "in_dim above %d", INT8_IN);
    FG_REQUIRE(p->pre_stride == 0, "an 8-bit layer keeps no pre-activation");
    return FG_OK;
}

struct Int8Ws {
    signed char *x, *w;
};
static long long int8_stride(int cols) { return (cols + 15) / 16 * 16; }

static size_t int8_carve(const fg_linear_params* p, const Strides& t, void* ws, size_t bytes, Int8Ws& f) {
    Carve c(ws, bytes);
    f = Int8Ws{};
    if (p->rows <= GEMV_ROWS) return 0;
    if (t.x % 16 || (p->unaligned & FG_LINEAR_X)) f.x = c.take<signed char>((size_t)p->rows * int8_stride(p->in_dim));
    if (t.w % 16 || (p->unaligned & FG_LINEAR_W)) f.w = c.take<signed char>((size_t)p->out_dim * int8_stride(p->in_dim));
    return c.used;
}

static int pack_int8(const void*& p, long long& ld, signed char* room, long long rows, int cols, cudaStream_t s) {
    if (!room) return FG_OK;
    const long long stride = int8_stride(cols), n = rows * (stride / 16);
    FG_REQUIRE(n <= 0x7fffffffll * 256, "operand too large");
    pack_int8_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(static_cast<const signed char*>(p), room, rows, ld, cols, stride);
    p = room;
    ld = stride;
    return check_launch("pack_int8_kernel");
}

}  // namespace fg

using namespace fg;

extern "C" {

int fg_quantize_rows(const void* x, int32_t dtype, int64_t rows, int32_t dim, int64_t x_stride, int8_t* q, int64_t q_stride,
                     float* scale, void* stream) {
    return c_entry([&]() -> int {
        FG_REQUIRE(float_dtype(dtype), "unknown dtype %d", dtype);
        FG_REQUIRE(rows >= 0 && dim >= 1, "bad shape");
        const long long ldx = x_stride ? x_stride : dim, ldq = q_stride ? q_stride : dim;
        FG_REQUIRE(ldx >= dim && ldq >= dim, "row stride below the row length");
        if (dim > QUANTIZE_DIM) return fail(FG_ERR_UNSUPPORTED, "dim above %d", QUANTIZE_DIM);
        if (rows == 0) return FG_OK;
        FG_REQUIRE(x && q && scale, "null buffer");
        const QuantArgs g{x, reinterpret_cast<signed char*>(q), scale, rows, ldx, ldq, dim, 0};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return dtype == FG_DTYPE_F32   ? launch_quantize<float>(g, s)
               : dtype == FG_DTYPE_F16 ? launch_quantize<__half>(g, s)
                                       : launch_quantize<__nv_bfloat16>(g, s);
    });
}

int fg_linear_int8_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        Strides t;
        const int rc = int8_check(params, t);
        if (rc) return rc;
        Int8Ws f;
        *bytes = int8_carve(params, t, nullptr, 0, f);
        return FG_OK;
    });
}

int fg_linear_int8(const fg_linear_params* params, const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale,
                   const void* bias, const void* residual, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&]() -> int {
        Strides t;
        int rc = int8_check(params, t);
        if (rc) return rc;
        if (params->rows == 0) return FG_OK;
        FG_REQUIRE(x && x_scale && w && w_scale && y, "null buffer");
        FG_REQUIRE(aligned(x, 16) || (params->unaligned & FG_LINEAR_X), "x is off 16 bytes and not named in unaligned");
        FG_REQUIRE(aligned(w, 16) || (params->unaligned & FG_LINEAR_W), "w is off 16 bytes and not named in unaligned");
        Int8Ws f;
        if ((rc = adapter_ws(workspace, workspace_bytes, int8_carve(params, t, nullptr, 0, f)))) return rc;
        int8_carve(params, t, workspace, workspace_bytes, f);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const Epilogue e{bias, residual, nullptr, y, t.r, 0, t.y, params->activation};
        GemmShape g{params->rows, params->out_dim, params->in_dim, t.x, 1, t.w, 1};
        if (params->rows <= GEMV_ROWS)
            return params->dtype == FG_DTYPE_F32   ? gemv_int8<float>(x, w, g, x_scale, w_scale, e, s)
                   : params->dtype == FG_DTYPE_F16 ? gemv_int8<__half>(x, w, g, x_scale, w_scale, e, s)
                                                   : gemv_int8<__nv_bfloat16>(x, w, g, x_scale, w_scale, e, s);
        const void *a = x, *b = w;
        if ((rc = pack_int8(a, g.am, f.x, params->rows, params->in_dim, s))) return rc;
        if ((rc = pack_int8(b, g.bn, f.w, params->out_dim, params->in_dim, s))) return rc;
        return tc_int8(params->dtype, a, x_scale, b, w_scale, g, e, s);
    });
}

}  // extern "C"
