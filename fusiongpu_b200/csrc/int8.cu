// int8.cu -- rows as codes of 8 bits with a scale each, and the linear layer of such rows.
//
//   s = max |x| / 127,  q = 127 x / max |x| rounded to nearest, ties to even
//   y = act(xs ws (xq wq^T) + bias) + residual
//
// The sums are 32-bit integers (127^2 or 128^2 times at most 131,071), exact in any
// order.  In 32 bits each of three steps rounds once: the sum as a float (past 2^24), its
// product with ws, and that one's with xs, to which the bias is added in the same
// operation; then the result to its type.  The sum times ws has to stay within float32's
// range, which a ws below 2^96 does.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace fg {

// ---- codes of rows -----------------------------------------------------------------
//
// A group of threads holds its row in registers, so that memory is read once: eight up
// to 128 columns, a warp up to 2,048 (16 bits) or 1,024 (32), a block of 256 up to 8,192 or
// 4,096; longer rows are read again from L2.
constexpr int QR_NT = 256, QR_TURNS = 8;
constexpr int QUANTIZE_DIM = 1 << 30;

// Two values' magnitudes against the largest so far, as the type's bits: of two 16-bit
// values in one instruction, where a NaN wins.
__device__ __forceinline__ uint32_t larger(uint32_t top, float a, float b) {
    return max(top, max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}
__device__ __forceinline__ uint32_t larger(uint32_t top, __half a, __half b) {
    const __half2 t = __hmax2_nan(*reinterpret_cast<const __half2*>(&top), __habs2(__halves2half2(a, b)));
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t larger(uint32_t top, __nv_bfloat16 a, __nv_bfloat16 b) {
    const __nv_bfloat162 t = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&top), __habs2(__halves2bfloat162(a, b)));
    return *reinterpret_cast<const uint32_t*>(&t);
}
// ... and as the bits of a float, whose order as integers puts a NaN above all numbers.
template <class T>
__device__ __forceinline__ uint32_t float_bits(uint32_t top) {
    if (sizeof(T) == 4) return top;
    const unsigned short lo = (unsigned short)top, hi = (unsigned short)(top >> 16);
    const float a = to_f32(*reinterpret_cast<const T*>(&lo)), b = to_f32(*reinterpret_cast<const T*>(&hi));
    return max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu);
}

struct QuantRow {
    float top, inv, up;  // inv: 127 / top, nearly; up: a power of two that brings top to where 127 top and 127 / top are ordinary numbers
    bool finite;         // no infinity or NaN in the row
    bool fast;           // inv is an ordinary number
};

// 127 x / top rounded to nearest, ties to even, for a value near a half between codes: the
// remainder 127 x - r top of the nearest candidate, as a sum of two floats without an
// error, against top / 2.
__device__ __forceinline__ float exact_code(float x, const QuantRow& q) {
    x *= q.up;
    const float top = q.top * q.up, half = 0.5f * top;
    const float r = rintf(x * (127.0f / top)), p = 127.0f * x, t = r * top;
    const float rest = fmaf(127.0f, x, -p) - fmaf(r, top, -t), e = p - t;  // 127 x - r top = e + rest
    const float over = (fabsf(e) - half) + (e < 0.0f ? -rest : rest);
    const bool odd = (int)r & 1;
    return over > 0.0f || (over == 0.0f && odd) ? r + (e < 0.0f ? -1.0f : 1.0f) : r;
}

// Codes 127 x / top of N values, rounded to nearest, ties to even.  x times 127 / top plus
// 1.5 2^23 rounds the product once to an integer, which the sum's low byte holds; the
// quotient is off by 1.5 2^-23 of it.
//   bfloat16: exact ties are frequent (the largest value has 8 bits), and nothing else comes
//   near a half: with t = 127 m 2^-e / n, m and n of 8 bits, a value that is none is 2^-e / 255
//   from it at least, t at most 254 2^-e.  So what lies within 2^-22 t of a half is a tie, and
//   goes to twice the rounded half of the quotient, which is even.
//   float16 and float32: the quotient is taken 2^-21 too small and too large; where both give
//   the same integers, those are right.  Else, float16: the remainder 127 x - r top is exact
//   in 32 bits, and a code whose remainder reaches top / 2 is put right.  float32: again
//   without an error.
template <class T, int N>
__device__ __forceinline__ void codes_of(uint32_t (&out)[N / 4], const T (&v)[N], const QuantRow& q) {
    constexpr float magic = 12582912.0f;
    uint32_t c[N], differ = 0;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const uint64_t inv = pair2(q.inv, q.inv), half = pair2(0.5f * q.inv, 0.5f * q.inv), m = pair2(magic, magic), minus = pair2(-magic, -magic);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t x = pair2(to_f32(v[i]), to_f32(v[i + 1])), r = fma2(x, inv, m), back = add2(r, minus);
            float a, b, d, e, s, t;
            unpair2(back, a, b);
            unpair2(fma2(x, inv, pair2(-a, -b)), d, e);
            unpair2(fma2(x, half, m), s, t);
            const bool tie0 = fmaf(fabsf(a), 2.3841858e-7f, fabsf(d)) >= 0.5f, tie1 = fmaf(fabsf(b), 2.3841858e-7f, fabsf(e)) >= 0.5f;
            unpair2(r, a, b);
            c[i] = tie0 ? __float_as_uint(s) * 2 : __float_as_uint(a);
            c[i + 1] = tie1 ? __float_as_uint(t) * 2 : __float_as_uint(b);
        }
    } else {
        const float low = q.inv - q.inv * 4.7683716e-7f, high = q.inv + q.inv * 4.7683716e-7f;
        const uint64_t l = pair2(low, low), h = pair2(high, high), m = pair2(magic, magic);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t x = pair2(to_f32(v[i]), to_f32(v[i + 1]));
            float a, b, d, e;
            unpair2(fma2(x, l, m), a, b);
            unpair2(fma2(x, h, m), d, e);
            c[i] = __float_as_uint(a);
            c[i + 1] = __float_as_uint(b);
            differ |= (c[i] ^ __float_as_uint(d)) | (c[i + 1] ^ __float_as_uint(e));
        }
    }
    if (differ || !q.fast) {
        if (sizeof(T) == 4 || !q.fast) {
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = q.finite && q.top > 0.0f ? __float_as_uint(exact_code(to_f32(v[i]), q) + magic) : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float e = fmaf(__uint_as_float(c[i]) - magic, -q.top, 127.0f * to_f32(v[i])), over = fabsf(e) - 0.5f * q.top;
                if (over > 0.0f || (over == 0.0f && (c[i] & 1))) c[i] += e < 0.0f ? -1 : 1;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; i += 4)
        out[i / 4] = __byte_perm(__byte_perm(c[i], c[i + 1], 0x0040), __byte_perm(c[i + 2], c[i + 3], 0x0040), 0x5410);
}

struct QuantArgs {
    const void* x;
    signed char* q;
    float* scale;
    long long rows, ldx, ldq;
    int dim, turns, unit, wide;  // turns: rows of a group; unit: bytes that x's rows start on, up to 16; wide: q's start on 8
};

// VEC neighbouring columns, `unit` bytes at a time: what the rows' starts allow.
template <class T, int VEC>
__device__ __forceinline__ void qr_load(T (&v)[VEC], const T* p, int left, int unit, bool whole = false) {
    if (left <= 0) {  // behind the row's end
        *reinterpret_cast<uint4*>(v) = make_uint4(0, 0, 0, 0);
    } else if (whole || (unit == 16 && left >= VEC)) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    } else if (unit >= 8 && left >= VEC) {
        reinterpret_cast<uint2*>(v)[0] = reinterpret_cast<const uint2*>(p)[0];
        reinterpret_cast<uint2*>(v)[1] = reinterpret_cast<const uint2*>(p)[1];
    } else if (unit >= 4 && left >= VEC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(v)[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = i < left ? p[i] : from_f32<T>(0.0f);
    }
}

template <class T, int VEC>
__device__ __forceinline__ void qr_store(signed char* p, const T (&v)[VEC], const QuantRow& q, int left, int wide, bool whole = false) {
    if (left <= 0) return;
    uint32_t codes[VEC / 4];
    codes_of<T, VEC>(codes, v, q);
    if (whole || (wide && left >= VEC)) {
        if constexpr (VEC == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(codes[0], codes[1]);
        else
            *reinterpret_cast<uint32_t*>(p) = codes[0];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < left) p[i] = (signed char)(codes[i / 4] >> (i % 4 * 8));
    }
}

// The row's largest magnitude, in all of its L threads.
template <class T, int L>
__device__ __forceinline__ QuantRow row_of(uint32_t top, uint32_t* s) {
    top = float_bits<T>(top);
    if (L < 32) {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    } else {
        top = __reduce_max_sync(0xffffffffu, top);
    }
    if (L > 32) {
        __syncthreads();  // the last row's readers are done with s
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < L / 32; ++w) top = max(top, s[w]);
    }
    QuantRow q;
    q.finite = top < 0x7f800000u;
    q.top = __uint_as_float(top);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.inv) : "f"(q.top));
    q.inv *= 127.0f;
    q.up = q.top < 1e-18f ? 18446744073709551616.0f : q.top > 1e30f ? 1.0f / 65536.0f : 1.0f;  // 2^64, 2^-16
    q.fast = q.finite && q.up == 1.0f;
    return q;
}
// top / 127, correctly rounded: one correction of the product with the rounded 1 / 127, which
// gives the division's bits for all significands; tiny and huge rows divide.
__device__ __forceinline__ float scale_of(const QuantRow& q) {
    if (!q.fast) return q.finite ? q.top / 127.0f : NAN;
    constexpr float y = 1.0f / 127.0f;
    const float r = q.top * y;
    return fmaf(fmaf(r, -127.0f, q.top), y, r);
}

__host__ __device__ constexpr int qr_blocks(int per) { return per <= 4 ? 4 : 2; }  // an SM

// L threads a row (8, 32 or the block), PER pieces of 16 bytes each.  A block takes as many
// rows at a time as it has groups, QR_TURNS times or, of few rows, as one round of blocks
// needs; a group asks for its next row before it works on this one.  Bound by memory, and
// nearly by issue slots (66 %): 1M x 768 float16 342 us, 6.7 TB/s (a row a group: 501; 32 rows
// a group 351, one round of blocks 390: they drift apart, and memory serves neighbours
// best); 2M x 128 bfloat16 147 (202 with a remainder for its ties).  Narrow rows are bound by
// issue slots: 3M x 40 float16 138.
//
// WHOLE: all pieces are loaded and stored whole.
template <class T, int L, int PER, bool WHOLE>
__global__ void __launch_bounds__(QR_NT, qr_blocks(PER)) quantize_kernel(const QuantArgs g) {
    constexpr int VEC = 16 / sizeof(T), GROUPS = QR_NT / L;
    __shared__ uint32_t s[QR_NT / 32];
    const int lane = threadIdx.x % L;
    const long long x_step = GROUPS * g.ldx, q_step = GROUPS * g.ldq;
    long long first = (long long)blockIdx.x * g.turns * GROUPS, row = first + threadIdx.x / L;  // `first`: the block's, so that its threads stay together
    const long long end = min(first + (long long)g.turns * GROUPS, g.rows);
    const T* x = static_cast<const T*>(g.x) + row * g.ldx + lane * VEC;  // of the next row
    signed char* out = g.q + row * g.ldq + lane * VEC;
    alignas(16) T next[PER][VEC];
    auto fetch = [&](bool here) {
#pragma unroll
        for (int k = 0; k < PER; ++k)
            qr_load<T, VEC>(next[k], x + k * L * VEC, here ? g.dim - (k * L + lane) * VEC : 0, WHOLE ? 16 : g.unit, WHOLE);
        x += x_step;
    };
    fetch(row < g.rows);
    for (; first < end; first += GROUPS, row += GROUPS, out += q_step) {
        alignas(16) T v[PER][VEC];
#pragma unroll
        for (int k = 0; k < PER; ++k) *reinterpret_cast<uint4*>(v[k]) = *reinterpret_cast<const uint4*>(next[k]);
        if (first + GROUPS < end) fetch(row + GROUPS < g.rows);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) top = larger(top, v[k][i], v[k][i + 1]);
        const QuantRow q = row_of<T, L>(top, s);
        if (row >= g.rows) continue;
        if (lane == 0) g.scale[row] = scale_of(q);
#pragma unroll
        for (int k = 0; k < PER; ++k) qr_store<T, VEC>(out + k * L * VEC, v[k], q, g.dim - (k * L + lane) * VEC, WHOLE ? 1 : g.wide, WHOLE);
    }
}

// Rows of any length, read twice.
template <class T>
__global__ void __launch_bounds__(QR_NT) quantize_long_kernel(const QuantArgs g) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ uint32_t s[QR_NT / 32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(g.x) + row * g.ldx;
    alignas(16) T v[VEC];
    uint32_t top = 0;
#pragma unroll 4
    for (int c = threadIdx.x * VEC; c < g.dim; c += QR_NT * VEC) {
        qr_load<T, VEC>(v, x + c, g.dim - c, g.unit);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) top = larger(top, v[i], v[i + 1]);
    }
    const QuantRow q = row_of<T, QR_NT>(top, s);
    if (threadIdx.x == 0) g.scale[row] = scale_of(q);
    for (int c = threadIdx.x * VEC; c < g.dim; c += QR_NT * VEC) {
        qr_load<T, VEC>(v, x + c, g.dim - c, g.unit);
        qr_store<T, VEC>(g.q + row * g.ldq + c, v, q, g.dim - c, g.wide);
    }
}

template <class T>
static int launch_quantize(QuantArgs g, cudaStream_t s) {
    constexpr int VEC = 16 / (int)sizeof(T);
    g.unit = 16;
    while (g.unit > (int)sizeof(T) && !(aligned(g.x, g.unit) && g.ldx * (int)sizeof(T) % g.unit == 0)) g.unit /= 2;
    g.wide = aligned(g.q, 8) && g.ldq % 8 == 0;
    const long long pieces = (g.dim + VEC - 1) / VEC;
    const bool warps = pieces <= 32 * 8;
    if (!warps && pieces > 4 * QR_NT) {
        FG_REQUIRE(g.rows <= 0x7fffffffll, "too many rows");
        quantize_long_kernel<T><<<(unsigned)g.rows, QR_NT, 0, s>>>(g);
        return check_launch("quantize_long_kernel");
    }
    const bool eights = pieces <= 8 * (sizeof(T) == 2 ? 2 : 4);
    const int lanes = eights ? 8 : warps ? 32 : QR_NT, per = (int)((pieces + lanes - 1) / lanes);
    auto of = [&](auto l, auto whole) {
        constexpr int L = decltype(l)::value;
        constexpr bool W = decltype(whole)::value;
        return per <= 1 ? &quantize_kernel<T, L, 1, W> : per <= 2 ? &quantize_kernel<T, L, 2, W> : per <= 3 ? &quantize_kernel<T, L, 3, W> : &quantize_kernel<T, L, 4, W>;
    };
    auto way = [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        if (per > 4) return per <= 6 ? &quantize_kernel<T, 32, 6, W> : &quantize_kernel<T, 32, 8, W>;
        return eights ? of(std::integral_constant<int, 8>(), whole) : warps ? of(std::integral_constant<int, 32>(), whole) : of(std::integral_constant<int, QR_NT>(), whole);
    };
    auto kernel = g.unit == 16 && g.wide && g.dim % VEC == 0 ? way(std::true_type()) : way(std::false_type());
    const long long blocks = (g.rows + QR_NT / lanes - 1) / (QR_NT / lanes);
    const long long most = (long long)qr_blocks(per) * std::max(1, device_attr(cudaDevAttrMultiProcessorCount));
    g.turns = (int)std::min<long long>(QR_TURNS, (blocks + most - 1) / most);
    kernel<<<(unsigned)((blocks + g.turns - 1) / g.turns), QR_NT, 0, s>>>(g);
    return check_launch("quantize_kernel");
}

// ---- a few rows: a warp a column, four codes at a time -----------------------------
//
// Bound by the latency of the loads: 768 -> 1536 2.6 us for one row, 3.1 for eight.
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
    if (lane < R && lane < g.m) {
        Epilogue rest = e;  // the bias is in the product with the scales
        rest.bias = nullptr;
        epilogue_store<T>(rest, lane, n, fmaf((float)mine * ws[n], xs[lane], e.bias ? to_f32(static_cast<const T*>(e.bias)[n]) : 0.0f));
    }
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
    const long long i = blockIdx.x * 256ll + threadIdx.x, per = stride / 16;
    const long long row = i <= 0x7fffffff ? (long long)((unsigned)i / (unsigned)per) : i / per;  // 64 bits take a long division
    if (row >= rows) return;
    const int c0 = (int)(i - row * per) * 16;
    const signed char* from = in + row * ld + c0;
    const uintptr_t start = reinterpret_cast<uintptr_t>(from);
    alignas(16) signed char v[16];
    if (c0 + 16 <= cols && (start & 15) == 0) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(from);
    } else if (c0 + 16 <= cols && (start & 3) == 0) {
#pragma unroll
        for (int c = 0; c < 4; ++c) reinterpret_cast<uint32_t*>(v)[c] = reinterpret_cast<const uint32_t*>(from)[c];
    } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = c0 + c < cols ? from[c] : (signed char)0;
    }
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
        const QuantArgs g{x, reinterpret_cast<signed char*>(q), scale, rows, ldx, ldq, dim, 0, 0, 0};
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
