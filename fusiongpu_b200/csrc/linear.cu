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

// 64 x 64 tile per block of 256 threads, 4 x 4 outputs each, fp32 FMA.  a_plane: A in two
// parts, that many elements apart.
template <class T>
__global__ void __launch_bounds__(256) gemm_simt_kernel(const T* a, long long a_plane, const T* b, const GemmShape g, const Epilogue e) {
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
            float v = 0.0f;
            if (m0 + ra < g.m && k0 + ka < g.k) {
                const T* p = a + (m0 + ra) * g.am + (k0 + ka) * g.ak;
                v = to_f32(p[0]);
                if (a_plane) v = of_parts<T>(p[0], p[a_plane]);
            }
            sa[ka][ra] = v;
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

static int simt_gemm_check(const GemmShape& g, long long* tiles) {
    *tiles = ((g.m + SG_T - 1) / SG_T) * ((g.n + SG_T - 1) / SG_T);
    FG_REQUIRE(*tiles <= 0x7fffffffll, "%lld x %lld outputs: too many tiles", g.m, g.n);
    return FG_OK;
}

// ---- operands as the tensor cores take them ------------------------------------
//
// A matrix whose rows do not start on 16-byte boundaries is copied to one whose rows
// do; a float32 matrix becomes three bf16 planes, x = x0 + x1 + x2, each the rounding
// of what the ones before leave (a value past bf16's range is cut instead, an infinity
// or NaN has zeros behind it; bf16's last place is 2^-133, which values below 2^-109
// feel).  One pass over memory, eight columns a thread.
template <class T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs a) {
    long long i = blockIdx.x * 256ll + threadIdx.x;
    for (int k = 0; k < a.jobs; ++k) {
        const PackJob& j = a.job[k];
        const long long per_row = pack_stride(j.cols) / 8, n = j.rows * per_row;
        if (i >= n) {
            i -= n;
            continue;
        }
        // 64 bits take a division of a hundred instructions
        const long long row = i <= 0x7fffffff ? (long long)((unsigned)i / (unsigned)per_row) : i / per_row;
        const int col = (int)(i - row * per_row) * 8, left = j.cols - col;
        const T* in = static_cast<const T*>(j.in) + row * j.ld + col;
        alignas(16) T v[8];
        // as many bytes at a time as the row's start allows (rows on 8: 40,000 x 500 -> 64
        // bfloat16 27 us, 48 element by element; on 16, which are not packed, 15)
        const uintptr_t start = reinterpret_cast<uintptr_t>(in);
        if (left >= 8 && (start & 15) == 0) {
#pragma unroll
            for (int c = 0; c < (int)sizeof(T) / 2; ++c) reinterpret_cast<uint4*>(v)[c] = reinterpret_cast<const uint4*>(in)[c];
        } else if (left >= 8 && (start & 7) == 0) {
#pragma unroll
            for (int c = 0; c < (int)sizeof(T); ++c) reinterpret_cast<uint2*>(v)[c] = reinterpret_cast<const uint2*>(in)[c];
        } else if (left >= 8 && (start & 3) == 0) {
#pragma unroll
            for (int c = 0; c < 2 * (int)sizeof(T); ++c) reinterpret_cast<uint32_t*>(v)[c] = reinterpret_cast<const uint32_t*>(in)[c];
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = c < left ? in[c] : from_f32<T>(0.0f);
        }
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(static_cast<T*>(j.out) + row * pack_stride(j.cols) + col) = *reinterpret_cast<uint4*>(v);
        } else {
            alignas(16) __nv_bfloat16 o[3][8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                __nv_bfloat16 p[3];
                split3(v[c], p);
                o[0][c] = p[0];
                o[1][c] = p[1];
                o[2][c] = p[2];
            }
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(j.out) + row * pack_stride(j.cols) + col;
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(out + q * j.plane) = *reinterpret_cast<const uint4*>(o[q]);
        }
        return;
    }
}

template <class T>
static int pack(const PackArgs& a, cudaStream_t s) {
    long long n = 0;
    for (int k = 0; k < a.jobs; ++k) n += a.job[k].rows * (pack_stride(a.job[k].cols) / 8);
    if (n == 0) return FG_OK;
    FG_REQUIRE(n <= 0x7fffffffll * 256, "operands too large");
    pack_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    return check_launch("pack_kernel");
}

// ---- a few rows: the weights are read once ---------------------------------------
//
// A warp takes C output columns for all R rows: 32 lanes along k, 16 bytes a lane
// where the rows allow, then R C sums over the warp, halved at each step: lane l ends
// with one of them.  Bound by the latency of the loads, so all of a step's are asked
// for at once (8 rows of 1536 -> 768 f16: 4.5 us; with a branch on the row between
// them 11.3), and for one row of a large matrix by its bytes: 768 -> 1536 f16 2.3 us,
// 4096 -> 4096 5.8 us (5.8 TB/s, of which L2 holds a part).
//
// GATED: the two columns are a gate's and its partner's, `up` rows of w apart.
template <class T, int R, int C, bool GATED>
__global__ void __launch_bounds__(128) gemv_kernel(const T* __restrict__ x, const T* __restrict__ w, const GemmShape g,
                                                   int wide, const Epilogue e, int up) {
    constexpr int VEC = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    const long long n = (blockIdx.x * 4ll + (threadIdx.x >> 5)) * (GATED ? 1 : C);
    if (n >= (GATED ? up : g.n)) return;
    const T *wr[C], *xr[R];  // rows and columns past the last are the last again: no branch keeps loads apart
#pragma unroll
    for (int c = 0; c < C; ++c) wr[c] = w + (GATED ? n + (c ? up : 0) : min(n + c, g.n - 1)) * g.bn;
#pragma unroll
    for (int r = 0; r < R; ++r) xr[r] = x + min((long long)r, g.m - 1) * g.am;
    float acc[R * C];
#pragma unroll
    for (int i = 0; i < R * C; ++i) acc[i] = 0.0f;
    long long k0 = 0;
    if (wide) {
#pragma unroll(R* C > 4 ? 2 : 4)
        for (long long k = lane * VEC; k + VEC <= g.k; k += 32 * VEC) {
            alignas(16) T a[R][VEC], b[C][VEC];
#pragma unroll
            for (int c = 0; c < C; ++c) *reinterpret_cast<uint4*>(b[c]) = *reinterpret_cast<const uint4*>(wr[c] + k);
#pragma unroll
            for (int r = 0; r < R; ++r) *reinterpret_cast<uint4*>(a[r]) = *reinterpret_cast<const uint4*>(xr[r] + k);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        acc[r * C + c] = fmaf(to_f32(a[r][i]), to_f32(b[c][i]), acc[r * C + c]);
        }
        k0 = g.k / VEC * VEC;
    }
    for (long long k = k0 + lane; k < g.k; k += 32) {
        float b[C];
#pragma unroll
        for (int c = 0; c < C; ++c) b[c] = to_f32(wr[c][k]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float a = to_f32(xr[r][k]);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[r * C + c] = fmaf(a, b[c], acc[r * C + c]);
        }
    }
    int held = 0;  // which sum this lane ends with
#pragma unroll
    for (int o = 16, count = R * C; o > 0; o >>= 1) {
        if (count > 1) {
            count /= 2;
            const bool upper = lane & o;
            held += upper ? count : 0;
#pragma unroll
            for (int i = 0; i < R * C / 2; ++i)
                if (i < count) {
                    const float keep = upper ? acc[i + count] : acc[i], give = upper ? acc[i] : acc[i + count];
                    acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
        } else {
            acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
        }
    }
    const int row = held / C;
    if constexpr (GATED) {  // the partner's sum is in the lane of the last halving
        const float p = __shfl_xor_sync(0xffffffffu, acc[0], 16 / R);
        if (lane % (32 / (R * C)) == 0 && held % C == 0 && row < g.m) gated_store<T>(e, up, row, n, acc[0], p);
        return;
    }
    const long long col = n + held % C;
    if (lane % (32 / (R * C)) == 0 && row < g.m && col < g.n) epilogue_store<T>(e, row, col, acc[0]);
}

template <class T, int R, int C>
static int gemv_columns(const void* x, const void* w, const GemmShape& g, const Epilogue& e, cudaStream_t s) {
    auto lies = [&](const void* p, long long ld) { return aligned(p, 16) && ld * (int)sizeof(T) % 16 == 0; };
    gemv_kernel<T, R, C, false><<<(unsigned)((g.n + 4 * C - 1) / (4 * C)), 128, 0, s>>>(
        static_cast<const T*>(x), static_cast<const T*>(w), g, lies(x, g.am) && lies(w, g.bn), e, 0);
    return check_launch("gemv_kernel");
}

template <class T, int R>
static int gemv_gated(const void* x, const void* w, const GemmShape& g, const Epilogue& e, int up, cudaStream_t s) {
    auto lies = [&](const void* p, long long ld) { return aligned(p, 16) && ld * (int)sizeof(T) % 16 == 0; };
    gemv_kernel<T, R, 2, true><<<(unsigned)((up + 3) / 4), 128, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(w), g,
                                                                        lies(x, g.am) && lies(w, g.bn), e, up);
    return check_launch("gemv_kernel");
}

// Two columns a warp where columns alone give every SM 16 warps (4096 x 4096 f16, 8
// rows: 14.6 us with two, 18.7 with one; 1536 x 768: 5.5 and 4.5).
template <class T, int R>
static int gemv_of(const void* x, const void* w, const GemmShape& g, const Epilogue& e, cudaStream_t s) {
    return g.n > 16ll * device_attr(cudaDevAttrMultiProcessorCount) ? gemv_columns<T, R, 2>(x, w, g, e, s)
                                                                    : gemv_columns<T, R, 1>(x, w, g, e, s);
}

template <class T>
static int gemv(const void* x, const void* w, const GemmShape& g, const Epilogue& e, cudaStream_t s) {
    return g.m == 1   ? gemv_columns<T, 1, 1>(x, w, g, e, s)
           : g.m == 2 ? gemv_of<T, 2>(x, w, g, e, s)
           : g.m <= 4 ? gemv_of<T, 4>(x, w, g, e, s)
                      : gemv_of<T, GEMV_ROWS>(x, w, g, e, s);
}

template <class T>
static int gemm(const Operand& a, const Operand& b, const GemmShape& g, const Epilogue& e, void* ws, cudaStream_t s) {
    if (g.m == 0 || g.n == 0) return FG_OK;
    constexpr int dtype = sizeof(T) == 4 ? FG_DTYPE_F32 : std::is_same<T, __half>::value ? FG_DTYPE_F16 : FG_DTYPE_BF16;
    if ((sizeof(T) == 2 || a.plane) && tc_gemm_fits(a.p, b.p, g)) return tc_gemm(dtype, a.p, a.plane, b.p, b.plane, g, e, ws, s);
    long long tiles;
    const int rc = simt_gemm_check(g, &tiles);
    if (rc) return rc;
    gemm_simt_kernel<T><<<(unsigned)tiles, 256, 0, s>>>(static_cast<const T*>(a.p), sizeof(T) == 2 ? a.plane : 0,
                                                         static_cast<const T*>(b.p), g, e);
    return check_launch("gemm_simt_kernel");
}

// GELU's and SiLU's dz is worked out in 32 bits, and 16-bit operands take it in two parts
// (split2): rounded to one, the gradients were off by 0.0023 of their norm, not the 0.0017
// of their own rounding, and float16 lost terms below 3e-8 and made those past 65504
// infinite.  ReLU's is dy or 0, exact as it is.
static bool in_parts(const fg_linear_params* p) {
    return p->dtype != FG_DTYPE_F32 && (p->activation == FG_ACT_GELU || p->activation == FG_ACT_SILU);
}

// dz = dy act'(pre) and the column sums of dz, in one pass over dy and pre: a warp
// takes 32 x VEC columns of every eighth row of its block's range, two rows at a
// time, sums them in registers, and the block writes one partial row.  Bound by memory
// and by GELU's arithmetic: 10,000 x 1536 bf16 with GELU 25.8 us, of which its two parts of
// dz are 31 MB more to write (4.8 TB/s), with ReLU 21 us (4.4), at three blocks an SM.
constexpr int DZ_WARPS = 8;

struct DzArgs {
    const void *dy, *pre;
    void* dz;     // NULL: not stored
    float* part;  // NULL: no sums
    long long lddy, ldp, rows, per, plane;
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
__global__ void __launch_bounds__(DZ_WARPS * 32, 3) dz_kernel(const DzArgs g) {
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
                constexpr bool TWO = sizeof(T) == 2 && (ACT == FG_ACT_GELU || ACT == FG_ACT_SILU);
                alignas(16) T o[VEC], low[TWO ? VEC : 1];
#pragma unroll
                for (int i = 0; i < VEC; i += 2) {
                    float v0 = to_f32(d[u][i]), v1 = to_f32(d[u][i + 1]);
                    dz_pair<ACT, sizeof(T) == 2>(v0, v1, to_f32(p[u][i]), to_f32(p[u][i + 1]));
                    v0 = i < left ? v0 : 0.0f;  // columns past the last
                    v1 = i + 1 < left ? v1 : 0.0f;
                    sum[i] += v0;
                    sum[i + 1] += v1;
                    if constexpr (TWO) {
                        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
                        split2(v0, v1, *reinterpret_cast<T2*>(o + i), *reinterpret_cast<T2*>(low + i));
                    } else {
                        o[i] = from_f32<T>(v0);
                        o[i + 1] = from_f32<T>(v1);
                    }
                }
                if (g.dz) {  // an operand as the tensor cores take it: one or two of 16 bits, or three planes; padded rows
                    const long long at = q * pack_stride(g.dim) + j;
                    if constexpr (sizeof(T) == 2) {
                        *reinterpret_cast<uint4*>(static_cast<T*>(g.dz) + at) = *reinterpret_cast<const uint4*>(o);
                        if constexpr (TWO)
                            *reinterpret_cast<uint4*>(static_cast<T*>(g.dz) + g.plane + at) = *reinterpret_cast<const uint4*>(low);
                    } else {
                        alignas(8) __nv_bfloat16 pl[3][VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            __nv_bfloat16 w[3];
                            split3(o[i], w);
                            pl[0][i] = w[0];
                            pl[1][i] = w[1];
                            pl[2][i] = w[2];
                        }
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(g.dz) + k * g.plane + at) =
                                *reinterpret_cast<const uint2*>(pl[k]);
                    }
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

// Row ranges: three blocks to an SM over the column tiles, 16 rows at least to a range.
static int dz_split(long long rows, int dim, int elem) {
    const int cols = 32 * (16 / elem), tiles = (dim + cols - 1) / cols;
    const long long fill = std::max(1ll, 3ll * std::max(1, device_attr(cudaDevAttrMultiProcessorCount)) / tiles);
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

int linear_check(const fg_linear_params* p, Strides& t) {
    FG_REQUIRE(p, "null params");
    FG_REQUIRE(p->rows >= 0 && p->in_dim >= 1 && p->out_dim >= 1, "bad linear shape");
    if (p->rows > LINEAR_MAX || p->in_dim > LINEAR_MAX || p->out_dim > LINEAR_MAX)
        return fail(FG_ERR_UNSUPPORTED, "a dimension above %lld", LINEAR_MAX);
    FG_REQUIRE(float_dtype(p->dtype), "unknown dtype %d", p->dtype);
    FG_REQUIRE((p->unaligned & ~(FG_LINEAR_X | FG_LINEAR_W | FG_LINEAR_DY)) == 0, "unknown operand in unaligned %d", p->unaligned);
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

struct ForwardWs {
    void *x, *w, *product;
};

static size_t forward_carve(const fg_linear_params* p, const Strides& t, void* ws, size_t bytes, ForwardWs& f) {
    Carve c(ws, bytes);
    f = ForwardWs{};
    if (p->rows <= GEMV_ROWS) return 0;
    if (needs_pack(p->dtype, t.x, p->unaligned & FG_LINEAR_X)) f.x = c.take<char>(pack_bytes(p->dtype, p->rows, p->in_dim));
    if (needs_pack(p->dtype, t.w, p->unaligned & FG_LINEAR_W)) f.w = c.take<char>(pack_bytes(p->dtype, p->out_dim, p->in_dim));
    const size_t n = tc_gemm_workspace(tc_products(p->dtype, false), forward_shape(p, t));
    if (n) f.product = c.take<char>(n);
    return c.used;
}

// x or w: as it lies, or queued to be packed.
Operand operand(int dtype, const void* p, long long rows, int cols, long long ld, bool off, void* room, PackArgs& a) {
    if (!needs_pack(dtype, ld, off)) return {p, ld, 0};
    const long long stride = pack_stride(cols), plane = dtype == FG_DTYPE_F32 ? rows * stride : 0;
    a.job[a.jobs++] = PackJob{p, room, rows, ld, plane, cols};
    return {room, stride, plane};
}

template <class T>
static int linear_forward(const fg_linear_params* p, const Strides& t, const void* x, const void* w, const Epilogue& e,
                          const ForwardWs& f, cudaStream_t s) {
    if (p->rows <= GEMV_ROWS) return gemv<T>(x, w, forward_shape(p, t), e, s);
    PackArgs jobs{};
    const Operand a = operand(p->dtype, x, p->rows, p->in_dim, t.x, p->unaligned & FG_LINEAR_X, f.x, jobs);
    const Operand b = operand(p->dtype, w, p->out_dim, p->in_dim, t.w, p->unaligned & FG_LINEAR_W, f.w, jobs);
    const int rc = pack<T>(jobs, s);
    if (rc) return rc;
    return gemm<T>(a, b, GemmShape{p->rows, p->out_dim, p->in_dim, a.ld, 1, b.ld, 1}, e, f.product, s);
}

// ---- gradients of a few rows: one launch -----------------------------------------
//
// The first blocks take dx, 64 columns each: w is read once, a warp taking every
// sixteenth of its rows, and dz of 512 columns at a time is worked out in shared
// memory; the others take dw and db, four rows of w each.  dz stays in 32 bits.  Bound by
// the latency of w's loads, 32 rows of it under way in a block, and so by out_dim; the
// launches of more rows (dz, its sums, two products) are bound by their number.  Measured,
// theirs in brackets: bf16 768 -> 1536 one row 10.9 us (17.8), eight 22.2 (18.7, but a call
// is 25 us, not 29); four rows of 2048 -> 2560 23.6 (27.2), of 1024 -> 4096 36 (23), of
// 8192 -> 8192 143 (101); eight of 8192 -> 1024 35 (27).  float32, four rows: 1024 -> 4096
// 38 (53), 64 -> 8192 70 (35).
bool few(const fg_linear_params* p) {
    const int wide = p->dtype == FG_DTYPE_F32 ? 2 : 1;
    return p->rows >= 1 && (p->rows <= 4 ? p->out_dim <= 2560 * wide
                                         : p->rows <= GEMV_ROWS && p->out_dim <= 1536 * wide &&
                                               (long long)p->in_dim * p->out_dim <= 1 << 22);
}

constexpr int FEW_NT = 512, FEW_COLS = 64, FEW_OUT = 4;

template <class T>
__device__ __forceinline__ float dz_of(const FewArgs& g, int r, int o) {
    if (g.up) {
        const int j = o < g.up ? o : o - g.up;
        const T* pre = static_cast<const T*>(g.pre) + r * g.ldp;
        const float d = to_f32(static_cast<const T*>(g.dy)[r * g.lddy + j]), z = to_f32(pre[j]);
        return o < g.up ? d * to_f32(pre[g.up + j]) * activate_grad<false>(z, g.act) : d * activate<false>(z, g.act);
    }
    const float d = to_f32(static_cast<const T*>(g.dy)[r * g.lddy + o]);
    return g.act == FG_ACT_NONE ? d : d * activate_grad<false>(to_f32(static_cast<const T*>(g.pre)[r * g.ldp + o]), g.act);
}

template <class T, int R>
__global__ void __launch_bounds__(FEW_NT) few_rows_kernel(const FewArgs g) {
    __shared__ float s[FEW_NT / 32][R][FEW_COLS];  // warps' sums; before, dz of 512 columns
    float* dz = &s[0][0][0];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if ((int)blockIdx.x < g.dx_blocks) {
        const int j0 = blockIdx.x * FEW_COLS + lane, j1 = j0 + 32;
        const T* w = static_cast<const T*>(g.w);
        float acc[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][0] = acc[r][1] = 0.0f;
        for (int base = 0; base < g.out_dim; base += FEW_NT) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; ++r) dz[r * FEW_NT + tid] = r < g.rows && base + tid < g.out_dim ? dz_of<T>(g, r, base + tid) : 0.0f;
            __syncthreads();
            const int last = min(FEW_NT, g.out_dim - base) - 1, c0 = min(j0, g.in_dim - 1), c1 = min(j1, g.in_dim - 1);
#pragma unroll 16
            for (int o = warp; o < FEW_NT; o += FEW_NT / 32) {
                if (o > last) break;
                const T* row = w + (base + o) * g.ldw;
                const float a = to_f32(row[c0]), b = to_f32(row[c1]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    acc[r][0] = fmaf(dz[r * FEW_NT + o], a, acc[r][0]);
                    acc[r][1] = fmaf(dz[r * FEW_NT + o], b, acc[r][1]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[warp][r][lane] = acc[r][0];
            s[warp][r][lane + 32] = acc[r][1];
        }
        __syncthreads();
        const int r = tid / FEW_COLS, c = tid % FEW_COLS, j = blockIdx.x * FEW_COLS + c;
        if (r < min(R, g.rows) && j < g.in_dim) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < FEW_NT / 32; ++k) v += s[k][r][c];
            static_cast<T*>(g.dx)[(long long)r * g.in_dim + j] = from_f32<T>(v);
        }
        return;
    }
    const int o0 = (blockIdx.x - g.dx_blocks) * FEW_OUT;
    if (tid < FEW_OUT * R) {
        const int r = tid / FEW_OUT, o = o0 + tid % FEW_OUT;
        dz[tid] = r < g.rows && o < g.out_dim ? dz_of<T>(g, r, o) : 0.0f;
    }
    __syncthreads();
    if (g.db && tid < FEW_OUT && o0 + tid < g.out_dim) {
        float v = 0.0f;
        for (int r = 0; r < R; ++r) v += dz[r * FEW_OUT + tid];
        static_cast<T*>(g.db)[o0 + tid] = from_f32<T>(v);
    }
    if (!g.dw) return;
    for (int i = tid; i < g.in_dim; i += FEW_NT) {
        float v[FEW_OUT] = {};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float x = r < g.rows ? to_f32(static_cast<const T*>(g.x)[r * g.ldx + i]) : 0.0f;
#pragma unroll
            for (int k = 0; k < FEW_OUT; ++k) v[k] = r < g.rows ? fmaf(dz[r * FEW_OUT + k], x, v[k]) : v[k];
        }
#pragma unroll
        for (int k = 0; k < FEW_OUT; ++k)
            if (o0 + k < g.out_dim) static_cast<T*>(g.dw)[(long long)(o0 + k) * g.in_dim + i] = from_f32<T>(v[k]);
    }
}

template <class T>
static int few_rows(FewArgs g, cudaStream_t s) {
    g.dx_blocks = g.dx ? (g.in_dim + FEW_COLS - 1) / FEW_COLS : 0;
    const int blocks = g.dx_blocks + (g.dw || g.db ? (g.out_dim + FEW_OUT - 1) / FEW_OUT : 0);
    if (!blocks) return FG_OK;
    auto kernel = g.rows == 1 ? &few_rows_kernel<T, 1>
                  : g.rows == 2 ? &few_rows_kernel<T, 2>
                  : g.rows <= 4 ? &few_rows_kernel<T, 4>
                                : &few_rows_kernel<T, GEMV_ROWS>;
    kernel<<<blocks, FEW_NT, 0, s>>>(g);
    return check_launch("few_rows_kernel");
}

struct BackwardWs {
    void *dz, *x, *w, *product;
    float* part;
};

static size_t backward_carve(const fg_linear_params* p, const Strides& t, void* ws, size_t bytes, BackwardWs& w) {
    Carve c(ws, bytes);
    w = BackwardWs{};
    if (few(p)) return 0;
    if (p->activation != FG_ACT_NONE || needs_pack(p->dtype, t.y, p->unaligned & FG_LINEAR_DY))
        w.dz = c.take<char>(pack_bytes(p->dtype, p->rows, p->out_dim) * (in_parts(p) ? 2 : 1));
    if (needs_pack(p->dtype, t.x, p->unaligned & FG_LINEAR_X)) w.x = c.take<char>(pack_bytes(p->dtype, p->rows, p->in_dim));
    if (needs_pack(p->dtype, t.w, p->unaligned & FG_LINEAR_W)) w.w = c.take<char>(pack_bytes(p->dtype, p->out_dim, p->in_dim));
    const int products = tc_products(p->dtype, in_parts(p));
    const size_t n = std::max(tc_gemm_workspace(products, dx_shape(p, t, t.y)), tc_gemm_workspace(products, dw_shape(p, t, t.y)));
    if (n) w.product = c.take<char>(n);
    w.part = c.take<float>((size_t)dz_split(p->rows, p->out_dim, dtype_size(p->dtype)) * p->out_dim);
    return c.used;
}

template <class T>
static int linear_backward(const fg_linear_params* p, const Strides& t, const void* dy, const void* x, const void* w,
                           const void* pre, void* dx, void* dw, void* dbias, const BackwardWs& ws, cudaStream_t s) {
    if (few(p))
        return few_rows<T>(FewArgs{dy, x, w, pre, dx, dw, dbias, t.y, t.x, t.w, t.p, (int)p->rows, p->in_dim, p->out_dim,
                                   p->activation, 0, 0},
                           s);
    const bool act = p->activation != FG_ACT_NONE, store = (act || needs_pack(p->dtype, t.y, p->unaligned & FG_LINEAR_DY)) && (dx || dw);
    const int split = p->rows ? dz_split(p->rows, p->out_dim, sizeof(T)) : 0;
    const long long plane = p->dtype == FG_DTYPE_F32 || in_parts(p) ? p->rows * pack_stride(p->out_dim) : 0;
    int rc;
    if (split && (store || dbias)) {
        const DzArgs g{dy, act ? pre : nullptr, store ? ws.dz : nullptr, dbias ? ws.part : nullptr, t.y, t.p, p->rows, 0,
                       plane, p->out_dim, p->activation, 0};
        if ((rc = launch_dz<T>(g, split, s))) return rc;
    }
    if (dbias) {
        dz_reduce_kernel<T><<<(p->out_dim + 31) / 32, 1024, 0, s>>>(ws.part, split, p->out_dim, (T*)dbias);
        if ((rc = check_launch("dz_reduce_kernel"))) return rc;
    }
    const Operand dz = store ? Operand{ws.dz, pack_stride(p->out_dim), plane} : Operand{dy, t.y, 0};
    PackArgs jobs{};
    Operand xo{}, wo{};
    if (dx && p->rows) wo = operand(p->dtype, w, p->out_dim, p->in_dim, t.w, p->unaligned & FG_LINEAR_W, ws.w, jobs);
    if (dw && p->rows) xo = operand(p->dtype, x, p->rows, p->in_dim, t.x, p->unaligned & FG_LINEAR_X, ws.x, jobs);
    if ((rc = pack<T>(jobs, s))) return rc;
    Epilogue e{};
    e.ldy = p->in_dim;
    if (dx && p->rows) {
        e.y = dx;
        rc = gemm<T>(dz, wo, GemmShape{p->rows, p->in_dim, p->out_dim, dz.ld, 1, 1, wo.ld}, e, ws.product, s);
        if (rc) return rc;
    }
    if (dw) {
        e.y = dw;
        rc = gemm<T>(dz, xo, GemmShape{p->out_dim, p->in_dim, p->rows, 1, dz.ld, 1, xo.ld}, e, ws.product, s);
        if (rc) return rc;
    }
    return FG_OK;
}

// ---- for the gated layer ---------------------------------------------------------

#define FG_TYPED(call)                                  \
    (dtype == FG_DTYPE_F32   ? call(float)              \
     : dtype == FG_DTYPE_F16 ? call(__half)             \
                             : call(__nv_bfloat16))

int linear_pack(int dtype, const PackArgs& a, cudaStream_t s) {
#define FG_CALL(T) pack<T>(a, s)
    return FG_TYPED(FG_CALL);
#undef FG_CALL
}

int linear_gemm(int dtype, const Operand& a, const Operand& b, const GemmShape& g, const Epilogue& e, void* ws, cudaStream_t s) {
#define FG_CALL(T) gemm<T>(a, b, g, e, ws, s)
    return FG_TYPED(FG_CALL);
#undef FG_CALL
}

int linear_gemv_gated(int dtype, const void* x, const void* w, const GemmShape& g, const Epilogue& e, int up, cudaStream_t s) {
#define FG_CALL(T)                                        \
    (g.m == 1   ? gemv_gated<T, 1>(x, w, g, e, up, s)     \
     : g.m == 2 ? gemv_gated<T, 2>(x, w, g, e, up, s)     \
     : g.m <= 4 ? gemv_gated<T, 4>(x, w, g, e, up, s)     \
                : gemv_gated<T, GEMV_ROWS>(x, w, g, e, up, s))
    return FG_TYPED(FG_CALL);
#undef FG_CALL
}

int linear_few_rows(int dtype, const FewArgs& g, cudaStream_t s) {
#define FG_CALL(T) few_rows<T>(g, s)
    return FG_TYPED(FG_CALL);
#undef FG_CALL
}

int linear_column_sums(int dtype, const float* part, int parts, int dim, void* out, cudaStream_t s) {
#define FG_CALL(T) (dz_reduce_kernel<T><<<(dim + 31) / 32, 1024, 0, s>>>(part, parts, dim, static_cast<T*>(out)), check_launch("dz_reduce_kernel"))
    return FG_TYPED(FG_CALL);
#undef FG_CALL
}
#undef FG_TYPED

}  // namespace fg

using namespace fg;

extern "C" {

int fg_linear_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        Strides t;
        const int rc = linear_check(params, t);
        if (rc) return rc;
        ForwardWs f;
        *bytes = forward_carve(params, t, nullptr, 0, f);
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
        ForwardWs f;
        const int bad = adapter_ws(workspace, workspace_bytes, forward_carve(params, t, nullptr, 0, f));
        if (bad) return bad;
        forward_carve(params, t, workspace, workspace_bytes, f);
        const Epilogue e{bias, residual, pre, y, t.r, t.p, t.y, params->activation};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return params->dtype == FG_DTYPE_F32   ? linear_forward<float>(params, t, x, w, e, f, s)
               : params->dtype == FG_DTYPE_F16 ? linear_forward<__half>(params, t, x, w, e, f, s)
                                               : linear_forward<__nv_bfloat16>(params, t, x, w, e, f, s);
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
