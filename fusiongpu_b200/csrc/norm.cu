// norm.cu -- layer norm over rows and its gradients.
//
//   y = (x - m) r w + b,   m = avg(x),  r = 1 / sqrt(avg((x - m)^2) + eps)
//   h = (x - m) r,  a = dy w:   dx = r (a - avg(a) - h avg(a h)),
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// Both are bound by memory: forward reads x and writes y, backward reads x and
// dy and writes dx, each once.  A row lives in the registers of a group of G
// threads -- 8 (rows up to 16 elements a thread: four rows to a warp, so that
// short rows still fill 128-byte requests), 32 (up to 512, of 16 bits 768, backward
// 1024), 128 (up to 4096) or 512 -- and the variance is taken over the centred values,
// a second pass that costs no memory traffic.  The weight's gradients are summed in
// registers over the rows a group takes in turn, joined per block in shared memory,
// and written as one partial row per block, which ln_reduce_kernel adds in one fixed
// order: no atomics, the same bits every time.  Measured, forward and backward with
// the weight's gradients: 1,000,000 x 128 f32 162 and 238 us (6.3, 6.5 TB/s), 260,000
// x 768 f16 149 and 218 us (5.4, 5.5 TB/s), 50,000 x 4096 bf16 158 and 249 us (5.2,
// 4.9 TB/s), 10,000 x 768 f16 8.1 and 13.4 us, one row 3.1 and 5.7 us.
#include <algorithm>

#include "adapter_common.cuh"
#include "packed.cuh"

namespace fg {

constexpr int LN_MAX_DIM = 16384;

struct NormArgs {
    const void *x, *dy, *w, *b;
    const float *mean, *rstd;
    void *y, *dx;
    float *out_mean, *out_rstd, *part;
    long long rows, ldx, ldy, lddx;
    int dim, w_f32;
    int params;  // the weight's gradients are wanted
    float eps;
};

// VEC elements of a row: one 16-byte access where every row and the parameters start
// on a 16-byte boundary (wide), else single ones, in the same place of the same thread: the
// results do not depend on alignment.  VEC is 1 where dim is no multiple of 16 bytes.
template <class T, int VEC>
struct Chunk {
    T v[VEC];
};

template <class T, int VEC>
__device__ __forceinline__ void load_chunk(Chunk<T, VEC>& c, const T* p, int wide) {
    if (VEC * sizeof(T) == 16 && wide) {  // read once: not kept in L1, which holds the parameters
        uint4 u;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                     : "l"(p));
        *reinterpret_cast<uint4*>(c.v) = u;
    } else {
        // not __ldg: for 16-bit types that is an asm that may be moved above the caller's bounds check
#pragma unroll
        for (int i = 0; i < VEC; ++i) c.v[i] = p[i];
    }
}

template <class T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const float* f, int wide) {
    alignas(16) T v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = from_f32<T>(f[i]);
    if (VEC * sizeof(T) == 16 && wide) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[i] = v[i];
    }
}

// VEC parameters from column j: of T or float, `absent` without any.
template <class T, int VEC>
__device__ __forceinline__ void load_params(float* f, const void* p, int f32, int wide, int j, float absent) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = absent;
    } else if (VEC == 1 || !wide) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = f32 ? static_cast<const float*>(p)[j + i] : to_f32(static_cast<const T*>(p)[j + i]);
    } else if (f32) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + j + i));
            f[i] = q.x;
            f[i + 1] = q.y;
            f[i + 2] = q.z;
            f[i + 3] = q.w;
        }
    } else {
        alignas(16) T v[VEC];
        *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + j));
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = to_f32(v[i]);
    }
}

template <int G>
constexpr int ln_block() {
    return G < 128 ? 256 : G;
}

// Sum over the group's threads, in each of them.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* s) {
    if (G > 32) return block_sum<ln_block<G>()>(v, s);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Blocks of the forward kernel per SM: by registers, a thread holding w, b, a row and
// the next in its own type (of G = 512, one row).
constexpr int ln_forward_per_sm(int G, int E, int bytes) {
    return G == 512 ? 1 : 65536 / ((G == 128 ? 128 : 256) * (E * (3 + bytes / 4) + 32 + E * (bytes & 2) / 4));
}

// Groups take rows in turn: the parameters are read once and stay in registers, and
// the next row is fetched before this one is worked on.  (With a row's parameters
// read from L1 for every row instead, 260,000 x 768 f16 with float parameters took
// 256 us, not 149: 6 KB of them to a row of 1.5 KB.)  Not so for G = 512, whose
// registers hold one row: there w and b are read for each.  16-bit rows of 769 to 1024
// columns go to 128 threads: 200,000 x 1024 f16 166 us, in one warp each 168.
template <class T, int VEC, int NCH, int G, bool WIDE>
__global__ void __launch_bounds__(ln_block<G>(), ln_forward_per_sm(G, NCH* VEC, sizeof(T))) ln_forward_kernel(const NormArgs g) {
    constexpr int NT = ln_block<G>(), RPB = NT / G, E = NCH * VEC;
    constexpr bool HOLD = G < 512;
    __shared__ float s[NT / 32];
    const int gl = threadIdx.x % G;
    const float inv = 1.0f / (float)g.dim;
    const long long step = (long long)gridDim.x * RPB;
    Chunk<T, VEC> c[NCH];
    auto fetch = [&](long long r) {
        if (r >= g.rows) return;
        const T* x = static_cast<const T*>(g.x) + r * g.ldx;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int j = (k * G + gl) * VEC;
            if (j < g.dim) load_chunk<T, VEC>(c[k], x + j, WIDE);
        }
    };
    float w[HOLD ? E : VEC], b[HOLD ? E : VEC];
    auto params = [&](int k, int at) {
        const int j = (k * G + gl) * VEC;
        if (j < g.dim) {
            load_params<T, VEC>(w + at, g.w, g.w_f32, WIDE, j, 1.0f);
            load_params<T, VEC>(b + at, g.b, g.w_f32, WIDE, j, 0.0f);
        }
    };
    const long long first = (long long)blockIdx.x * RPB + threadIdx.x / G;
    fetch(first);
    if (HOLD) {
#pragma unroll
        for (int k = 0; k < NCH; ++k) params(k, k * VEC);
    }
    // every thread of a warp stays in the loop as long as one of its rows exists
    for (long long r = first, r0 = r - (threadIdx.x % 32) / G; (G > 32 ? r : r0) < g.rows; r += step, r0 += step) {
        float v[E], t = 0.0f;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const bool have = r < g.rows && (k * G + gl) * VEC < g.dim;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[k * VEC + i] = have ? to_f32(c[k].v[i]) : 0.0f;
                t += v[k * VEC + i];
            }
        }
        fetch(r + step);
        const float mean = group_sum<G>(t, s) * inv;
        t = 0.0f;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const bool have = (k * G + gl) * VEC < g.dim;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[k * VEC + i] -= mean;
                if (have) t = fmaf(v[k * VEC + i], v[k * VEC + i], t);
            }
        }
        const float rstd = 1.0f / sqrtf(group_sum<G>(t, s) * inv + g.eps);
        if (r >= g.rows) continue;
        T* y = static_cast<T*>(g.y) + r * g.ldy;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int j = (k * G + gl) * VEC, at = HOLD ? k * VEC : 0;
            if (!HOLD) params(k, 0);
            if (j < g.dim) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = fmaf(__fmul_rn(v[k * VEC + i], rstd), w[at + i], b[at + i]);
                store_chunk<T, VEC>(y + j, o, WIDE);
            }
        }
        if (g.out_mean && gl == 0) {
            g.out_mean[r] = mean;
            g.out_rstd[r] = rstd;
        }
    }
}

// Backward: threads of a block and blocks per SM, by registers: a thread holds two sums
// and w for each of its E columns, x and dy of a row and, AHEAD, of the next one, in
// their own type (16-bit ones two to a register, but where VEC is 1).
constexpr int ln_row_regs(int E, int VEC, int bytes) { return 2 * E * (VEC == 1 ? 4 : bytes) / 4; }
constexpr bool ln_ahead(int E, int VEC, int bytes) { return ln_row_regs(E, VEC, bytes) <= 32; }
constexpr int ln_backward_regs(int E, int VEC, int bytes) {
    return 3 * E + ln_row_regs(E, VEC, bytes) * (ln_ahead(E, VEC, bytes) ? 2 : 1) + 32;
}
constexpr int ln_backward_block(int G, int E, int VEC, int bytes) {
    const int regs = ln_backward_regs(E, VEC, bytes);
    return G >= 128 ? G : regs > 128 && regs <= 168 ? 384 : 256;
}
constexpr int ln_backward_per_sm(int G, int E, int VEC, int bytes) {
    const int n = 65536 / (128 * ln_backward_regs(E, VEC, bytes));
    return G == 512 ? 1 : G == 128 ? (n < 6 ? n : 6) : ln_backward_regs(E, VEC, bytes) > 128 ? 1 : 2;
}

// Sums of two values over the group.
template <int G>
__device__ __forceinline__ void group_sum2(float& a, float& b, float (*s)[2]) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (G <= 32) return;
    __syncthreads();  // the previous call's readers are done with s
    if ((threadIdx.x & 31) == 0) {
        s[threadIdx.x >> 5][0] = a;
        s[threadIdx.x >> 5][1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) {
        a += s[w][0];
        b += s[w][1];
    }
}

// Groups take rows in turn; x and dy of the next row are fetched before this one
// is worked on, and stay in their own type until they are used.  The sums for the
// weight's gradients are in registers (G = 512: in shared memory, each thread its own
// columns, and w is read for each row).  Instructions bound it next to memory, so the
// arithmetic is packed, two columns an instruction, and rows on 16-byte boundaries are a
// kernel without any branch on that, whose loads the compiler leaves ahead of the work:
// 260,000 x 768 f16 300 us without either, 287 packed, 218 with both.  16-bit rows of
// 769 to 1024 columns: 216 us in one warp each, 290 over 128 threads (200,000 x 1024).
template <class T, int VEC, int NCH, int G, bool WIDE>
__global__ void __launch_bounds__(ln_backward_block(G, NCH* VEC, VEC, sizeof(T)),
                                  ln_backward_per_sm(G, NCH* VEC, VEC, sizeof(T))) ln_backward_kernel(const NormArgs g) {
    constexpr int E = NCH * VEC, NT = ln_backward_block(G, E, VEC, sizeof(T)), RPB = NT / G;
    constexpr bool SMEM = G == 512, AHEAD = ln_ahead(E, VEC, sizeof(T));
    extern __shared__ __align__(16) float sm[];  // rows of sums, stored four at a time where dim is a multiple of 4
    __shared__ float s[NT / 32][2];
    const int gl = threadIdx.x % G;
    const float inv = 1.0f / (float)g.dim;
    const long long step = (long long)gridDim.x * RPB;
    uint64_t dw[SMEM ? 1 : E / 2], db[SMEM ? 1 : E / 2];
    constexpr int P = VEC < 2 ? 2 : VEC;  // columns whose parameters are loaded and results stored together
    float w[SMEM ? P : E];
    auto column = [&](int e) { return (e / VEC * G + gl) * VEC + e % VEC; };
    auto params = [&](int e) {  // of columns e .. e + P - 1
#pragma unroll
        for (int i = 0; i < P; i += VEC) {
            float* at = w + (SMEM ? i : e + i);
            if (column(e + i) < g.dim)
                load_params<T, VEC>(at, g.w, g.w_f32, WIDE, column(e + i), 1.0f);
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k) at[k] = 0.0f;
        }
    };
    auto weights = [&](int e) { return pair2(w[SMEM ? e % P : e], w[SMEM ? e % P + 1 : e + 1]); };
    if (SMEM) {
        for (int k = 0; k < NCH; ++k)
            for (int i = 0; i < VEC; ++i) {
                const int j = (k * G + gl) * VEC + i;
                if (j < g.dim) sm[j] = sm[g.dim + j] = 0.0f;
            }
    } else {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) dw[i] = db[i] = 0;
    }
    // Columns and rows that are not there are zeros, and add nothing.
    struct Row {
        Chunk<T, VEC> x[NCH], d[NCH];
        float mean, rstd;
        __device__ __forceinline__ float2 get(const Chunk<T, VEC> (&c)[NCH], int e) const {
            return make_float2(to_f32(c[e / VEC].v[e % VEC]), to_f32(c[(e + 1) / VEC].v[(e + 1) % VEC]));
        }
    };
    auto clear = [&](Row& row) {
        row.mean = row.rstd = 0.0f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) row.x[k].v[i] = row.d[k].v[i] = from_f32<T>(0.0f);
    };
    auto fetch = [&](Row& row, long long r) {
        if (r >= g.rows) {
            clear(row);
            return;
        }
        const T* x = static_cast<const T*>(g.x) + r * g.ldx;
        const T* d = static_cast<const T*>(g.dy) + r * g.ldy;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int j = (k * G + gl) * VEC;
            if (j < g.dim) {
                load_chunk<T, VEC>(row.x[k], x + j, WIDE);
                load_chunk<T, VEC>(row.d[k], d + j, WIDE);
            }
        }
        row.mean = __ldg(g.mean + r);
        row.rstd = __ldg(g.rstd + r);
    };
    Row cur, next;
    const long long first = (long long)blockIdx.x * RPB + threadIdx.x / G;
    clear(AHEAD ? next : cur);
    if (AHEAD) fetch(next, first);
    if (!SMEM) {
#pragma unroll
        for (int e = 0; e < E; e += P) params(e);
    }
    for (long long r = first, r0 = r - (threadIdx.x % 32) / G; (G > 32 ? r : r0) < g.rows; r += step, r0 += step) {
        if (AHEAD) {
            cur = next;
            fetch(next, r + step);
        } else {
            fetch(cur, r);
        }
        const uint64_t off = pair2(-cur.mean, -cur.mean), by = pair2(cur.rstd, cur.rstd);
        uint64_t sa2 = 0, sah2 = 0;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 xf = cur.get(cur.x, e), df = cur.get(cur.d, e);
            const uint64_t d = pair2(df.x, df.y), h = mul2(add2(pair2(xf.x, xf.y), off), by);
            if (SMEM && e % P == 0) params(e);
            const uint64_t a = mul2(d, weights(e));
            if (SMEM) {
                float dh[2];
                unpair2(mul2(d, h), dh[0], dh[1]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = column(e + i);
                    if (j < g.dim) {
                        sm[j] += dh[i];
                        sm[g.dim + j] += i ? df.y : df.x;
                    }
                }
            } else {
                dw[SMEM ? 0 : e / 2] = fma2(d, h, dw[SMEM ? 0 : e / 2]);
                db[SMEM ? 0 : e / 2] = add2(d, db[SMEM ? 0 : e / 2]);
            }
            sa2 = add2(sa2, a);
            sah2 = fma2(a, h, sah2);
        }
        if (!g.dx) continue;
        float sa, sah, sa1, sah1;
        unpair2(sa2, sa, sa1);
        unpair2(sah2, sah, sah1);
        sa += sa1;
        sah += sah1;
        group_sum2<G>(sa, sah, s);
        if (r >= g.rows) continue;
        const uint64_t ma = pair2(-sa * inv, -sa * inv), mah = pair2(-sah * inv, -sah * inv);
        T* dx = static_cast<T*>(g.dx) + r * g.lddx;
        float o[P];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            if (SMEM && e % P == 0) params(e);
            const float2 xf = cur.get(cur.x, e), df = cur.get(cur.d, e);
            const uint64_t h = mul2(add2(pair2(xf.x, xf.y), off), by);
            const uint64_t a = fma2(pair2(df.x, df.y), weights(e), ma);  // dy w - avg(a)
            unpair2(mul2(by, fma2(h, mah, a)), o[e % P], o[e % P + 1]);
            if ((e + 2) % P == 0) {
#pragma unroll
                for (int i = 0; i < P; i += VEC) {
                    const int j = column(e + 2 - P + i);
                    if (j < g.dim) store_chunk<T, VEC>(dx + j, o + i, WIDE);
                }
            }
        }
    }
    if (!g.params) return;
    float* part = g.part + (size_t)blockIdx.x * 2 * g.dim;
    // A thread's sums, four columns at a time where its columns come in fours (then
    // dim is a multiple of 4), to `to`; the groups of a warp are added first.
    constexpr int Q = VEC >= 4 ? 4 : 1;
    auto put = [&](float* to) {
#pragma unroll
        for (int e = 0; e < E; e += Q) {
            alignas(16) float f[2][Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const int at = SMEM ? 0 : (e + i) / 2;
                float u[2], v[2];
                unpair2(dw[at], u[0], u[1]);
                unpair2(db[at], v[0], v[1]);
                f[0][i] = u[(e + i) & 1];
                f[1][i] = v[(e + i) & 1];
#pragma unroll
                for (int o = G; o < 32; o <<= 1) {
                    f[0][i] += __shfl_xor_sync(0xffffffffu, f[0][i], o);
                    f[1][i] += __shfl_xor_sync(0xffffffffu, f[1][i], o);
                }
            }
            const int j = column(e);
            if (j < g.dim && (G >= 32 || (threadIdx.x & 31) < G)) {
                if (Q == 4) {
                    *reinterpret_cast<float4*>(to + j) = *reinterpret_cast<const float4*>(f[0]);
                    *reinterpret_cast<float4*>(to + g.dim + j) = *reinterpret_cast<const float4*>(f[1]);
                } else {
                    to[j] = f[0][0];
                    to[g.dim + j] = f[1][0];
                }
            }
        }
    };
    if (G == 128) {
        put(part);
        return;
    }
    // the warps of the block, in order
    if (!SMEM) put(sm + (threadIdx.x >> 5) * 2 * g.dim);
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * g.dim; j += NT) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < (SMEM ? 1 : NT / 32); ++w) v += sm[w * 2 * g.dim + j];
        part[j] = v;
    }
}

// Adds the partial rows: 32 columns per block, 16 threads of two along them; group w
// of 64 takes the rows w, w + 64, ... in order, then the groups are added in order.
template <class P>
__global__ void __launch_bounds__(1024) ln_reduce_kernel(const float* part, int parts, int dim, P* dw, P* db) {
    __shared__ float s[64][33];
    const int c = threadIdx.x % 16 * 2, group = threadIdx.x / 16, j0 = blockIdx.x * 32;
    float2 v = make_float2(0.0f, 0.0f);
    if (j0 + c < 2 * dim) {
#pragma unroll 16
        for (int p = group; p < parts; p += 64) {
            const float2 u = __ldg(reinterpret_cast<const float2*>(part + (size_t)p * 2 * dim + j0 + c));
            v.x += u.x;
            v.y += u.y;
        }
    }
    s[group][c] = v.x;
    s[group][c + 1] = v.y;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = j0 + lane;
    const float two = s[2 * warp][lane] + s[2 * warp + 1][lane];
    __syncthreads();
    s[warp][lane] = two;
    __syncthreads();
    if (warp == 0 && j < 2 * dim) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) sum += s[w][lane];
        P* out = j < dim ? dw : db;
        if (out) out[j < dim ? j : j - dim] = from_f32<P>(sum);
    }
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

// Blocks of the backward pass: the SMs filled once, two rows at least to a group and
// four to a block, whose partial row is written and read again.  (1,000 x 1536 f16:
// 9.9 us with two rows a block, 8.0 with four, 10.2 with twelve.)
static int norm_parts(long long rows, int rows_per_block, int per_sm) {
    const long long least = std::max(2 * rows_per_block, 4), want = (rows + least - 1) / least;
    const long long fill = (long long)std::max(1, device_attr(cudaDevAttrMultiProcessorCount)) * per_sm;
    return (int)std::min(fill, std::max(want, 1ll));
}

static size_t norm_ws(long long rows, int dim) {  // for whichever group the type selects: at most six blocks an SM
    return (size_t)norm_parts(rows, 1, 6) * 2 * dim * sizeof(float);
}

template <class T, int VEC, int NCH, int G, bool WIDE>
static int launch_norm(const NormArgs& g, bool backward, int* parts, cudaStream_t st) {
    constexpr int NT = ln_block<G>();
    if (!backward) {
        const long long blocks = (g.rows + NT / G - 1) / (NT / G);
        const long long fill = (long long)std::max(1, device_attr(cudaDevAttrMultiProcessorCount)) *
                               ln_forward_per_sm(G, NCH * VEC, sizeof(T));
        ln_forward_kernel<T, VEC, NCH, G, WIDE><<<(unsigned)std::min(blocks, fill), NT, 0, st>>>(g);
        return check_launch("ln_forward_kernel");
    }
    constexpr int E = NCH * VEC, BT = ln_backward_block(G, E, VEC, sizeof(T));
    const int smem = (G == 128 ? 0 : G == 512 ? 1 : BT / 32) * 2 * g.dim * (int)sizeof(float);
    auto kernel = &ln_backward_kernel<T, VEC, NCH, G, WIDE>;
    if (smem > 40 * 1024) FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), smem));
    *parts = norm_parts(g.rows, BT / G, ln_backward_per_sm(G, E, VEC, sizeof(T)));
    kernel<<<*parts, BT, smem, st>>>(g);
    return check_launch("ln_backward_kernel");
}

// The group and the chunks per thread that hold a row.
template <class T>
static int dispatch_norm(NormArgs g, bool backward, int* parts, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    auto lies = [&](const void* p, long long ld) { return !p || (aligned(p, 16) && ld * sizeof(T) % 16 == 0); };
    const bool vec = g.dim % V == 0;
    const bool wide = lies(g.x, g.ldx) && lies(backward ? g.dy : g.y, g.ldy) && lies(g.dx, g.lddx) && lies(g.w, 0) && lies(g.b, 0);
#define FG_NORM(VEC, NCH, G) \
    if (g.dim <= (VEC) * (NCH) * (G))   \
    return wide && VEC > 1 ? launch_norm<T, VEC, NCH, G, (VEC > 1)>(g, backward, parts, st) \
                           : launch_norm<T, VEC, NCH, G, false>(g, backward, parts, st)
    if constexpr (V == 8) {
        if (vec) {
            FG_NORM(8, 1, 8);
            FG_NORM(8, 2, 8);
            FG_NORM(8, 2, 32);
            FG_NORM(8, 3, 32);
            if (backward) FG_NORM(8, 4, 32);
            FG_NORM(8, 1, 128);
            FG_NORM(8, 2, 128);
            FG_NORM(8, 4, 128);
            FG_NORM(8, 4, 512);
        }
    } else {
        if (vec) {
            FG_NORM(4, 2, 8);
            FG_NORM(4, 4, 8);
            FG_NORM(4, 2, 32);
            FG_NORM(4, 4, 32);
            FG_NORM(4, 2, 128);
            FG_NORM(4, 4, 128);
            FG_NORM(4, 8, 128);
            FG_NORM(4, 8, 512);
        }
    }
    FG_NORM(1, 16, 8);
    FG_NORM(1, 16, 32);
    FG_NORM(1, 8, 128);
    FG_NORM(1, 16, 128);
    FG_NORM(1, 32, 128);
    return launch_norm<T, 1, 32, 512, false>(g, backward, parts, st);
#undef FG_NORM
}

template <class T>
static int norm_forward(const NormArgs& g, cudaStream_t s) {
    return dispatch_norm<T>(g, false, nullptr, s);
}

template <class T>
static int norm_backward(NormArgs g, void* dw, void* db, cudaStream_t s) {
    g.params = dw || db;
    int n = 0;
    if (g.rows && (g.dx || g.params)) {
        const int rc = dispatch_norm<T>(g, true, &n, s);
        if (rc) return rc;
    }
    if (!g.params) return FG_OK;
    const int nb = (2 * g.dim + 31) / 32;
    if (g.w_f32)
        ln_reduce_kernel<float><<<nb, 1024, 0, s>>>(g.part, n, g.dim, (float*)dw, (float*)db);
    else
        ln_reduce_kernel<T><<<nb, 1024, 0, s>>>(g.part, n, g.dim, (T*)dw, (T*)db);
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
        *bytes = norm_ws(rows, dim);
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
        if (dweight || dbias) rc = adapter_ws(workspace, workspace_bytes, norm_ws(rows, dim));
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
