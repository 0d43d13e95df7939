// gated.cu -- gated layer and its gradients.
//
//   [z p] = x w^T + bias (w: the gates' rows, then their partners'),  y = act(z) p
//   dz = dy p act'(z),  dp = dy act(z),  dx = [dz dp] w,  dw = [dz dp]^T x,
//   dbias = sum over rows of [dz dp]
//
// Forward: one product whose tiles hold a gate's columns and its partner's (linear_tc.cu,
// TC_GATED), so that z and p meet in the epilogue and are written only for the backward
// pass.  Backward: one pass over dy, z and p, then the linear layer's two products.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"

namespace fg {

// ---- dz and dp, and their column sums ----------------------------------------------
//
// A group of L lanes takes L x VEC gates of every so many rows and sums its columns in
// registers; the block writes one partial row.  L is 32, or 16 or 8 for layers as narrow as
// that (100,000 x 40 float16 19 us, 64 with whole warps).  A lane's VEC gates lie beside each
// other where the operand's halves start on 16 bytes, else L apart, so that a group's
// accesses of one element are in order (1,777 x 333 bfloat16 6.8 us, 14.1 beside each
// other).  Both factors are products of values of the layer's type, so 16-bit ones enter the
// products in two parts (split2) whatever the activation.  Bound by the latency of its loads
// and by memory: 10,000 x 1024 bfloat16 28 us (143 MB, 5.1 TB/s), float16 30, float32 46 (55
// with two blocks an SM).
constexpr int GD_WARPS = 8;

struct GatedDz {
    const void *dy, *pre;
    void* dz;     // [rows][2 up] of operands, stride pack_stride(2 up); NULL: not stored
    float* part;  // NULL: no sums
    long long lddy, ldp, rows, plane;
    int up, act;
    int in_wide, out_wide;  // all rows and halves start on 16 bytes
};

// act(z) and act'(z) of two columns.
template <int ACT, bool FAST>
__device__ __forceinline__ void act_both(float z, float& a, float& d) {
    if (ACT == FG_ACT_SILU) {
        const float c = z < -100.0f ? -100.0f : z, s = sigmoid<FAST>(c);
        a = c * s;
        d = s * fmaf(fminf(c, 100.0f), 1.0f - s, 1.0f);
        if (z != z) d = z;
    } else if (ACT == FG_ACT_GELU && !FAST) {  // one Phi for both
        const float c = fminf(fmaxf(z, -100.0f), 100.0f), phi = 0.5f * erfcf(z * -0.70710678f);
        a = fmaxf(z, -100.0f) * phi;
        d = fmaf(c, expf(-0.5f * z * z) * 0.39894228f, phi);
    } else {
        a = activate<FAST>(z, ACT);
        d = activate_grad<FAST>(z, ACT);
    }
}
template <int ACT, bool FAST>
__device__ __forceinline__ void act_both2(float z0, float z1, float& a0, float& a1, float& d0, float& d1) {
    if (ACT == FG_ACT_GELU && FAST) {
        a0 = d0 = z0;
        a1 = d1 = z1;
        gelu2(a0, a1);
        gelu_grad2(d0, d1);
    } else {
        act_both<ACT, FAST>(z0, a0, d0);
        act_both<ACT, FAST>(z1, a1, d1);
    }
}

// VEC values of a row: from p on, or `step` apart.
template <class T, int VEC>
__device__ __forceinline__ void gd_load(T (&v)[VEC], const T* p, int left, int wide, int step) {
    if (wide && left >= VEC) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = i * step < left ? p[i * step] : from_f32<T>(0.0f);
    }
}
template <class E, int VEC>
__device__ __forceinline__ void gd_store(E* p, const E (&v)[VEC], int left, int wide, int step) {
    if (wide && left >= VEC) {
        if constexpr (sizeof(E) * VEC == 16)
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
        else
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i * step < left) p[i * step] = v[i];
    }
}

template <class T, int ACT, int L>
__global__ void __launch_bounds__(GD_WARPS * 32, 3) gated_dz_kernel(const GatedDz g) {
    constexpr int VEC = 16 / sizeof(T);
    constexpr bool FAST = sizeof(T) == 2;
    using E = typename std::conditional<FAST, T, __nv_bfloat16>::type;  // of an operand
    constexpr int GROUPS = GD_WARPS * 32 / L;
    __shared__ float s[GROUPS][L * VEC];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const int step = g.out_wide ? 1 : L, j = blockIdx.x * L * VEC + lane * (g.out_wide ? VEC : 1), left = g.up - j;
    const long long ldz = pack_stride(2ll * g.up);
    float sum[2][VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[0][i] = sum[1][i] = 0.0f;
    if (left > 0)
        for (long long r = (long long)blockIdx.y * GROUPS + group; r < g.rows; r += (long long)gridDim.y * GROUPS) {
            alignas(16) T d[VEC], z[VEC], p[VEC];
            const T* pre = static_cast<const T*>(g.pre) + r * g.ldp + j;
            gd_load<T, VEC>(d, static_cast<const T*>(g.dy) + r * g.lddy + j, left, g.in_wide, step);
            gd_load<T, VEC>(z, pre, left, g.in_wide, step);
            gd_load<T, VEC>(p, pre + g.up, left, g.in_wide, step);
            float o[2][VEC];
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                float a0, a1, e0, e1;
                act_both2<ACT, FAST>(to_f32(z[i]), to_f32(z[i + 1]), a0, a1, e0, e1);
                const float d0 = to_f32(d[i]), d1 = to_f32(d[i + 1]);
                o[0][i] = d0 * to_f32(p[i]) * e0;
                o[0][i + 1] = d1 * to_f32(p[i + 1]) * e1;
                o[1][i] = d0 * a0;
                o[1][i + 1] = d1 * a1;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[h][i] += o[h][i];
                if (!g.dz) continue;
                E* out = static_cast<E*>(g.dz) + r * ldz + h * g.up + j;
                if constexpr (FAST) {
                    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
                    alignas(16) T hi[VEC], low[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i += 2)
                        split2(o[h][i], o[h][i + 1], *reinterpret_cast<T2*>(hi + i), *reinterpret_cast<T2*>(low + i));
                    gd_store<T, VEC>(out, hi, left, g.out_wide, step);
                    gd_store<T, VEC>(out + g.plane, low, left, g.out_wide, step);
                } else {
                    alignas(8) __nv_bfloat16 pl[3][VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        __nv_bfloat16 w[3];
                        split3(o[h][i], w);
                        pl[0][i] = w[0];
                        pl[1][i] = w[1];
                        pl[2][i] = w[2];
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) gd_store<__nv_bfloat16, VEC>(out + k * g.plane, pl[k], left, g.out_wide, step);
                }
            }
        }
    if (!g.part) return;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[group][lane * (g.out_wide ? VEC : 1) + i * step] = h ? sum[1][i] : sum[0][i];
        __syncthreads();
        for (int c = threadIdx.x; c < L * VEC; c += GD_WARPS * 32) {
            const int col = blockIdx.x * L * VEC + c;
            if (col >= g.up) break;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < GROUPS; ++w) v += s[w][c];
            g.part[(size_t)blockIdx.y * 2 * g.up + (size_t)h * g.up + col] = v;
        }
    }
}

// Lanes of a group: as few as hold the layer's width.
static int gated_dz_lanes(int up, int elem) {
    const int pieces = (up + 16 / elem - 1) / (16 / elem);
    return pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32;
}

// Row ranges: three blocks to an SM over the column tiles, two rows to a group at least.
static int gated_dz_split(long long rows, int up, int elem) {
    const int lanes = gated_dz_lanes(up, elem), cols = lanes * (16 / elem), least = 2 * GD_WARPS * 32 / lanes, tiles = (up + cols - 1) / cols;
    const long long fill = std::max(1ll, 3ll * std::max(1, device_attr(cudaDevAttrMultiProcessorCount)) / tiles);
    return (int)std::max(1ll, std::min(fill, (rows + least - 1) / least));
}

template <class T, int L>
static void launch_gated_dz_of(const GatedDz& g, int split, cudaStream_t s) {
    constexpr int cols = L * (16 / (int)sizeof(T));
    const dim3 grid((g.up + cols - 1) / cols, split);
    switch (g.act) {
        case FG_ACT_RELU: gated_dz_kernel<T, FG_ACT_RELU, L><<<grid, GD_WARPS * 32, 0, s>>>(g); break;
        case FG_ACT_GELU: gated_dz_kernel<T, FG_ACT_GELU, L><<<grid, GD_WARPS * 32, 0, s>>>(g); break;
        case FG_ACT_SILU: gated_dz_kernel<T, FG_ACT_SILU, L><<<grid, GD_WARPS * 32, 0, s>>>(g); break;
        default: gated_dz_kernel<T, FG_ACT_NONE, L><<<grid, GD_WARPS * 32, 0, s>>>(g);
    }
}

template <class T>
static int launch_gated_dz(GatedDz g, int split, cudaStream_t s) {
    constexpr int VEC = 16 / (int)sizeof(T);
    auto lies = [&](const void* p, long long ld) { return aligned(p, 16) && ld * (int)sizeof(T) % 16 == 0; };
    g.in_wide = lies(g.dy, g.lddy) && lies(g.pre, g.ldp) && g.up % VEC == 0;
    g.out_wide = g.up % VEC == 0;
    switch (gated_dz_lanes(g.up, sizeof(T))) {
        case 8: launch_gated_dz_of<T, 8>(g, split, s); break;
        case 16: launch_gated_dz_of<T, 16>(g, split, s); break;
        default: launch_gated_dz_of<T, 32>(g, split, s);
    }
    return check_launch("gated_dz_kernel");
}

// ---- host side ---------------------------------------------------------------------

constexpr int GATED_IN = 32768, GATED_OUT = 1 << 29;  // the sums' length; tensor coordinates

// `q`: the layer as its products see it, with both halves' columns.
static int gated_check(const fg_linear_params* p, fg_linear_params& q, Strides& t) {
    FG_REQUIRE(p, "null params");
    FG_REQUIRE(p->rows >= 0 && p->in_dim >= 1 && p->out_dim >= 1, "bad layer shape");
    if (p->in_dim > GATED_IN || p->out_dim > GATED_OUT)
        return fail(FG_ERR_UNSUPPORTED, "in_dim above %d or out_dim above %d", GATED_IN, GATED_OUT);
    FG_REQUIRE(p->residual_stride == 0, "a gated layer has no residual");
    q = *p;
    q.out_dim = 2 * p->out_dim;
    q.y_stride = 0;
    const int rc = linear_check(&q, t);
    if (rc) return rc;
    t.y = p->y_stride ? p->y_stride : p->out_dim;
    FG_REQUIRE(t.y >= p->out_dim, "row stride below the row length");
    return FG_OK;
}

// An operand off 16 bytes has room in the workspace where `unaligned` names it.
static int gated_operand_check(const fg_linear_params* p, const void* x, const void* w) {
    if (p->dtype == FG_DTYPE_F32) return FG_OK;
    FG_REQUIRE(aligned(x, 16) || (p->unaligned & FG_LINEAR_X), "x is off 16 bytes and not named in unaligned");
    FG_REQUIRE(aligned(w, 16) || (p->unaligned & FG_LINEAR_W), "w is off 16 bytes and not named in unaligned");
    return FG_OK;
}

struct GatedWs {
    void *x, *w, *dz, *product;
    float* part;
};

static size_t gated_carve(const fg_linear_params& q, const Strides& t, void* ws, size_t bytes, GatedWs& f) {
    Carve c(ws, bytes);
    f = GatedWs{};
    if (q.rows <= GEMV_ROWS) return 0;
    if (needs_pack(q.dtype, t.x, q.unaligned & FG_LINEAR_X)) f.x = c.take<char>(pack_bytes(q.dtype, q.rows, q.in_dim));
    if (needs_pack(q.dtype, t.w, q.unaligned & FG_LINEAR_W)) f.w = c.take<char>(pack_bytes(q.dtype, q.out_dim, q.in_dim));
    return c.used;
}

static int gated_forward(const fg_linear_params& q, const Strides& t, const void* x, const void* w, const Epilogue& e,
                         const GatedWs& f, cudaStream_t s) {
    if (q.rows <= GEMV_ROWS)
        return linear_gemv_gated(q.dtype, x, w, GemmShape{q.rows, q.out_dim, q.in_dim, t.x, 1, t.w, 1}, e, q.out_dim / 2, s);
    PackArgs jobs{};
    const Operand a = operand(q.dtype, x, q.rows, q.in_dim, t.x, q.unaligned & FG_LINEAR_X, f.x, jobs);
    const Operand b = operand(q.dtype, w, q.out_dim, q.in_dim, t.w, q.unaligned & FG_LINEAR_W, f.w, jobs);
    const int rc = linear_pack(q.dtype, jobs, s);
    if (rc) return rc;
    return tc_gated(q.dtype, a.p, a.plane, b.p, b.plane, GemmShape{q.rows, q.out_dim, q.in_dim, a.ld, 1, b.ld, 1}, e, s);
}

// dx = dz w and dw = dz^T x of both halves at once, in as many parts as fill the GPU (dw of
// 10,000 x 768 -> 1024, 24 tiles: three parts 47 us, two 64; float32 140 and 196).
static GemmShape gated_dx(const fg_linear_params& q, long long ldw) {
    return {q.rows, q.in_dim, q.out_dim, pack_stride(q.out_dim), 1, 1, ldw, true};
}
static GemmShape gated_dw(const fg_linear_params& q, long long ldx) {
    return {q.out_dim, q.in_dim, q.rows, 1, pack_stride(q.out_dim), 1, ldx, true};
}

static size_t gated_backward_carve(const fg_linear_params& q, const Strides& t, void* ws, size_t bytes, GatedWs& w) {
    Carve c(ws, bytes);
    w = GatedWs{};
    if (few(&q)) return 0;
    const bool f32 = q.dtype == FG_DTYPE_F32;
    w.dz = c.take<char>(pack_bytes(q.dtype, q.rows, q.out_dim) * (f32 ? 1 : 2));
    if (needs_pack(q.dtype, t.x, q.unaligned & FG_LINEAR_X)) w.x = c.take<char>(pack_bytes(q.dtype, q.rows, q.in_dim));
    if (needs_pack(q.dtype, t.w, q.unaligned & FG_LINEAR_W)) w.w = c.take<char>(pack_bytes(q.dtype, q.out_dim, q.in_dim));
    const int products = tc_products(q.dtype, !f32);
    const size_t n = std::max(tc_gemm_workspace(products, gated_dx(q, t.w)), tc_gemm_workspace(products, gated_dw(q, t.x)));
    if (n) w.product = c.take<char>(n);
    w.part = c.take<float>((size_t)gated_dz_split(q.rows, q.out_dim / 2, dtype_size(q.dtype)) * q.out_dim);
    return c.used;
}

static int gated_backward(const fg_linear_params& q, const Strides& t, const void* dy, const void* x, const void* w,
                          const void* pre, void* dx, void* dw, void* dbias, const GatedWs& ws, cudaStream_t s) {
    const int up = q.out_dim / 2;
    if (few(&q))
        return linear_few_rows(q.dtype, FewArgs{dy, x, w, pre, dx, dw, dbias, t.y, t.x, t.w, t.p, (int)q.rows, q.in_dim, q.out_dim,
                                                q.activation, 0, up}, s);
    const int split = q.rows ? gated_dz_split(q.rows, up, dtype_size(q.dtype)) : 0;
    const long long plane = q.rows * pack_stride(q.out_dim);
    int rc;
    if (split && (dx || dw || dbias)) {
        const GatedDz g{dy, pre, dx || dw ? ws.dz : nullptr, dbias ? ws.part : nullptr, t.y, t.p, q.rows, plane, up, q.activation, 0, 0};
        rc = q.dtype == FG_DTYPE_F32   ? launch_gated_dz<float>(g, split, s)
             : q.dtype == FG_DTYPE_F16 ? launch_gated_dz<__half>(g, split, s)
                                       : launch_gated_dz<__nv_bfloat16>(g, split, s);
        if (rc) return rc;
    }
    if (dbias && (rc = linear_column_sums(q.dtype, ws.part, split, q.out_dim, dbias, s))) return rc;
    const Operand dz{ws.dz, pack_stride(q.out_dim), plane};
    PackArgs jobs{};
    Operand xo{}, wo{};
    if (dx && q.rows) wo = operand(q.dtype, w, q.out_dim, q.in_dim, t.w, q.unaligned & FG_LINEAR_W, ws.w, jobs);
    if (dw && q.rows) xo = operand(q.dtype, x, q.rows, q.in_dim, t.x, q.unaligned & FG_LINEAR_X, ws.x, jobs);
    if ((rc = linear_pack(q.dtype, jobs, s))) return rc;
    Epilogue e{};
    e.ldy = q.in_dim;
    if (dx && q.rows) {
        e.y = dx;
        if ((rc = linear_gemm(q.dtype, dz, wo, gated_dx(q, wo.ld), e, ws.product, s))) return rc;
    }
    if (dw) {
        e.y = dw;
        if ((rc = linear_gemm(q.dtype, dz, xo, gated_dw(q, xo.ld), e, ws.product, s))) return rc;
    }
    return FG_OK;
}

}  // namespace fg

using namespace fg;

extern "C" {

int fg_gated_linear_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        fg_linear_params q;
        Strides t;
        const int rc = gated_check(params, q, t);
        if (rc) return rc;
        GatedWs f;
        *bytes = gated_carve(q, t, nullptr, 0, f);
        return FG_OK;
    });
}

int fg_gated_linear(const fg_linear_params* params, const void* x, const void* w, const void* bias, void* pre, void* y,
                    void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&]() -> int {
        fg_linear_params q;
        Strides t;
        int rc = gated_check(params, q, t);
        if (rc) return rc;
        if (params->rows == 0) return FG_OK;
        FG_REQUIRE(x && w && y, "null buffer");
        if ((rc = gated_operand_check(params, x, w))) return rc;
        GatedWs f;
        if ((rc = adapter_ws(workspace, workspace_bytes, gated_carve(q, t, nullptr, 0, f)))) return rc;
        gated_carve(q, t, workspace, workspace_bytes, f);
        return gated_forward(q, t, x, w, Epilogue{bias, nullptr, pre, y, 0, t.p, t.y, q.activation}, f,
                             static_cast<cudaStream_t>(stream));
    });
}

int fg_gated_linear_backward_workspace_size(const fg_linear_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        fg_linear_params q;
        Strides t;
        const int rc = gated_check(params, q, t);
        if (rc) return rc;
        GatedWs w;
        *bytes = gated_backward_carve(q, t, nullptr, 0, w);
        return FG_OK;
    });
}

int fg_gated_linear_backward(const fg_linear_params* params, const void* dy, const void* x, const void* w, const void* pre,
                             void* dx, void* dw, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&]() -> int {
        fg_linear_params q;
        Strides t;
        int rc = gated_check(params, q, t);
        if (rc) return rc;
        if (params->rows) {
            FG_REQUIRE(dy && pre, "null dy or pre");
            FG_REQUIRE(!dx || w, "dx needs w");
            FG_REQUIRE(!dw || x, "dw needs x");
            if ((rc = gated_operand_check(params, dw ? x : nullptr, dx ? w : nullptr))) return rc;
        }
        GatedWs ws;
        if ((rc = adapter_ws(workspace, workspace_bytes, gated_backward_carve(q, t, nullptr, 0, ws)))) return rc;
        gated_backward_carve(q, t, workspace, workspace_bytes, ws);
        return gated_backward(q, t, dy, x, w, pre, dx, dw, dbias, ws, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
