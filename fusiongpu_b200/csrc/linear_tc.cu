// linear_tc.cu -- the linear layer's products on the 5th-generation tensor cores:
// C(m, n) = sum over k of A(m, k) B(n, k), 16-bit operands, fp32 accumulators in
// TMEM.  float32 operands come as three bf16 planes, x = x0 + x1 + x2 (8 bits of
// the significand each), and the product as the six plane products that reach
// 2^-24 of it: the same kernels with six times the K blocks.  The tensor cores cut
// their sums rather than round them, about 1e-8 of the running value for every 16
// products; so float32 sums are taken from TMEM after at most 512 k, the smallest
// plane products first, and added in fp32, and 16-bit ones run over 32,768 k at most
// before they meet other parts.  A 16-bit dz comes as two planes (split2): the lower one's
// products are summed first, then the upper one's.  Either operand may have unit stride along k (K-major: x and w of the
// forward pass, dz of dx = dz w) or along its rows (MN-major: w of dx, both
// operands of dw = dz^T x), so no pass over memory transposes anything.
//
// The gated layer's product (TC_GATED) is a mode of the same kernels, whose tiles hold gates
// and their partners: 10,000 x 768 -> 1024 bfloat16 31 us, 36 with both pre-activations
// kept.  So is that of rows of 8-bit codes (TC_INT8): 1M x 768 -> 768 float16 661 us, 764 with
// bias and residual (16-bit operands: 1,109); in long runs, at the power cap, 762 and 904
// (1,323).  float32 results 848, and 1,342 with bias and residual.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"
#include "tc_common.cuh"

namespace fg {

constexpr int GT_M = 128;          // UMMA M: rows of a tile, TMEM lanes
constexpr int GT_K = 64;           // elements of a K block: one 128-byte swizzle row
constexpr int GT_NT = 64 + 256;    // TMA warp, MMA warp, 8 epilogue warps
constexpr int GT_RING = 192 * 1024;
constexpr int GT_RUN = 512;        // K blocks that a 16-bit product's accumulator sums at most
constexpr int GP_CHUNK = 8;        // and a float32 one

// What the kernels multiply and what becomes of the sums.
enum {
    TC_WHOLE,  // A and B as they are
    TC_PARTS,  // A in two parts
    TC_GATED,  // B's rows j and up + j together: act(z_j) z_(up + j)
    TC_INT8    // codes of 8 bits, 32-bit integer sums, times the scales of their row and column
};

struct TcArgs {
    int kt, mt, nt;     // K blocks, row tiles, column tiles
    int m, n;
    int a_mn, b_mn;
    int split;          // parts of a tile's K range: CTAs of a cluster, or passes of the pairs
    int m_pad;          // pairs with split > 1: rows of a part's partial tiles
    int vec;            // outputs, residual and bias allow 4-column accesses
    int direct;         // pairs: some of them do not start on 16-byte boundaries, which TMA needs
    int products;       // plane products: 1; 2: A in two parts; 6: float32, both in three
    GemmShape f;        // products > 1: the operands as they lie, for results that are not finite
    const void *fa, *fb;
    long long a_plane, b_plane;
    uint32_t idesc;
    Epilogue e;
    int up;             // TC_GATED: rows of B from a gate's to its partner's
    const float *xs, *ws;  // TC_INT8: scales of A's and B's rows
    int quads;             // ws (and a 32-bit bias) on 16 bytes, n a multiple of 4
};

// Planes of the i-th plane product.
__device__ __forceinline__ int plane_a(int i, int products) {  // 0; 1 0; 0 2 1 0 1 0
    return products == 1 ? 0 : products == 2 ? 1 - i : (280 >> (2 * i)) & 3;
}
__device__ __forceinline__ int plane_b(int i, int products) { return products < 6 ? 0 : (82 >> (2 * i)) & 3; }  // 2 0 1 1 0 0

// An infinite operand times the small planes of the other has any sign, and an f16 part past
// its range is a NaN: a result that is not finite is taken again, one product at a time.
template <class T>
__device__ __noinline__ float retake(const TcArgs& g, int m, int n) {
    using E = typename std::conditional<sizeof(T) == 4, __nv_bfloat16, T>::type;  // of a plane
    float z = 0.0f;
    auto whole = [](const E* p, long long step) { return to_f32(p[0]) + to_f32(p[step]) + to_f32(p[2 * step]); };
    for (long long k = 0; k < g.f.k && z == z; ++k) {
        const E* a = static_cast<const E*>(g.fa) + m * g.f.am + k * g.f.ak;
        const E* b = static_cast<const E*>(g.fb) + n * g.f.bn + k * g.f.bk;
        if constexpr (sizeof(T) == 4)
            z = fmaf(whole(a, g.a_plane), whole(b, g.b_plane), z);
        else
            z = fmaf(of_parts<T>(a[0], a[g.a_plane]), to_f32(b[0]), z);
    }
    return z;
}
template <class T>
__device__ __forceinline__ float finite_or_retake(const TcArgs& g, int m, int n, float z) {
    return !(fabsf(z) <= FLT_MAX) ? retake<T>(g, m, n) : z;
}

template <int BN>
struct RingOf {
    static constexpr int A = GT_M * GT_K * 2, B = BN * GT_K * 2, STAGE = A + B;
    static constexpr int N = GT_RING / STAGE > 8 ? 8 : GT_RING / STAGE;
};

// An integer sum, its bits in a float's place, times its column's and row's scales, and the bias.
__device__ __forceinline__ float dequantised(float sum, float xs, float ws, float bias) {
    return fmaf((float)__float_as_int(sum) * ws, xs, bias);
}

template <class T>
__device__ __forceinline__ float4 load4(const T* p) {
    T v[4];
    *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p);
    return make_float4(to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3]));
}

template <>
__device__ __forceinline__ float4 load4<float>(const float* p) {
    return *reinterpret_cast<const float4*>(p);
}

template <class T>
__device__ __forceinline__ void store4(T* p, float4 f) {
    T v[4] = {from_f32<T>(f.x), from_f32<T>(f.y), from_f32<T>(f.z), from_f32<T>(f.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}

template <>
__device__ __forceinline__ void store4<float>(float* p, float4 f) {
    *reinterpret_cast<float4*>(p) = f;
}

// One tile of 128 x BN per cluster, its K blocks divided over the cluster's
// CTAs.  Each CTA's partial tile goes from TMEM to its shared memory (where the
// operand ring was); then each CTA adds one slice of the columns over the cluster,
// from its own rank onwards -- were all to begin with rank 0, they would queue for its
// shared memory: 100 x 1536 -> 768 bf16 8.2 us, so 7.6 -- and finishes it.
//
// TC_GATED: half of B's rows are gates, the other half their partners, so a tile has BN /
// 2 outputs.  TC_INT8: integer sums, exact in any order.
template <class T, int BN, int MODE>
__global__ void __launch_bounds__(GT_NT, 1)
    gemm_split_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const __grid_constant__ TcArgs g) {
    using Ring = RingOf<BN>;
    constexpr bool PARTS = MODE == TC_PARTS, PLANES = sizeof(T) == 4 && MODE != TC_INT8;
    constexpr int BO = MODE == TC_GATED ? BN / 2 : BN;      // outputs of a tile's row
    constexpr int KB = MODE == TC_INT8 ? 2 * GT_K : GT_K;   // elements of a K block
    constexpr int LDP = BN + 4;  // partial row: 4 floats of padding keep 16-byte stores off each other's banks
    static_assert(GT_M * LDP * 4 <= Ring::N * Ring::STAGE, "the partial tile fits the ring");
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t full[Ring::N], empty[Ring::N], acc_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail, s_lost;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* ring = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~static_cast<uintptr_t>(1023));
    float* part = reinterpret_cast<float*>(ring);
    const int S = g.split, rank = S > 1 ? (int)tc::cluster_rank() : 0;
    const int tile = (int)(blockIdx.x / (unsigned)S);
    const int m0 = tile / g.nt * GT_M, n0 = tile % g.nt * BO;
    const int kb0 = (int)((long long)g.kt * rank / S), kb1 = (int)((long long)g.kt * (rank + 1) / S);
    // accumulators: one, or for float32 as many as TMEM holds, each for GP_CHUNK K blocks
    constexpr int NA = PLANES ? 512 / BN : 1;
    const int share = PLANES ? GP_CHUNK : kb1 - kb0, shares = (kb1 - kb0 + share - 1) / share;
    constexpr int products = PLANES ? 6 : PARTS ? 2 : 1;

    if (warp == 2 && tc::elect_one()) {
        tc::prefetch_map(&ta);
        tc::prefetch_map(&tb);
    }
    if (tid == 0) {
        s_fail = s_lost = 0;
        for (int i = 0; i < Ring::N; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        tc::mbar_init(&acc_full, 1);
        tc::fence_mbar_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&tmem_slot, NA * BN);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t taddr = tmem_slot;
    volatile int* fail = &s_fail;
    int gone = 0;

    if (warp == 0) {
        if (tc::elect_one()) {  // ---- TMA producer
            int i = 0;
            bool ok = true;
            auto load = [&](int kb, int product) {
                const int st = i % Ring::N, k = kb * KB;
                ok = tc::mbar_wait_or_fail(&empty[st], ((i / Ring::N) & 1) ^ 1, fail);
                if (!ok) return;
                unsigned char *sa = ring + st * Ring::STAGE, *sb = sa + Ring::A;
                tc::mbar_arrive_expect_tx(&full[st], Ring::STAGE);
                const int pa = plane_a(product, products), pb = plane_b(product, products);
                if (g.a_mn) {
                    for (int c = 0; c < GT_M / 64; ++c)
                        tc::tma_load_3d(sa + c * 8192, &ta, &full[st], m0 + c * 64, k, pa);
                } else {
                    tc::tma_load_3d(sa, &ta, &full[st], k, m0, pa);
                }
                if (g.b_mn) {
                    for (int c = 0; c < BN / 64; ++c)
                        tc::tma_load_3d(sb + c * 8192, &tb, &full[st], n0 + c * 64, k, pb);
                } else if (MODE == TC_GATED) {
                    tc::tma_load_3d(sb, &tb, &full[st], k, n0, pb);
                    tc::tma_load_3d(sb + BO * 128, &tb, &full[st], k, g.up + n0, pb);
                } else {
                    tc::tma_load_3d(sb, &tb, &full[st], k, n0, pb);
                }
                ++i;
            };
            for (int c0 = kb0; c0 < kb1 && ok; c0 += share)
                for (int q = 0; q < products && ok; ++q)
                    for (int kb = c0; kb < min(c0 + share, kb1) && ok; ++kb) load(kb, q);
            if (!ok)  // copies in flight land before the block ends
                for (int j = i > Ring::N ? i - Ring::N : 0; j < i; ++j)
                    tc::mbar_wait(&full[j % Ring::N], (j / Ring::N) & 1);
        }
    } else if (warp == 1) {
        // ---- MMA issuer: the warp stays together, one elected lane issues
        bool ok = true;
        int i = 0;
        const uint64_t da0 = g.a_mn ? tc::desc_mnmajor_sw128(ring, 8192) : tc::desc_kmajor_sw128(ring);
        const uint64_t db0 = g.b_mn ? tc::desc_mnmajor_sw128(ring + Ring::A, 8192) : tc::desc_kmajor_sw128(ring + Ring::A);
        const uint32_t ka = g.a_mn ? 128 : 2, kbs = g.b_mn ? 128 : 2;  // 16 k, in 16-byte units
        for (int c0 = kb0, acc = 0; c0 < kb1 && ok; c0 += share, ++acc) {
            const int n = (min(c0 + share, kb1) - c0) * products;
            for (int u = 0; u < n; ++u, ++i) {
                const int st = i % Ring::N;
                ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&full[st], (i / Ring::N) & 1, fail));
                if (!ok) break;
                tc::fence_after_sync();
                const uint64_t da = da0 + st * (Ring::STAGE / 16), db = db0 + st * (Ring::STAGE / 16);
                if (tc::elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < GT_K / 16; ++kk) {
                        const uint32_t d = taddr + (uint32_t)(acc * BN);
                        if (std::is_same<T, __half>::value && PARTS && kk == 0 && 2 * u == n)  // on to the upper part
                            tc::umma_shifted<F16_PART_SHIFT>(d, da, db, g.idesc);
                        else if (MODE == TC_INT8)
                            tc::umma_i8(d, da + ka * kk, db + kbs * kk, g.idesc, (u | kk) != 0);
                        else
                            tc::umma_bf16(d, da + ka * kk, db + kbs * kk, g.idesc, (u | kk) != 0);
                    }
                    tc::umma_commit(&empty[st]);
                    if (u + 1 == n && c0 + share >= kb1) tc::umma_commit(&acc_full);
                }
                __syncwarp();
            }
        }
    } else {  // ---- epilogue warps: TMEM -> partial tile in shared memory
        const int q4 = warp & 3, half = (warp - 2) >> 2;
        const bool ok = tc::mbar_wait_warp(&acc_full, 0, fail);
        gone = !ok;
        if (MODE == TC_INT8 && !ok) s_lost = 1;
        tc::fence_after_sync();
        float* row = part + (q4 * 32 + lane) * LDP;
#pragma unroll 1
        for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
            float v[32];
            tc::tmem_ld_32x32(taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)c, v);
            for (int a = 1; a < shares; ++a) {
                float x[32];
                tc::tmem_ld_32x32(taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(a * BN + c), x);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += x[j];
            }
#pragma unroll
            for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(row + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
        tc::fence_before_sync();
    }
    if (__syncthreads_or(gone) && MODE != TC_INT8) {  // a wait that ran out leaves NaN, not a plausible number, once no copy is under way to the ring
        for (int i = tid; i < GT_M * LDP; i += GT_NT) part[i] = NAN;
        __syncthreads();
    }
    if (S > 1) tc::cluster_sync();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(taddr, NA * BN);
    }

    // Four positions per thread and round, their residuals and biases loaded first:
    // one memory latency a round.
    constexpr int U = MODE == TC_GATED ? 2 : 4;
    constexpr bool FAST = sizeof(T) == 2;
    constexpr float scale = PartsOf<T>::hi;
    const int slice = BO / S, per_row = slice / 4;
    const uint32_t pbase = tc::smem_u32(part);
    const Epilogue& e = g.e;
    bool lost = false;  // an integer sum has no NaN: the CTAs say that theirs never came
    if (MODE == TC_INT8)
        for (int s = 0; s < S; ++s) lost |= (S > 1 ? tc::ld_cluster_u32(tc::smem_u32(&s_lost), s) : (uint32_t)s_lost) != 0;
    for (int i0 = tid; i0 < GT_M * per_row; i0 += U * GT_NT) {
        int row[U], col[U];
        uint32_t at[U];
        float4 res[U], bias[U];
        float4 by[U];  // TC_GATED: the partners' bias; TC_INT8: the columns' scales
        float xs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * GT_NT, r = i / per_row, c = rank * slice + (i - r * per_row) * 4;
            row[u] = i < GT_M * per_row ? m0 + r : g.m;
            col[u] = n0 + c;
            at[u] = (uint32_t)(r * LDP + c) * 4;
            res[u] = bias[u] = by[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            xs[u] = 0.0f;
            if (row[u] < g.m && col[u] < g.n) {
                const T* rp = static_cast<const T*>(e.residual) + row[u] * e.ldr + col[u];
                const T* bp = static_cast<const T*>(e.bias) + col[u];
                if (MODE == TC_INT8) xs[u] = g.xs[row[u]];
                if (g.vec && col[u] + 4 <= g.n) {
                    if (e.residual) res[u] = load4(rp);
                    if (e.bias) bias[u] = load4(bp);
                    if (MODE == TC_GATED && e.bias) by[u] = load4(bp + g.up);
                    if (MODE == TC_INT8) by[u] = load4(g.ws + col[u]);
                } else {
                    float* rf = &res[u].x;
                    float* bf = &bias[u].x;
                    float* yf = &by[u].x;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col[u] + j < g.n) {
                            if (e.residual) rf[j] = to_f32(rp[j]);
                            if (e.bias) bf[j] = to_f32(bp[j]);
                            if (MODE == TC_GATED && e.bias) yf[j] = to_f32(bp[g.up + j]);
                            if (MODE == TC_INT8) yf[j] = g.ws[col[u] + j];
                        }
                }
            }
        }
        auto sums = [&](uint32_t a) {
            if (S == 1) return *reinterpret_cast<const float4*>(reinterpret_cast<const char*>(part) + a);
            float4 z = tc::ld_cluster_f4(pbase + a, rank);
            for (int s = 1; s < S; ++s) {
                const float4 v = tc::ld_cluster_f4(pbase + a, (rank + s) & (S - 1));
                if (MODE == TC_INT8) {
                    z = make_float4(__int_as_float(__float_as_int(z.x) + __float_as_int(v.x)),
                                    __int_as_float(__float_as_int(z.y) + __float_as_int(v.y)),
                                    __int_as_float(__float_as_int(z.z) + __float_as_int(v.z)),
                                    __int_as_float(__float_as_int(z.w) + __float_as_int(v.w)));
                } else {
                    z.x += v.x;
                    z.y += v.y;
                    z.z += v.z;
                    z.w += v.w;
                }
            }
            return z;
        };
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row[u] >= g.m || col[u] >= g.n) continue;
            float4 z = sums(at[u]);
            const bool whole = col[u] + 4 <= g.n;
            if (PARTS) z = make_float4(z.x * scale, z.y * scale, z.z * scale, z.w * scale);
            if (MODE == TC_INT8) {
                z = make_float4(dequantised(z.x, xs[u], by[u].x, bias[u].x), dequantised(z.y, xs[u], by[u].y, bias[u].y),
                                dequantised(z.z, xs[u], by[u].z, bias[u].z), dequantised(z.w, xs[u], by[u].w, bias[u].w));
                if (lost) z = make_float4(NAN, NAN, NAN, NAN);
            }
            auto retaken = [&](float4& z, int c) {
                z.x = finite_or_retake<T>(g, row[u], c, z.x);
                if (col[u] + 1 < g.n) z.y = finite_or_retake<T>(g, row[u], c + 1, z.y);
                if (col[u] + 2 < g.n) z.z = finite_or_retake<T>(g, row[u], c + 2, z.z);
                if (col[u] + 3 < g.n) z.w = finite_or_retake<T>(g, row[u], c + 3, z.w);
            };
            if (products > 1) retaken(z, col[u]);
            if (MODE != TC_INT8) {
                z.x += bias[u].x;
                z.y += bias[u].y;
                z.z += bias[u].z;
                z.w += bias[u].w;
            }
            auto put = [&](void* out, long long at, const float4& v) {
                T* p = static_cast<T*>(out) + at;
                if (g.vec && whole) {
                    store4(p, v);
                } else {
                    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col[u] + j < g.n) p[j] = from_f32<T>(f[j]);
                }
            };
            if (e.pre) put(e.pre, row[u] * e.ldp + col[u], z);
            float4 y = z;
            if (e.act == FG_ACT_GELU && FAST) {
                gelu2(y.x, y.y);
                gelu2(y.z, y.w);
            } else if (e.act != FG_ACT_NONE) {
                y = make_float4(activate<FAST>(z.x, e.act), activate<FAST>(z.y, e.act), activate<FAST>(z.z, e.act),
                                activate<FAST>(z.w, e.act));
            }
            if (MODE == TC_GATED) {
                float4 p = sums(at[u] + BO * 4);
                if (products > 1) retaken(p, g.up + col[u]);
                p.x += by[u].x;
                p.y += by[u].y;
                p.z += by[u].z;
                p.w += by[u].w;
                if (e.pre) put(e.pre, row[u] * e.ldp + g.up + col[u], p);
                y = make_float4(y.x * p.x, y.y * p.y, y.z * p.z, y.w * p.w);
            }
            y.x += res[u].x;
            y.y += res[u].y;
            y.z += res[u].z;
            y.w += res[u].w;
            put(e.y, row[u] * e.ldy + col[u], y);
        }
    }
    if (S > 1) tc::cluster_sync();  // a peer may still read this CTA's partial tile
}

// ---- many tiles: persistent CTA pairs -----------------------------------------------
//
// A cluster of two CTAs takes 256 x BN tiles in turn; each MMA (cta_group::2)
// spans both: a CTA holds 128 rows of A, half of B and the accumulators of its
// 128 rows, so a K block brings 32 KB into each CTA instead of the 48 KB that a
// 128 x 256 tile of its own would need.  TMEM holds two accumulators, and the
// epilogue of a tile runs while the next one is multiplied: a warp takes its 32
// rows x 64 columns through a 4 KB buffer that TMA fills with the residual and
// stores from (whole 128-byte rows, clipped at the matrix's edge).  16 epilogue
// warps hide the chain TMEM load, residual, fence, store of each: 8 warps of two
// chunks took 10,200 cycles for a tile of 6,144 cycles of products (width 768).
constexpr int GP_A = GT_M * GT_K * 2;
constexpr int GP_BUF = 4096;   // 32 rows x 128 bytes, 128-byte swizzle
constexpr int GP_EPI = 16;     // epilogue warps, each 32 rows x 64 columns of a tile
constexpr int GP_NT = 64 + GP_EPI * 32;

// Operand stages and the epilogue's buffers: 4 KB a warp, or for float32 8 KB, which
// hold the running sums of its 32 rows x 64 columns.
template <class T, int BN, int MODE>
struct PairOf {
    static constexpr int B = BN / 2 * GT_K * 2, STAGE = GP_A + B;
    static constexpr bool TWO = sizeof(T) == 4 || MODE == TC_INT8;  // buffers a warp
    static constexpr bool GATED = sizeof(T) == 2 && MODE == TC_GATED;  // room for both pre-activations and the result
    static constexpr int STAGES = TWO ? 3 : GATED ? 4 : 5;
    static constexpr int BUF = TWO ? 2 * GP_BUF : GATED ? GP_BUF * 3 / 2 : GP_BUF;
    static constexpr int SMEM = STAGES * STAGE + GP_EPI * (BUF + (sizeof(T) == 4 ? 0 : 128));
    static constexpr int WARPS = BN / 64 * 4;         // epilogue warps of a tile
    static constexpr int GROUPS = GP_EPI / WARPS;     // that take tiles in turn
};

template <class T>
__device__ __forceinline__ uint4 pack8(const float* v) {
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

template <class T>
__device__ __forceinline__ void add8(float* v, uint4 u) {
    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2<T>(x[k]);
        unpair2(add2(pair2(v[2 * k], v[2 * k + 1]), pair2(f.x, f.y)), v[2 * k], v[2 * k + 1]);
    }
}

template <int ACT, bool FAST = true>
__device__ __forceinline__ void activate_all(float (&v)[2][32]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            if (ACT == FG_ACT_GELU && FAST) {
                gelu2(v[h][j], v[h][j + 1]);
            } else {
                v[h][j] = activate<FAST>(v[h][j], ACT);
                v[h][j + 1] = activate<FAST>(v[h][j + 1], ACT);
            }
        }
}

// v[0] = act(v[0]) v[1]
template <int ACT>
__device__ __forceinline__ void gate_all(float (&v)[2][32]) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        if (ACT == FG_ACT_GELU) {
            gelu2(v[0][j], v[0][j + 1]);
        } else if (ACT != FG_ACT_NONE) {
            v[0][j] = activate<true>(v[0][j], ACT);
            v[0][j + 1] = activate<true>(v[0][j + 1], ACT);
        }
        unpair2(mul2(pair2(v[0][j], v[0][j + 1]), pair2(v[1][j], v[1][j + 1])), v[0][j], v[0][j + 1]);
    }
}

// Columns 2 lane and 2 lane + 1 of a 64-column piece of the bias, packed; fetched
// before the accumulator is waited for (the operand ring leaves no L1 to find it in).
template <class T>
__device__ __forceinline__ uint32_t fetch_bias(const T* b, int lane, int left, int direct) {
    if (2 * lane + 2 <= left && !direct) return __ldg(reinterpret_cast<const unsigned*>(b) + lane);
    const unsigned short* p = reinterpret_cast<const unsigned short*>(b) + 2 * lane;
    uint32_t u = 0;
    if (2 * lane < left) u = p[0];
    if (2 * lane + 1 < left) u |= (uint32_t)p[1] << 16;
    return u;
}

// A warp's 32 rows of 128 bytes between its swizzled buffer and a matrix whose rows
// start anywhere: row by row, neighbouring lanes on neighbouring columns, R rows
// under way at once.
template <class T, bool OUT, int R>
__device__ __forceinline__ void copy_rows(unsigned char* buf, T* matrix, long long ld, int row0, int col0, int rows, int cols,
                                          int lane) {
    constexpr int PER = 128 / 32 / (int)sizeof(T);  // columns a lane
    __syncwarp();
#pragma unroll 1
    for (int r0 = 0; r0 < 32 && row0 + r0 < rows; r0 += R) {
        T v[R][PER];
#pragma unroll
        for (int k = 0; k < 2; ++k)  // read, then write
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int c = lane + 32 * i, at = r0 + r;
                    T* p = matrix + (row0 + at) * ld + col0 + c;
                    T* q = reinterpret_cast<T*>(buf + at * 128 + ((c * (int)sizeof(T)) ^ ((at & 7) << 4)));
                    if (col0 + c < cols && row0 + at < rows) {
                        if (k == 0)
                            v[r][i] = OUT ? *q : *p;
                        else
                            *(OUT ? p : q) = v[r][i];
                    }
                }
    }
    __syncwarp();
}

// A warp's 32 rows of 64 bytes from its buffer (64-byte swizzle) to a matrix whose rows start
// anywhere, as copy_rows does.
template <class T>
__device__ __forceinline__ void store_half(const unsigned char* buf, T* matrix, long long ld, int row0, int col0, int rows, int cols, int lane) {
    __syncwarp();
    if (col0 + lane < cols) {
        T* p = matrix + row0 * ld + col0 + lane;
#pragma unroll 8
        for (int r = 0; r < 32; ++r)
            if (row0 + r < rows) p[r * ld] = *reinterpret_cast<const T*>(buf + r * 64 + ((lane * 2) ^ ((r >> 1 & 3) << 4)));
    }
    __syncwarp();
}

template <class T>
__device__ __forceinline__ void add_bias(float (&v)[2][32], const unsigned char* b) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; j += 8) add8<T>(&v[h][j], *reinterpret_cast<const uint4*>(b + (32 * h + j) * 2));
}

// Integer sums of 64 columns, times their scales and the row's, and the bias.  Columns past
// the last take the last one's scale; they are not stored.  QUADS: scales (and a bias of 32
// bits, which lies in global memory) on 16 bytes, their number a multiple of 4.
template <class T, bool QUADS>
__device__ __forceinline__ void dequantise_all(float (&v)[2][32], const float* ws, int col, int n, float xs, const unsigned char* bias) {
    const uint64_t x = pair2(xs, xs);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
            const int c = col + 32 * h + j;
            float s[8], b[8];
            if (QUADS) {
                *reinterpret_cast<float4*>(s) = __ldg(reinterpret_cast<const float4*>(ws + min(c, n - 4)));
                *reinterpret_cast<float4*>(s + 4) = __ldg(reinterpret_cast<const float4*>(ws + min(c + 4, n - 4)));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] = __ldg(ws + min(c + i, n - 1));
            }
            if (bias && sizeof(T) == 4) {
                const float* f = reinterpret_cast<const float*>(bias);
                if (QUADS) {
                    *reinterpret_cast<float4*>(b) = __ldg(reinterpret_cast<const float4*>(f + min(c, n - 4)));
                    *reinterpret_cast<float4*>(b + 4) = __ldg(reinterpret_cast<const float4*>(f + min(c + 4, n - 4)));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[i] = __ldg(f + min(c + i, n - 1));
                }
            } else if (bias) {
                const uint4 u = *reinterpret_cast<const uint4*>(bias + (32 * h + j) * 2);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack2<typename std::conditional<sizeof(T) == 4, __half, T>::type>(w[i]);
                    b[2 * i] = f.x;
                    b[2 * i + 1] = f.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float &p = v[h][j + i], &q = v[h][j + i + 1];
                const uint64_t sum = pair2((float)__float_as_int(p), (float)__float_as_int(q));
                unpair2(fma2(mul2(sum, pair2(s[i], s[i + 1])), x, pair2(b[i], b[i + 1])), p, q);
            }
        }
}

// Waits for a copy into a buffer of this warp.  When another role has failed the first
// wait ends early, and the copy, which may still land, is waited for by itself.
__device__ __forceinline__ bool copy_landed(uint64_t* bar, uint32_t parity, volatile int* fail) {
    return tc::mbar_wait_warp(bar, parity, fail) || __all_sync(0xffffffffu, tc::mbar_wait(bar, parity));
}

// NaN in `cols` columns of a warp's 32 rows, past a buffer that a copy may yet land in.
template <class T>
__device__ __noinline__ void store_nan(void* matrix, long long ld, int row0, int col0, int rows, int last, int cols) {
    const int row = row0 + (int)(threadIdx.x & 31);
    if (!matrix || row >= rows) return;
    for (int c = col0; c < min(col0 + cols, last); ++c) static_cast<T*>(matrix)[row * ld + c] = from_f32<T>(NAN);
}

// DIRECT: outputs, residual or bias do not start on 16-byte boundaries, which TMA
// needs: they pass row by row between memory and the buffer.
//
// TC_GATED: the leader holds 128 gates' rows of B and its peer their partners', so that
// an accumulator's halves are the two factors of 128 outputs; a warp takes 32 of each.
// 16-bit results leave in rows of 64 bytes (64-byte swizzle); both pre-activations and the
// result have 2 KB each of a warp's buffer, so that none waits for another's store.
template <class T, int BN, bool DIRECT, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GP_NT, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap ty, const __grid_constant__ CUtensorMap tp,
                     const __grid_constant__ CUtensorMap tr, const __grid_constant__ TcArgs g) {
    using P = PairOf<T, BN, MODE>;
    constexpr int GP_STAGES = P::STAGES;
    constexpr bool PARTS = MODE == TC_PARTS, PLANES = sizeof(T) == 4 && MODE != TC_INT8;
    constexpr int BO = MODE == TC_GATED ? BN / 2 : BN, PC = MODE == TC_GATED ? 32 : 64;  // outputs of a tile's row, a warp's
    constexpr int KB = MODE == TC_INT8 ? 2 * GT_K : GT_K;
    static_assert(sizeof(T) == 2 || BN == 256, "float32 takes 256 columns");
    static_assert(MODE != TC_GATED || BN == 256, "gated tiles have 128 columns");
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t full[GP_STAGES], empty[GP_STAGES], acc_full[2], acc_empty[2], res_full[MODE == TC_INT8 ? 2 * GP_EPI : GP_EPI];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail, s_odd;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)tc::cluster_rank();
    unsigned char *ring = dsmem, *bufs = ring + GP_STAGES * P::STAGE, *biases = bufs + GP_EPI * P::BUF;
    const int pairs = (int)(gridDim.x >> 1), items = g.mt * g.nt * g.split;
    auto k_begin = [&](int part) { return (int)((long long)g.kt * part / g.split); };
    constexpr int chunk = PLANES ? GP_CHUNK : 1 << 30;
    constexpr int products = PLANES ? 6 : PARTS ? 2 : 1;
    constexpr float scale = PartsOf<T>::hi;

    if (warp == 2 && tc::elect_one()) {
        tc::prefetch_map(&ta);
        tc::prefetch_map(&tb);
        if (!DIRECT) {
            tc::prefetch_map(&ty);
            if (g.e.pre) tc::prefetch_map(&tp);
            if (MODE == TC_GATED ? g.e.pre != nullptr : g.e.residual != nullptr) tc::prefetch_map(&tr);
        }
    }
    if (tid == 0) {
        s_fail = s_odd = 0;
        for (int i = 0; i < GP_STAGES; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&acc_full[i], 1);
            tc::mbar_init(&acc_empty[i], 2 * P::WARPS);
        }
        for (int w = 0; w < (MODE == TC_INT8 ? 2 * GP_EPI : GP_EPI); ++w) tc::mbar_init(&res_full[w], 1);
        tc::fence_mbar_init();
    }
    if (tid == 0 && (tc::smem_u32(dsmem) & 1023)) s_fail = 1;  // swizzled tiles start on 1,024 bytes
    if (warp == 1) tc::tmem_alloc_pair(&tmem_slot, 2 * BN);
    tc::fence_before_sync();
    __syncthreads();
    tc::cluster_sync();  // the peer's barriers are ready too
    tc::fence_after_sync();
    const uint32_t taddr = tmem_slot;
    volatile int* fail = &s_fail;

    if (warp == 0) {
        if (tc::elect_one()) {  // ---- TMA producer (each CTA its own halves)
            int i = 0;
            bool ok = true;
            for (int w = blockIdx.x >> 1; w < items && ok; w += pairs) {
                const int t = w / g.split, sp = w - t * g.split, k1 = k_begin(sp + 1);
                const int m0 = t / g.nt * 2 * GT_M + rank * GT_M;
                const int n0 = t % g.nt * BO + rank * (MODE == TC_GATED ? g.up : BN / 2);
                auto load = [&](int kb, int product) {
                    const int st = i % GP_STAGES, k = kb * KB;
                    ok = tc::mbar_wait_or_fail(&empty[st], ((i / GP_STAGES) & 1) ^ 1, fail);
                    if (!ok) return;
                    unsigned char *sa = ring + st * P::STAGE, *sb = sa + GP_A;
                    if (rank == 0) tc::mbar_arrive_expect_tx(&full[st], 2 * P::STAGE);
                    const uint32_t bar = tc::leader_addr(&full[st]);
                    const int pa = plane_a(product, products), pb = plane_b(product, products);
                    if (g.a_mn) {
                        for (int c = 0; c < GT_M / 64; ++c)
                            tc::tma_load_3d_pair(sa + c * 8192, &ta, bar, m0 + c * 64, k, pa);
                    } else {
                        tc::tma_load_3d_pair(sa, &ta, bar, k, m0, pa);
                    }
                    if (g.b_mn) {
                        for (int c = 0; c < BN / 128; ++c)
                            tc::tma_load_3d_pair(sb + c * 8192, &tb, bar, n0 + c * 64, k, pb);
                    } else {
                        tc::tma_load_3d_pair(sb, &tb, bar, k, n0, pb);
                    }
                    ++i;
                };
                for (int c0 = k_begin(sp); c0 < k1 && ok; c0 += min(chunk, k1 - c0))
                    for (int q = 0; q < products && ok; ++q)
                        for (int kb = c0; kb < c0 + min(chunk, k1 - c0) && ok; ++kb) load(kb, q);
            }
            if (!ok && rank == 0)  // copies in flight land before the blocks end
                for (int j = i > GP_STAGES ? i - GP_STAGES : 0; j < i; ++j)
                    tc::mbar_wait(&full[j % GP_STAGES], (j / GP_STAGES) & 1);
        }
    } else if (warp == 1) {
        if (rank == 0) {  // ---- MMA issuer of the pair: the warp stays together, one elected lane issues
            int i = 0, li = 0;
            bool ok = true;
            const uint64_t da0 = g.a_mn ? tc::desc_mnmajor_sw128(ring, 8192) : tc::desc_kmajor_sw128(ring);
            const uint64_t db0 = g.b_mn ? tc::desc_mnmajor_sw128(ring + GP_A, 8192) : tc::desc_kmajor_sw128(ring + GP_A);
            const uint32_t ka = g.a_mn ? 128 : 2, kbs = g.b_mn ? 128 : 2;
            for (int w = blockIdx.x >> 1; w < items && ok; w += pairs) {
                const int sp = w % g.split, k1 = k_begin(sp + 1);
                for (int c0 = k_begin(sp); c0 < k1 && ok; c0 += min(chunk, k1 - c0), ++li) {
                    const int n = min(chunk, k1 - c0) * products, acc = li & 1;
                    ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&acc_empty[acc], ((li >> 1) & 1) ^ 1, fail));
                    if (!ok) break;
                    tc::fence_after_sync();
                    for (int u = 0; u < n; ++u, ++i) {
                        const int st = i % GP_STAGES;
                        ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&full[st], (i / GP_STAGES) & 1, fail));
                        if (!ok) break;
                        tc::fence_after_sync();
                        const uint64_t da = da0 + st * (P::STAGE / 16), db = db0 + st * (P::STAGE / 16);
                        if (tc::elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < GT_K / 16; ++kk) {
                                const uint32_t d = taddr + (uint32_t)(acc * BN);
                                if (std::is_same<T, __half>::value && PARTS && kk == 0 && 2 * u == n)
                                    tc::umma_pair_shifted<F16_PART_SHIFT>(d, da, db, g.idesc);  // on to the upper part
                                else if (MODE == TC_INT8)
                                    tc::umma_pair_i8(d, da + ka * kk, db + kbs * kk, g.idesc, (u | kk) != 0);
                                else
                                    tc::umma_pair(d, da + ka * kk, db + kbs * kk, g.idesc, (u | kk) != 0);
                            }
                            tc::umma_commit_pair(&empty[st]);
                            if (u + 1 == n) tc::umma_commit_pair(&acc_full[acc]);
                        }
                        __syncwarp();
                    }
                }
            }
        }
    } else {  // ---- epilogue warps
        const int w = warp - 2, q4 = warp & 3, part = w / 4 % (BN / 64), group = w / P::WARPS;
        unsigned char* buf = bufs + w * P::BUF;
        const Epilogue& e = g.e;
        const int tr_rows = rank * GT_M + q4 * 32;
        const uint32_t sw = (uint32_t)(lane & 7) << 4;
        unsigned char* brow = buf + lane * 128;
        uint32_t res_phase = 0;
        auto fetch_residual = [&](int t) {  // lane 0, once the buffer is free
            tc::mbar_arrive_expect_tx(&res_full[w], GP_BUF);
            tc::tma_load_2d(buf, &tr, &res_full[w], t % g.nt * BN + part * 64, t / g.nt * 2 * GT_M + tr_rows);
        };
        const int step = pairs * P::GROUPS;
        int item = (blockIdx.x >> 1) + pairs * group, li = group;
        bool lost = false;      // a residual never came: this warp's results are NaN from there on
        bool odd_seen = false;  // a result that is not finite, stored as NaN and taken again at the end
        const bool ahead = sizeof(T) == 2 && MODE != TC_INT8 && e.residual && !e.pre;  // residuals a tile ahead (DIRECT: during its products)
        if (!DIRECT && ahead && item < items && tc::elect_one()) fetch_residual(item);
        if constexpr (MODE == TC_INT8 && sizeof(T) == 4) {
            // Bound by the results' bytes; both halves of 32 columns have a buffer, which the residual
            // fills during the products.
            float* residual = const_cast<float*>(static_cast<const float*>(e.residual));
            for (int i = 0; item < items; item += step, li += P::GROUPS, ++i) {
                const int acc = li & 1, col = item % g.nt * BN + part * 64, m0 = item / g.nt * 2 * GT_M + tr_rows;
                if (lost) {
                    store_nan<T>(e.y, e.ldy, m0, col, g.m, g.n, 64);
                    continue;
                }
                if (!DIRECT) {
                    if (tc::elect_one()) {
                        if (e.residual) {
                            tc::bulk_wait_read<0>();
                            tc::mbar_arrive_expect_tx(&res_full[w], 2 * GP_BUF);
                            for (int h = 0; h < 2; ++h) tc::tma_load_2d(buf + h * GP_BUF, &tr, &res_full[w], col + 32 * h, m0);
                        }
                    }
                    __syncwarp();
                } else if (e.residual) {
                    for (int h = 0; h < 2; ++h)
                        copy_rows<T, false, 8>(buf + h * GP_BUF, residual, e.ldr, m0, col + 32 * h, g.m, g.n, lane);
                }
                const float xs = m0 + lane < g.m ? __ldg(g.xs + m0 + lane) : 0.0f;
                const bool ok = tc::mbar_wait_warp(&acc_full[acc], (li >> 1) & 1, fail);
                tc::fence_after_sync();
                const uint32_t src = taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * BN + part * 64);
                float v[2][32];
                tc::tmem_ld_32x32_nowait(src, v[0]);
                tc::tmem_ld_32x32_nowait(src + 32, v[1]);
                tc::tmem_ld_wait(v[0]);
                tc::tmem_ld_wait(v[1]);
                tc::fence_before_sync();
                __syncwarp();
                if (tc::elect_one()) tc::mbar_arrive_leader(tc::leader_addr(&acc_empty[acc]));
                if (g.quads)
                    dequantise_all<T, true>(v, g.ws, col, g.n, xs, static_cast<const unsigned char*>(e.bias));
                else
                    dequantise_all<T, false>(v, g.ws, col, g.n, xs, static_cast<const unsigned char*>(e.bias));
                if (!ok) {  // a wait that ran out leaves NaN, not a plausible number
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[0][j] = v[1][j] = NAN;
                }
                switch (e.act) {
                    case FG_ACT_RELU: activate_all<FG_ACT_RELU, false>(v); break;
                    case FG_ACT_GELU: activate_all<FG_ACT_GELU, false>(v); break;
                    case FG_ACT_SILU: activate_all<FG_ACT_SILU, false>(v); break;
                }
                if (e.residual && !DIRECT) {
                    lost = !copy_landed(&res_full[w], i & 1, fail);
                    if (lost) {
                        store_nan<T>(e.y, e.ldy, m0, col, g.m, g.n, 64);
                        continue;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned char* hrow = brow + h * GP_BUF;
                    if (e.residual) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 r = *reinterpret_cast<const float4*>(hrow + (((uint32_t)j << 2) ^ sw));
                            v[h][j] += r.x;
                            v[h][j + 1] += r.y;
                            v[h][j + 2] += r.z;
                            v[h][j + 3] += r.w;
                        }
                    } else if (!DIRECT) {  // this half's results of the last tile have left it
                        if (tc::elect_one()) tc::bulk_wait_read<1>();
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4*>(hrow + (((uint32_t)j << 2) ^ sw)) = make_float4(v[h][j], v[h][j + 1], v[h][j + 2], v[h][j + 3]);
                    if (DIRECT) {
                        copy_rows<T, true, 1>(buf + h * GP_BUF, static_cast<T*>(e.y), e.ldy, m0, col + 32 * h, g.m, g.n, lane);
                        continue;
                    }
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (tc::elect_one()) {
                        if (m0 < g.m && col + 32 * h < g.n) tc::tma_store_2d(&ty, buf + h * GP_BUF, col + 32 * h, m0);
                        tc::bulk_commit();
                    }
                }
            }
        } else if constexpr (sizeof(T) == 4) {
            // Chunks of k are added to the sums in shared memory, a lane its own row, in
            // two halves of 32 columns; the last one is followed by the epilogue proper,
            // one step after the other: six products a K block hide it.
            for (; item < items; item += step) {
                const int t = item / g.split, sp = item - t * g.split, k1 = k_begin(sp + 1);
                const int col = t % g.nt * BO + part * PC, m0 = t / g.nt * 2 * GT_M + tr_rows;
                bool all_ok = true;
                if (tc::elect_one()) tc::bulk_wait_read<0>();
                __syncwarp();
                for (int c0 = k_begin(sp), first = 1; c0 < k1; c0 += min(chunk, k1 - c0), first = 0, ++li) {
                    const int acc = li & 1;
                    all_ok &= tc::mbar_wait_warp(&acc_full[acc], (li >> 1) & 1, fail);
                    tc::fence_after_sync();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[32];
                        tc::tmem_ld_32x32(taddr + ((uint32_t)(q4 * 32) << 16) +
                                              (uint32_t)(acc * BN + part * PC + (MODE == TC_GATED ? BO : 32) * h), v);
                        if (h == 1) {
                            tc::fence_before_sync();
                            __syncwarp();
                            if (tc::elect_one()) tc::mbar_arrive_leader(tc::leader_addr(&acc_empty[acc]));
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4* s = reinterpret_cast<float4*>(brow + h * GP_BUF + (((uint32_t)j << 2) ^ sw));
                            float4 x = first ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *s;
                            x.x += v[j];
                            x.y += v[j + 1];
                            x.z += v[j + 2];
                            x.w += v[j + 3];
                            *s = x;
                        }
                    }
                }
                if constexpr (MODE == TC_GATED) {
                    const bool in = m0 < g.m && col < g.n;
                    auto put = [&](const CUtensorMap* map, const void* from, bool last) {
                        tc::fence_proxy_async();
                        __syncwarp();
                        if (tc::elect_one()) {
                            if (in) tc::tma_store_2d(map, from, col, m0);
                            if (last) tc::bulk_commit();
                        }
                    };
                    // z and its partner: sums, marked where they are not finite, and the bias
                    bool odd = false;
#pragma unroll 2
                    for (int q = 0; q < 16; ++q) {
                        const int j = q % 8 * 4, c0 = q < 8 ? col : g.up + col;
                        float4* at = reinterpret_cast<float4*>(brow + q / 8 * GP_BUF + (((uint32_t)j << 2) ^ sw));
                        const float4 x = *at;
                        float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool finite = fabsf(v[i]) <= FLT_MAX;
                            odd |= !finite;
                            if (!finite || !all_ok) v[i] = NAN;  // a wait that ran out leaves NaN, too
                            if (e.bias && col + j + i < g.n) v[i] += __ldg(static_cast<const float*>(e.bias) + c0 + j + i);
                        }
                        *at = make_float4(v[0], v[1], v[2], v[3]);
                    }
                    odd_seen |= __any_sync(0xffffffffu, odd && all_ok);
                    if (e.pre && DIRECT) {
                        copy_rows<T, true, 1>(buf, static_cast<T*>(e.pre), e.ldp, m0, col, g.m, g.n, lane);
                        copy_rows<T, true, 1>(buf + GP_BUF, static_cast<T*>(e.pre) + g.up, e.ldp, m0, col, g.m, g.n, lane);
                    } else if (e.pre) {
                        put(&tp, buf, false);
                        put(&tr, buf + GP_BUF, true);
                        if (tc::elect_one()) tc::bulk_wait_read<0>();
                        __syncwarp();
                    }
#pragma unroll 1
                    for (int j = 0; j < 32; j += 4) {
                        float4* at = reinterpret_cast<float4*>(brow + (((uint32_t)j << 2) ^ sw));
                        const float4 z = *at, p = *reinterpret_cast<const float4*>(brow + GP_BUF + (((uint32_t)j << 2) ^ sw));
                        *at = make_float4(activate<false>(z.x, e.act) * p.x, activate<false>(z.y, e.act) * p.y,
                                          activate<false>(z.z, e.act) * p.z, activate<false>(z.w, e.act) * p.w);
                    }
                    if (DIRECT)
                        copy_rows<T, true, 1>(buf, static_cast<T*>(e.y), e.ldy, m0, col, g.m, g.n, lane);
                    else
                        put(&ty, buf, true);
                }
#pragma unroll 1
                for (int h = MODE == TC_GATED ? 2 : 0; h < 2; ++h) {
                    const int c0 = col + 32 * h;
                    const bool in = m0 < g.m && c0 < g.n;
                    if (lost) {
                        store_nan<T>(e.pre, e.ldp, m0, c0, g.m, g.n, 32);
                        store_nan<T>(e.y, e.ldy, m0, c0, g.m, g.n, 32);
                        continue;
                    }
                    unsigned char *hbuf = buf + h * GP_BUF, *hrow = brow + h * GP_BUF;
                    auto put = [&](const CUtensorMap* map, int y0, bool store) {
                        tc::fence_proxy_async();
                        __syncwarp();
                        if (tc::elect_one()) {
                            if (store) tc::tma_store_2d(map, hbuf, c0, y0);
                            tc::bulk_commit();
                        }
                    };
                    if (!all_ok) {  // a wait that ran out leaves NaN, not a plausible number
                        for (int j = 0; j < 32; ++j) reinterpret_cast<float*>(hrow)[j] = NAN;
                    }
                    if (g.split > 1) {  // this part's sums as they are; finish_kernel adds the parts
                        put(&ty, sp * g.m_pad + m0, c0 < g.n);
                        continue;
                    }
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(hrow + (((uint32_t)j << 2) ^ sw));
                        v[j] = x.x;
                        v[j + 1] = x.y;
                        v[j + 2] = x.z;
                        v[j + 3] = x.w;
                    }
                    auto stage = [&] {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4*>(hrow + (((uint32_t)j << 2) ^ sw)) =
                                make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    };
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < 32; ++j) odd |= !(fabsf(v[j]) <= FLT_MAX);
                    if (__any_sync(0xffffffffu, odd && all_ok)) {
                        odd_seen = true;
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = fabsf(v[j]) <= FLT_MAX ? v[j] : NAN;
                    }
                    if (e.bias) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c0 + j < g.n) v[j] += __ldg(static_cast<const float*>(e.bias) + c0 + j);
                    }
                    if (e.pre) {
                        stage();
                        if (DIRECT)
                            copy_rows<T, true, 1>(hbuf, static_cast<T*>(e.pre), e.ldp, m0, c0, g.m, g.n, lane);
                        else
                            put(&tp, m0, in);
                    }
                    if (e.act != FG_ACT_NONE) {
#pragma unroll 4
                        for (int j = 0; j < 32; ++j) v[j] = activate<false>(v[j], e.act);
                    }
                    // the sums and z were read and written here by ordinary accesses: before a copy lands on them
                    if (!DIRECT && e.residual) tc::fence_proxy_async();
                    if (tc::elect_one()) tc::bulk_wait_read<0>();
                    __syncwarp();
                    if (e.residual) {
                        if (DIRECT) {
                            copy_rows<T, false, 8>(hbuf, const_cast<T*>(static_cast<const T*>(e.residual)), e.ldr, m0, c0, g.m, g.n, lane);
                        } else {
                            if (tc::elect_one()) {
                                tc::mbar_arrive_expect_tx(&res_full[w], GP_BUF);
                                tc::tma_load_2d(hbuf, &tr, &res_full[w], c0, m0);
                            }
                            lost = !copy_landed(&res_full[w], res_phase, fail);
                            res_phase ^= 1;
                            if (lost) {
                                store_nan<T>(e.y, e.ldy, m0, c0, g.m, g.n, 32);
                                continue;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 r = *reinterpret_cast<const float4*>(hrow + (((uint32_t)j << 2) ^ sw));
                            v[j] += r.x;
                            v[j + 1] += r.y;
                            v[j + 2] += r.z;
                            v[j + 3] += r.w;
                        }
                    }
                    stage();
                    if (DIRECT)
                        copy_rows<T, true, 1>(hbuf, static_cast<T*>(e.y), e.ldy, m0, c0, g.m, g.n, lane);
                    else
                        put(&ty, m0, in);
                }
            }
        } else if constexpr (MODE == TC_GATED) {
            const uint32_t sw64 = (uint32_t)(lane >> 1 & 3) << 4;
            for (; item < items; item += step, li += P::GROUPS) {
                const int acc = li & 1, col = item % g.nt * BO + part * PC, m0 = item / g.nt * 2 * GT_M + tr_rows;
                unsigned char* bias = biases + w * 128;
                if (e.bias) {  // 32 of the gates, 32 of their partners
                    const T* b = static_cast<const T*>(e.bias) + (lane < 16 ? 0 : g.up) + col;
                    reinterpret_cast<uint32_t*>(bias)[lane] = fetch_bias<T>(b, lane & 15, g.n - col, DIRECT);
                    __syncwarp();
                }
                const bool ok = tc::mbar_wait_warp(&acc_full[acc], (li >> 1) & 1, fail);
                tc::fence_after_sync();
                const uint32_t src = taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * BN + part * PC);
                float v[2][32];
                tc::tmem_ld_32x32_nowait(src, v[0]);
                tc::tmem_ld_32x32_nowait(src + BO, v[1]);
                tc::tmem_ld_wait(v[0]);
                tc::tmem_ld_wait(v[1]);
                tc::fence_before_sync();
                __syncwarp();
                if (tc::elect_one()) tc::mbar_arrive_leader(tc::leader_addr(&acc_empty[acc]));
                if (!ok) {  // a wait that ran out leaves NaN, not a plausible number
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[0][j] = v[1][j] = NAN;
                }
                if (e.bias) add_bias<T>(v, bias);
                // rows of 64 bytes, 32 of them: a half of the buffer
                auto stage = [&](const float (&v)[32], int h) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4*>(buf + h * (GP_BUF / 2) + lane * 64 + (((uint32_t)j << 1) ^ sw64)) = pack8<T>(&v[j]);
                };
                const bool inside = m0 < g.m && col < g.n;
                if (e.pre && DIRECT) {
                    stage(v[0], 0);
                    stage(v[1], 1);
                    store_half<T>(buf, static_cast<T*>(e.pre), e.ldp, m0, col, g.m, g.n, lane);
                    store_half<T>(buf + GP_BUF / 2, static_cast<T*>(e.pre) + g.up, e.ldp, m0, col, g.m, g.n, lane);
                } else if (e.pre) {
                    if (tc::elect_one()) tc::bulk_wait_read<1>();  // the last tile's: its result may still leave
                    __syncwarp();
                    stage(v[0], 0);
                    stage(v[1], 1);
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (tc::elect_one()) {
                        if (inside) {
                            tc::tma_store_2d(&tp, buf, col, m0);
                            tc::tma_store_2d(&tr, buf + GP_BUF / 2, col, m0);
                        }
                        tc::bulk_commit();
                    }
                }
                switch (e.act) {
                    case FG_ACT_RELU: gate_all<FG_ACT_RELU>(v); break;
                    case FG_ACT_GELU: gate_all<FG_ACT_GELU>(v); break;
                    case FG_ACT_SILU: gate_all<FG_ACT_SILU>(v); break;
                    default: gate_all<FG_ACT_NONE>(v);
                }
                if (DIRECT) {
                    stage(v[0], 2);
                    store_half<T>(buf + GP_BUF, static_cast<T*>(e.y), e.ldy, m0, col, g.m, g.n, lane);
                    continue;
                }
                if (tc::elect_one()) {  // the last tile's result has left; this one's pre-activations may yet
                    if (e.pre)
                        tc::bulk_wait_read<1>();
                    else
                        tc::bulk_wait_read<0>();
                }
                __syncwarp();
                stage(v[0], 2);
                tc::fence_proxy_async();
                __syncwarp();
                if (tc::elect_one()) {
                    if (inside) tc::tma_store_2d(&ty, buf + GP_BUF, col, m0);
                    tc::bulk_commit();
                }
            }
        } else if constexpr (MODE == TC_INT8) {
            // A tile's products take 512 cycles for 128 k, so that the epilogue bounds short k (1M rows
            // of 128 codes 505 us, of 768 764, where the operands come from L2 too slowly): two
            // buffers a warp, and the next tile's residual travels during this one's epilogue (1M x
            // 768 -> 768 float16 with residual, at the power cap: 904 us, 946 with one buffer and one
            // value at a time).  The columns' scales come from L1, which the operands pass by.
            T* residual = const_cast<T*>(static_cast<const T*>(e.residual));
            auto fetch = [&](int it, int i) {  // lane 0, once the buffer is free
                tc::mbar_arrive_expect_tx(&res_full[2 * w + (i & 1)], GP_BUF);
                tc::tma_load_2d(buf + (i & 1) * GP_BUF, &tr, &res_full[2 * w + (i & 1)], it % g.nt * BN + part * 64,
                                it / g.nt * 2 * GT_M + tr_rows);
            };
            if (!DIRECT && e.residual && item < items && tc::elect_one()) fetch(item, 0);
            bool flying = false;  // after a copy that never came: the next one is under way, and lands before the block ends
            for (int i = 0; item < items; item += step, li += P::GROUPS, ++i) {
                const int acc = li & 1, col = item % g.nt * BN + part * 64, m0 = item / g.nt * 2 * GT_M + tr_rows;
                unsigned char *ibuf = buf + (i & 1) * GP_BUF, *irow = ibuf + lane * 128;
                if (lost) {
                    if (flying) tc::mbar_wait(&res_full[2 * w + (i & 1)], (i >> 1) & 1);
                    flying = false;
                    store_nan<T>(e.y, e.ldy, m0, col, g.m, g.n, 64);
                    continue;
                }
                if (!DIRECT) {
                    if (tc::elect_one()) {
                        tc::bulk_wait_read<0>();  // the last tile's results have left the other buffer
                        if (e.residual && item + step < items) fetch(item + step, i + 1);
                    }
                    __syncwarp();
                }
                unsigned char* bias = biases + w * 128;
                if (e.bias) {
                    reinterpret_cast<uint32_t*>(bias)[lane] = fetch_bias<T>(static_cast<const T*>(e.bias) + col, lane, g.n - col, DIRECT);
                    __syncwarp();
                }
                if (DIRECT && e.residual) copy_rows<T, false, 8>(ibuf, residual, e.ldr, m0, col, g.m, g.n, lane);
                const float xs = m0 + lane < g.m ? __ldg(g.xs + m0 + lane) : 0.0f;
                const bool ok = tc::mbar_wait_warp(&acc_full[acc], (li >> 1) & 1, fail);
                tc::fence_after_sync();
                const uint32_t src = taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * BN + part * 64);
                float v[2][32];
                tc::tmem_ld_32x32_nowait(src, v[0]);
                tc::tmem_ld_32x32_nowait(src + 32, v[1]);
                tc::tmem_ld_wait(v[0]);
                tc::tmem_ld_wait(v[1]);
                tc::fence_before_sync();
                __syncwarp();
                if (tc::elect_one()) tc::mbar_arrive_leader(tc::leader_addr(&acc_empty[acc]));
                if (g.quads)
                    dequantise_all<T, true>(v, g.ws, col, g.n, xs, e.bias ? bias : nullptr);
                else
                    dequantise_all<T, false>(v, g.ws, col, g.n, xs, e.bias ? bias : nullptr);
                if (!ok) {  // a wait that ran out leaves NaN, not a plausible number
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[0][j] = v[1][j] = NAN;
                }
                switch (e.act) {
                    case FG_ACT_RELU: activate_all<FG_ACT_RELU>(v); break;
                    case FG_ACT_GELU: activate_all<FG_ACT_GELU>(v); break;
                    case FG_ACT_SILU: activate_all<FG_ACT_SILU>(v); break;
                }
                if (e.residual) {
                    if (!DIRECT) {
                        lost = flying = !copy_landed(&res_full[2 * w + (i & 1)], (i >> 1) & 1, fail);
                        if (lost) {
                            store_nan<T>(e.y, e.ldy, m0, col, g.m, g.n, 64);
                            continue;
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
                            add8<T>(&v[h][j], *reinterpret_cast<const uint4*>(irow + (((uint32_t)(32 * h + j) << 1) ^ sw)));
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4*>(irow + (((uint32_t)(32 * h + j) << 1) ^ sw)) = pack8<T>(&v[h][j]);
                if (DIRECT) {
                    copy_rows<T, true, 1>(ibuf, static_cast<T*>(e.y), e.ldy, m0, col, g.m, g.n, lane);
                    continue;
                }
                tc::fence_proxy_async();
                __syncwarp();
                if (tc::elect_one()) {
                    if (m0 < g.m && col < g.n) tc::tma_store_2d(&ty, ibuf, col, m0);
                    tc::bulk_commit();
                }
            }
        } else {
        for (; item < items; item += step, li += P::GROUPS) {
            const int acc = li & 1, t = item / g.split;
            const int col = t % g.nt * BN + part * 64, m0 = t / g.nt * 2 * GT_M + tr_rows;
            const bool inside = m0 < g.m && col < g.n;
            if (!DIRECT && lost) {
                store_nan<T>(e.pre, e.ldp, m0, col, g.m, g.n, 64);
                store_nan<T>(e.y, e.ldy, m0, col, g.m, g.n, 64);
                continue;
            }
            unsigned char* bias = biases + w * 128;
            if (e.bias) {
                reinterpret_cast<uint32_t*>(bias)[lane] = fetch_bias<T>(static_cast<const T*>(e.bias) + col, lane, g.n - col, DIRECT);
                __syncwarp();
            }
            T* residual = const_cast<T*>(static_cast<const T*>(e.residual));
            if (DIRECT && ahead) copy_rows<T, false, 8>(buf, residual, e.ldr, m0, col, g.m, g.n, lane);
            const bool ok = tc::mbar_wait_warp(&acc_full[acc], (li >> 1) & 1, fail);
            tc::fence_after_sync();
            const uint32_t src = taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * BN + part * 64);
            float v[2][32];
            tc::tmem_ld_32x32_nowait(src, v[0]);
            tc::tmem_ld_32x32_nowait(src + 32, v[1]);
            tc::tmem_ld_wait(v[0]);
            tc::tmem_ld_wait(v[1]);
            tc::fence_before_sync();
            __syncwarp();
            if (tc::elect_one()) tc::mbar_arrive_leader(tc::leader_addr(&acc_empty[acc]));
            if (g.split > 1) {  // this part's sums as they are; finish_kernel adds the parts
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (tc::elect_one()) tc::bulk_wait_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4*>(brow + (((uint32_t)j << 2) ^ sw)) =
                            ok ? make_float4(v[h][j], v[h][j + 1], v[h][j + 2], v[h][j + 3])
                               : make_float4(NAN, NAN, NAN, NAN);
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (tc::elect_one()) {
                        if (col + 32 * h < g.n)
                            tc::tma_store_2d(&ty, buf, col + 32 * h, (item - t * g.split) * g.m_pad + m0);
                        tc::bulk_commit();
                    }
                }
                continue;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!ok) {  // a wait that ran out leaves NaN, not a plausible number
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[h][j] = NAN;
                }
            }
            if (PARTS) {
                bool odd = false;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        v[h][j] *= scale;
                        odd |= !(fabsf(v[h][j]) <= FLT_MAX);
                    }
                if (__any_sync(0xffffffffu, odd && ok)) {
                    odd_seen = true;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[h][j] = fabsf(v[h][j]) <= FLT_MAX ? v[h][j] : NAN;
                }
            }
            if (e.bias) add_bias<T>(v, bias);
            if (e.pre) {
                if (tc::elect_one()) tc::bulk_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4*>(brow + (((uint32_t)(32 * h + j) << 1) ^ sw)) = pack8<T>(&v[h][j]);
                if (DIRECT) {
                    copy_rows<T, true, 1>(buf, static_cast<T*>(e.pre), e.ldp, m0, col, g.m, g.n, lane);
                } else {
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (tc::elect_one()) {
                        if (inside) tc::tma_store_2d(&tp, buf, col, m0);
                        tc::bulk_commit();
                    }
                }
            }
            switch (e.act) {
                case FG_ACT_RELU: activate_all<FG_ACT_RELU>(v); break;
                case FG_ACT_GELU: activate_all<FG_ACT_GELU>(v); break;
                case FG_ACT_SILU: activate_all<FG_ACT_SILU>(v); break;
            }
            if (DIRECT) {
                if (e.residual && !ahead) copy_rows<T, false, 4>(buf, residual, e.ldr, m0, col, g.m, g.n, lane);
            } else if (!ahead) {  // the buffer's last store has read it
                if (tc::elect_one()) {
                    tc::bulk_wait_read<0>();
                    if (e.residual) fetch_residual(item);
                }
                __syncwarp();
            }
            if (e.residual) {
                if (!DIRECT) {
                    lost = !copy_landed(&res_full[w], res_phase, fail);
                    res_phase ^= 1;
                    if (lost) {
                        store_nan<T>(e.y, e.ldy, m0, col, g.m, g.n, 64);
                        continue;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        add8<T>(&v[h][j], *reinterpret_cast<const uint4*>(brow + (((uint32_t)(32 * h + j) << 1) ^ sw)));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 32; j += 8)
                    *reinterpret_cast<uint4*>(brow + (((uint32_t)(32 * h + j) << 1) ^ sw)) = pack8<T>(&v[h][j]);
            if (DIRECT) {
                copy_rows<T, true, 1>(buf, static_cast<T*>(e.y), e.ldy, m0, col, g.m, g.n, lane);
                continue;
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (tc::elect_one()) {
                if (inside) tc::tma_store_2d(&ty, buf, col, m0);
                tc::bulk_commit();
                if (ahead && item + step < items) {  // the next tile's residual travels during its products
                    tc::bulk_wait_read<0>();
                    fetch_residual(item + step);
                }
            }
        }
        }
        if (tc::elect_one()) {
            if (odd_seen) s_odd = 1;
            tc::bulk_wait_read<0>();
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::cluster_sync();  // no CTA leaves while its peer still reads its memory
    tc::fence_after_sync();
    if (warp == 1) tc::tmem_dealloc_pair(taddr, 2 * BN);
    // Results that are not finite lie in this CTA's tiles as NaN, and are taken again here,
    // where nothing waits: each is a sum over all of k by one thread.
    if (products == 1 || !s_odd || s_fail) return;
    if (warp >= 2 && tc::elect_one()) tc::bulk_wait();  // this block's stores have arrived
    __syncthreads();
    const Epilogue& e = g.e;
    const T* mark = static_cast<const T*>(e.pre ? e.pre : e.y);
    const long long ld = e.pre ? e.ldp : e.ldy;
    for (int t = blockIdx.x >> 1; t < items; t += pairs) {
        const int m0 = t / g.nt * 2 * GT_M + rank * GT_M, n0 = t % g.nt * BO;
        for (int i = tid; i < GT_M * BO; i += GP_NT) {
            const int row = m0 + i / BO, col = n0 + i % BO;
            if (row >= g.m || col >= g.n) continue;
            float y = to_f32(__ldcg(mark + row * ld + col));
            if (MODE == TC_GATED && e.pre) y += to_f32(__ldcg(mark + row * ld + g.up + col));
            if (MODE == TC_GATED ? !(fabsf(y) <= FLT_MAX) : y != y) {
                if (MODE == TC_GATED)
                    gated_store<T>(e, g.up, row, col, retake<T>(g, row, col), retake<T>(g, row, g.up + col));
                else
                    epilogue_store<T>(e, row, col, retake<T>(g, row, col));
            }
        }
    }
}

// The parts of split tiles, added in their order, and the epilogue: four columns a thread.
template <class T, bool PARTS>
__global__ void __launch_bounds__(256) finish_kernel(const float* part, const __grid_constant__ TcArgs g, long long ldp) {
    const int c4 = (g.n + 3) / 4;
    const long long i = blockIdx.x * 256ll + threadIdx.x, row = i / c4;
    if (row >= g.m) return;
    const int col = (int)(i - row * c4) * 4;
    const float* p = part + row * ldp + col;
    float4 z = *reinterpret_cast<const float4*>(p);
    for (int s = 1; s < g.split; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(p + s * (g.m_pad * ldp));
        z.x += v.x;
        z.y += v.y;
        z.z += v.z;
        z.w += v.w;
    }
    constexpr float scale = PARTS ? PartsOf<T>::hi : 1.0f;
    if (PARTS) z = make_float4(z.x * scale, z.y * scale, z.z * scale, z.w * scale);
    float v[4] = {z.x, z.y, z.z, z.w};
    if (sizeof(T) == 4 || PARTS) {
        for (int j = 0; j < 4; ++j)
            if (col + j < g.n) v[j] = finite_or_retake<T>(g, (int)row, col + j, v[j]);
        z = make_float4(v[0], v[1], v[2], v[3]);
    }
    if (g.vec && col + 4 <= g.n && !g.e.bias && !g.e.pre && !g.e.residual && g.e.act == FG_ACT_NONE)
        store4(static_cast<T*>(g.e.y) + row * g.e.ldy + col, z);
    else
        for (int j = 0; j < 4 && col + j < g.n; ++j) epilogue_store<T>(g.e, row, col + j, v[j]);
}

// ---- host side ---------------------------------------------------------------

// Operand of `rows` rows of 16-bit elements, or of bytes (unit stride along k: [rows][k], else [k][rows]), in
// `planes` planes `plane` elements apart.
static int operand_map(CUtensorMap* m, int dtype, const void* p, long long rows, long long k, long long ld, bool mn,
                       int box_rows, int planes, long long plane, bool bytes = false) {
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3] = {(cuuint64_t)(mn ? rows : k), (cuuint64_t)(mn ? k : rows), (cuuint64_t)planes};
    const int es = bytes ? 1 : 2;
    cuuint64_t strides[2] = {(cuuint64_t)ld * es, (cuuint64_t)plane * es};
    cuuint32_t box[3] = {(cuuint32_t)(128 / es), (cuuint32_t)(mn ? GT_K : box_rows), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : dtype == FG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           3, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FG_OK;
}

static int a_planes(const TcArgs& g) { return g.products == 6 ? 3 : g.products; }
static int b_planes(const TcArgs& g) { return g.products == 6 ? 3 : 1; }

// Instruction descriptor, kind::f16: f32 accumulators.
static uint32_t instr_desc(int dtype, int m, int n, bool a_mn, bool b_mn) {
    const uint32_t t = dtype == FG_DTYPE_F16 ? 0 : 1;
    return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Of signed bytes, kind::i8: 32-bit integer accumulators.
static uint32_t instr_desc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

bool tc_gemm_fits(const void* a, const void* b, const GemmShape& g) {
    const long long lda = g.ak == 1 ? g.am : g.ak, ldb = g.bk == 1 ? g.bn : g.bk;
    return aligned(a, 16) && aligned(b, 16) && lda % 8 == 0 && ldb % 8 == 0 && g.k > 0 && g.m < (1ll << 31) - 512 &&
           g.n < (1ll << 31) - 512 && g.k < (1ll << 31) - 512;
}

template <class T, int BN, int MODE = TC_WHOLE>
static int launch_split(int dtype, const void* a, const void* b, const GemmShape& s, TcArgs g, cudaStream_t st) {
    constexpr bool I8 = MODE == TC_INT8;
    constexpr int BO = MODE == TC_GATED ? BN / 2 : BN;
    CUtensorMap ta, tb;
    int rc = operand_map(&ta, dtype, a, s.m, s.k, g.a_mn ? s.ak : s.am, g.a_mn, GT_M, a_planes(g), g.a_plane, I8);
    if (!rc) rc = operand_map(&tb, dtype, b, s.n, s.k, g.b_mn ? s.bk : s.bn, g.b_mn, BO, b_planes(g), g.b_plane, I8);
    if (rc) return rc;
    g.idesc = I8 ? instr_desc_i8(GT_M, BN) : instr_desc(dtype, GT_M, BN, g.a_mn, g.b_mn);
    g.nt = (g.n + BO - 1) / BO;
    if (sizeof(T) == 4 && !I8)  // the plan's: each run of GP_CHUNK K blocks has its accumulator
        FG_REQUIRE((g.kt + g.split - 1) / g.split <= GP_CHUNK * (512 / BN), "%d K blocks: too many for a tile's accumulators", g.kt);
    const long long ctas = (long long)g.mt * g.nt * g.split;
    FG_REQUIRE(ctas <= 0x7fffffffll, "%d x %d outputs: too many tiles", g.m, g.n);
    auto kernel = &gemm_split_kernel<T, BN, MODE>;
    if constexpr (sizeof(T) == 2 && MODE == TC_WHOLE)
        if (g.products == 2) kernel = &gemm_split_kernel<T, BN, TC_PARTS>;
    const int smem = RingOf<BN>::N * RingOf<BN>::STAGE + 1024;
    FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(GT_NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = g.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ta, tb, g));
    return FG_OK;
}

// Matrix [rows][n] for the epilogue's TMA: boxes of 32 rows of 128 or 64 bytes.
static int tile_map(CUtensorMap* m, int dtype, const void* p, long long rows, long long n, long long ld, int wide = 128) {
    if (!p) return FG_OK;  // the kernel does not touch it
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int es = dtype_size(dtype);
    cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * es};
    cuuint32_t box[2] = {(cuuint32_t)(wide / es), 32};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType t = dtype == FG_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : dtype == FG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = enc(m, t, 2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           wide == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FG_OK;
}

template <class T, int BN, int MODE = TC_WHOLE>
static int launch_pair(int dtype, const void* a, const void* b, const GemmShape& s, TcArgs g, void* ws, cudaStream_t st) {
    constexpr bool I8 = MODE == TC_INT8;
    constexpr int BO = MODE == TC_GATED ? BN / 2 : BN, wide = MODE == TC_GATED && sizeof(T) == 2 ? 64 : 128;
    using P = PairOf<T, BN, MODE>;
    CUtensorMap ta, tb, ty = {}, tp = {}, tr = {};
    const Epilogue& e = g.e;
    const long long ld = (s.n + 3) / 4 * 4;
    g.mt = (g.m + 2 * GT_M - 1) / (2 * GT_M);
    g.nt = (g.n + BO - 1) / BO;
    g.m_pad = g.mt * 2 * GT_M;
    int rc = operand_map(&ta, dtype, a, s.m, s.k, g.a_mn ? s.ak : s.am, g.a_mn, GT_M, a_planes(g), g.a_plane, I8);
    if (!rc) rc = operand_map(&tb, dtype, b, s.n, s.k, g.b_mn ? s.bk : s.bn, g.b_mn, BN / 2, b_planes(g), g.b_plane, I8);
    if (g.split > 1) {
        if (!rc) rc = tile_map(&ty, FG_DTYPE_F32, ws, (long long)g.split * g.m_pad, ld, ld);
    } else if (!g.direct) {
        if (!rc) rc = tile_map(&ty, dtype, e.y, s.m, g.n, e.ldy, wide);
        if (!rc) rc = tile_map(&tp, dtype, e.pre, s.m, g.n, e.ldp, wide);
        // gated: the partners' part of pre, a map of its own, as the gates' ends at its last column
        if (!rc && MODE == TC_GATED && e.pre)
            rc = tile_map(&tr, dtype, static_cast<const char*>(e.pre) + (size_t)g.up * dtype_size(dtype), s.m, g.n, e.ldp, wide);
        if (!rc && MODE != TC_GATED) rc = tile_map(&tr, dtype, e.residual, s.m, s.n, e.ldr, wide);
    }
    if (rc) return rc;
    g.idesc = I8 ? instr_desc_i8(2 * GT_M, BN) : instr_desc(dtype, 2 * GT_M, BN, g.a_mn, g.b_mn);
    const long long items = (long long)g.mt * g.nt * g.split;
    FG_REQUIRE(items <= 0x3fffffffll && (long long)g.split * g.m_pad <= 0x7fffffffll, "%d x %d outputs: too many tiles", g.m,
               g.n);
    const bool direct = g.direct && g.split == 1;
    auto kernel = &gemm_pair_kernel<T, BN, false, MODE>;
    if (direct) kernel = &gemm_pair_kernel<T, BN, true, MODE>;
    if constexpr (sizeof(T) == 2 && MODE == TC_WHOLE)
        if (g.products == 2) kernel = direct ? &gemm_pair_kernel<T, BN, true, TC_PARTS> : &gemm_pair_kernel<T, BN, false, TC_PARTS>;
    FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), P::SMEM));
    const int pairs = std::max(1, device_attr(cudaDevAttrMultiProcessorCount) / 2);
    TcArgs k = g;
    if (g.split > 1) k.e.bias = k.e.residual = k.e.pre = nullptr;  // finish_kernel's
    kernel<<<2 * (unsigned)std::min<long long>(items, pairs), GP_NT, P::SMEM, st>>>(ta, tb, ty, tp, tr, k);
    rc = check_launch("gemm_pair_kernel");
    if (rc || g.split == 1) return rc;
    const long long n4 = (long long)g.m * ((g.n + 3) / 4);
    auto finish = sizeof(T) == 2 && g.products == 2 ? &finish_kernel<T, true> : &finish_kernel<T, false>;
    finish<<<(unsigned)((n4 + 255) / 256), 256, 0, st>>>(static_cast<const float*>(ws), g, ld);
    return check_launch("finish_kernel");
}

// The kernel, tile width and split that finish first by this estimate in
// microseconds, fitted to 16-bit runs of 1 to 7 waves of each (within 15 %): a K block takes
// a pair 0.39 (256 columns; 512 cycles of products) or 0.34 (128), a CTA of the
// other kernel 0.43, 0.30 or 0.21 (256, 128, 64); a tile's epilogue runs behind the
// next tile's products in the pair kernel, after them in the other.  Parts of a tile
// meet in distributed shared memory (clusters, of which 74, 32 and 14 of two, four
// and eight CTAs run at once) or, with pairs, in the workspace and one more launch.
// 10,000 x 768 -> 1536: forward pairs 256 26 us (128: 36; one CTA a tile: 65), dw in
// 4 parts of pairs 29 us (2 parts 38, clusters of 4 45); 100 x 1536 -> 768: clusters
// of 8, 64 columns, 7.8 us (of 4 8.3, unsplit 12, pairs 10).  Float32 counts as six times
// the K blocks; its epilogue, 32 columns at a time, is not in the estimate, which is
// therefore far off where k is short (160,930 x 32 -> 524: 69 us, measured 615).
struct TcPlan {
    bool pair;
    int bn, split;
    size_t ws;
};

static TcPlan tc_plan_of(const GemmShape& s, int products, bool direct, int mode = TC_WHOLE) {
    const int sms = std::max(2, device_attr(cudaDevAttrMultiProcessorCount));
    const int kt = (int)((s.k + GT_K - 1) / GT_K) * products;
    auto waves = [](long long tiles, int slots) { return (double)((tiles + slots - 1) / slots); };
    TcPlan best{false, 0, 1, 0};  // bn 0: none
    double least = 1e300;
    auto offer = [&](double cost, const TcPlan& p) {
        if (cost < least) {
            least = cost;
            best = p;
        }
    };
    const long long m2 = (s.m + 2 * GT_M - 1) / (2 * GT_M), m1 = (s.m + GT_M - 1) / GT_M;
    const int kb = (int)((s.k + GT_K - 1) / GT_K);
    for (int bn : {256, 128}) {
        if ((products == 6 || mode == TC_GATED) && bn == 128) break;
        const long long tiles = m2 * ((s.n + bn - 1) / bn);
        // 16-bit sums run over GT_RUN K blocks at most: parts go on past 32, and past a full
        // GPU, until they are that short (in 64 bits: kb may be 2^25).  Integer ones are exact at
        // any length (4,096 x 65,552 -> 4,096 8 bits 1,127 us with pairs, 1,228 a CTA a tile).
        auto too_long = [&](int parts) { return products < 6 && mode != TC_INT8 && kb > (long long)GT_RUN * parts; };
        for (int sp = 1; sp <= 32 || too_long(sp / 2); sp = s.any_parts && sp < 32 ? sp + 1 : sp * 2) {
            if ((direct || mode != TC_WHOLE) && sp > 1) break;
            if (sp > 1 && (sp > kb / 2 || (tiles * sp > sms && kb <= (long long)GT_RUN * (sp / 2)))) break;
            if (too_long(sp)) continue;
            const size_t ws = sp > 1 ? (size_t)sp * m2 * 2 * GT_M * ((s.n + 3) / 4 * 4) * 4 : 0;
            const double epi = bn == 256 ? 2.0 : 1.0, main = (kt + sp - 1) / sp * (bn == 256 ? 0.39 : 0.34);
            const double rows = !direct ? 0.0 : mode == TC_GATED ? 9.0 : bn == 256 ? 14.0 : 8.0;
            offer(6.0 + waves(tiles * sp, sms / 2) * (std::max(main, epi) + rows) + epi + (sp > 1 ? 3.0 + 1.5e-6 * ws / 6.0 : 0.0),
                  TcPlan{true, bn, sp, ws});
        }
    }
    for (int bn : {256, 128, 64}) {
        const long long tiles = m1 * ((s.n + bn - 1) / bn);
        for (int sp : {1, 2, 4, 8}) {
            if (sp > kb || (direct && sp > 1)) break;
            // the sums' length: 512 k for each of float32's 512 / bn accumulators
            if (mode != TC_INT8 && kb > (products < 6 ? GT_RUN : GP_CHUNK * 512 / bn) * sp && kb > 3) continue;
            const int slots = sp == 1 ? sms : sp == 2 ? sms / 2 : std::max(1, sp == 4 ? sms * 32 / 148 : sms * 14 / 148);
            // waves of clusters cost 1.3 times this estimate: gated float32 20,000 x 768 -> 100 in fours
            // 105 us, in pairs 77; 390 x 5,113 -> 620 in eights 72, in pairs 190; of 110 gated and
            // 8-bit layers, where the two choices differ, the better one but for three (at most 12
            // %).  Plain layers keep the order of their sums.
            const double again = mode != TC_WHOLE && sp > 1 && tiles > slots ? 1.3 : 1.0;
            const double main = (kt + sp - 1) / sp * (bn == 256 ? 0.43 : bn == 128 ? 0.30 : 0.21);
            const double rows = direct ? 0.055 * bn : 0.0;
            offer(again * (5.0 + waves(tiles, slots) * (main + 2.0 + 0.02 * bn / sp + rows)) + (sp == 8 ? 0.7 : 0.0), TcPlan{false, bn, sp, 0});
        }
    }
    return best;
}

// Outputs that go row by row cost a wave 8 or 14 us more with pairs, less with small
// tiles (1777 x 101 -> 333 bf16: 27 us with pairs, 12 in tiles of 64 columns).  Only
// tiles whose sums are not split are chosen anew: those add in one order whichever
// kernel takes them, so that a result does not depend on where it is written.
static TcPlan tc_plan(const GemmShape& s, int products, bool direct, int mode = TC_WHOLE) {
    const TcPlan p = tc_plan_of(s, products, false, mode);
    return direct && p.split == 1 ? tc_plan_of(s, products, true, mode) : p;
}

static TcArgs tc_args(const void* a, long long a_plane, const void* b, long long b_plane, const GemmShape& s, int products,
                      const Epilogue& e) {
    TcArgs g{};
    g.m = (int)s.m;
    g.n = (int)s.n;
    g.kt = (int)((s.k + GT_K - 1) / GT_K);
    g.mt = (int)((s.m + GT_M - 1) / GT_M);
    g.a_mn = s.ak != 1;
    g.b_mn = s.bk != 1;
    g.products = products;
    g.f = s;
    g.fa = a;
    g.fb = b;
    g.a_plane = a_planes(g) == 1 ? 16 : a_plane;  // one plane: any multiple of 16 bytes
    g.b_plane = b_planes(g) == 1 ? 16 : b_plane;
    g.e = e;
    return g;
}

static int no_plan(const GemmShape& s) {
    return fail(FG_ERR_UNSUPPORTED, "%lld x %lld outputs of %lld products: no tiles hold their sums", s.m, s.n, s.k);
}

// Do all of the epilogue's matrices start their rows on n bytes?
static bool epilogue_lies(const Epilogue& e, int es, int n) {
    auto lies = [&](const void* p, long long ld) { return !p || (aligned(p, n) && ld * es % n == 0); };
    return lies(e.y, e.ldy) && lies(e.bias, 0) && lies(e.pre, e.ldp) && lies(e.residual, e.ldr);
}

size_t tc_gemm_workspace(int products, const GemmShape& s) {
    return s.k > 0 ? tc_plan(s, products, false).ws : 0;
}

int tc_gemm(int dtype, const void* a, long long a_plane, const void* b, long long b_plane, const GemmShape& s,
            const Epilogue& e, void* ws, cudaStream_t st) {
    TcArgs g = tc_args(a, a_plane, b, b_plane, s, tc_products(dtype, a_plane != 0), e);
    const int es = dtype_size(dtype);
    g.vec = epilogue_lies(e, es, 4 * es);
    g.direct = !epilogue_lies(e, es, 16);
    const TcPlan p = tc_plan(s, g.products, g.direct);
    if (!p.bn) return no_plan(s);
    g.split = p.split;
#define FG_PRODUCT(T)                                                                        \
    (p.pair ? (sizeof(T) == 4 || p.bn == 256                                              \
                   ? launch_pair<T, 256>(dtype, a, b, s, g, ws, st)                       \
                   : launch_pair<T, sizeof(T) == 4 ? 256 : 128>(dtype, a, b, s, g, ws, st)) \
            : (p.bn == 256   ? launch_split<T, 256>(dtype, a, b, s, g, st)                \
               : p.bn == 128 ? launch_split<T, 128>(dtype, a, b, s, g, st)                \
                             : launch_split<T, 64>(dtype, a, b, s, g, st)))
    return dtype == FG_DTYPE_F32 ? FG_PRODUCT(float) : dtype == FG_DTYPE_F16 ? FG_PRODUCT(__half) : FG_PRODUCT(__nv_bfloat16);
#undef FG_PRODUCT
}

int tc_gated(int dtype, const void* a, long long a_plane, const void* b, long long b_plane, const GemmShape& s, const Epilogue& e,
             cudaStream_t st) {
    TcArgs g = tc_args(a, a_plane, b, b_plane, s, tc_products(dtype, false), e);
    const int es = dtype_size(dtype);
    g.n = g.up = (int)(s.n / 2);
    // the partners' bias and pre-activations start `up` columns on
    auto both = [&](int n) { return epilogue_lies(e, es, n) && ((!e.bias && !e.pre) || (long long)g.up * es % n == 0); };
    g.vec = both(4 * es);
    g.direct = !both(16);
    const TcPlan p = tc_plan(s, g.products, g.direct, TC_GATED);
    if (!p.bn) return no_plan(s);
    g.split = p.split;
#define FG_PRODUCT(T)                                                            \
    (p.pair        ? launch_pair<T, 256, TC_GATED>(dtype, a, b, s, g, nullptr, st) \
     : p.bn == 256 ? launch_split<T, 256, TC_GATED>(dtype, a, b, s, g, st)         \
     : p.bn == 128 ? launch_split<T, 128, TC_GATED>(dtype, a, b, s, g, st)         \
                   : launch_split<T, 64, TC_GATED>(dtype, a, b, s, g, st))
    return dtype == FG_DTYPE_F32 ? FG_PRODUCT(float) : dtype == FG_DTYPE_F16 ? FG_PRODUCT(__half) : FG_PRODUCT(__nv_bfloat16);
#undef FG_PRODUCT
}

int tc_int8(int dtype, const void* a, const float* xs, const void* b, const float* ws, const GemmShape& s, const Epilogue& e,
            cudaStream_t st) {
    TcArgs g = tc_args(a, 0, b, 0, s, 1, e);
    const int es = dtype_size(dtype);
    g.kt = (int)((s.k + 2 * GT_K - 1) / (2 * GT_K));
    g.xs = xs;
    g.ws = ws;
    g.vec = epilogue_lies(e, es, 4 * es) && aligned(ws, 16);
    g.quads = aligned(ws, 16) && s.n % 4 == 0 && (es == 2 || aligned(e.bias, 16));
    g.direct = !epilogue_lies(e, es, 16);
    GemmShape half = s;  // a K block holds 128 codes and takes the time of 64 elements of 16 bits
    half.k = (s.k + 1) / 2;
    const TcPlan p = tc_plan_of(half, 1, g.direct, TC_INT8);
    if (!p.bn) return no_plan(s);
    g.split = p.split;
#define FG_PRODUCT(T)                                                                       \
    (p.pair ? (sizeof(T) == 4 || p.bn == 256                                                 \
                   ? launch_pair<T, 256, TC_INT8>(dtype, a, b, s, g, nullptr, st)            \
                   : launch_pair<T, sizeof(T) == 4 ? 256 : 128, TC_INT8>(dtype, a, b, s, g, nullptr, st)) \
     : p.bn == 256 ? launch_split<T, 256, TC_INT8>(dtype, a, b, s, g, st)                    \
     : p.bn == 128 ? launch_split<T, 128, TC_INT8>(dtype, a, b, s, g, st)                    \
                   : launch_split<T, 64, TC_INT8>(dtype, a, b, s, g, st))
    return dtype == FG_DTYPE_F32 ? FG_PRODUCT(float) : dtype == FG_DTYPE_F16 ? FG_PRODUCT(__half) : FG_PRODUCT(__nv_bfloat16);
#undef FG_PRODUCT
}

}  // namespace fg
