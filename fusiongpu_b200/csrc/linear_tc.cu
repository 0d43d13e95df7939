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
};

// Planes of the i-th plane product.
__device__ __forceinline__ int plane_a(int i, int products) {  // 0; 1 0; 0 2 1 0 1 0
    return products == 1 ? 0 : products == 2 ? 1 - i : (280 >> (2 * i)) & 3;
}
__device__ __forceinline__ int plane_b(int i, int products) { return products < 6 ? 0 : (82 >> (2 * i)) & 3; }  // 2 0 1 1 0 0

// An infinite operand times the small planes of the other has any sign: a result
// that is not finite is taken again, one product at a time.
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
            z = fmaf(PartsOf<T>::hi * to_f32(a[0]) + PartsOf<T>::lo * to_f32(a[g.a_plane]), to_f32(b[0]), z);
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

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// 16 bytes at shared address `a` of CTA `rank` of the cluster.
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t a, uint32_t rank) {
    float4 v;
    asm volatile(
        "{\n\t.reg .b32 p;\n\t"
        "mapa.shared::cluster.u32 p, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [p];\n\t}\n"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(a), "r"(rank)
        : "memory");
    return v;
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
template <class T, int BN, bool PARTS>
__global__ void __launch_bounds__(GT_NT, 1)
    gemm_split_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const __grid_constant__ TcArgs g) {
    using Ring = RingOf<BN>;
    constexpr int LDP = BN + 4;  // partial row: 4 floats of padding keep 16-byte stores off each other's banks
    static_assert(GT_M * LDP * 4 <= Ring::N * Ring::STAGE, "the partial tile fits the ring");
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t full[Ring::N], empty[Ring::N], acc_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* ring = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~static_cast<uintptr_t>(1023));
    float* part = reinterpret_cast<float*>(ring);
    const int S = g.split, rank = S > 1 ? (int)cluster_rank() : 0;
    const int tile = (int)(blockIdx.x / (unsigned)S);
    const int m0 = tile / g.nt * GT_M, n0 = tile % g.nt * BN;
    const int kb0 = (int)((long long)g.kt * rank / S), kb1 = (int)((long long)g.kt * (rank + 1) / S);
    // accumulators: one, or for float32 as many as TMEM holds, each for GP_CHUNK K blocks
    constexpr int NA = sizeof(T) == 4 ? 512 / BN : 1;
    const int share = sizeof(T) == 4 ? GP_CHUNK : kb1 - kb0, shares = (kb1 - kb0 + share - 1) / share;
    constexpr int products = sizeof(T) == 4 ? 6 : PARTS ? 2 : 1;

    if (warp == 2 && tc::elect_one()) {
        tc::prefetch_map(&ta);
        tc::prefetch_map(&tb);
    }
    if (tid == 0) {
        s_fail = 0;
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

    if (warp == 0) {
        if (tc::elect_one()) {  // ---- TMA producer
            int i = 0;
            bool ok = true;
            auto load = [&](int kb, int product) {
                const int st = i % Ring::N, k = kb * GT_K;
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
            for (int j = 0; j < 32; j += 4)  // a wait that ran out leaves NaN, not a plausible number
                *reinterpret_cast<float4*>(row + c + j) =
                    ok ? make_float4(v[j], v[j + 1], v[j + 2], v[j + 3])
                       : make_float4(NAN, NAN, NAN, NAN);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (S > 1) cluster_sync();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(taddr, NA * BN);
    }

    // Four positions per thread and round, their residuals and biases loaded first:
    // one memory latency a round.
    constexpr int U = 4;
    constexpr bool FAST = sizeof(T) == 2;
    constexpr float scale = PartsOf<T>::hi;
    const int slice = BN / S, per_row = slice / 4;
    const uint32_t pbase = tc::smem_u32(part);
    const Epilogue& e = g.e;
    for (int i0 = tid; i0 < GT_M * per_row; i0 += U * GT_NT) {
        int row[U], col[U];
        uint32_t at[U];
        float4 res[U], bias[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * GT_NT, r = i / per_row, c = rank * slice + (i - r * per_row) * 4;
            row[u] = i < GT_M * per_row ? m0 + r : g.m;
            col[u] = n0 + c;
            at[u] = (uint32_t)(r * LDP + c) * 4;
            res[u] = bias[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (row[u] < g.m && col[u] < g.n) {
                const T* rp = static_cast<const T*>(e.residual) + row[u] * e.ldr + col[u];
                const T* bp = static_cast<const T*>(e.bias) + col[u];
                if (g.vec && col[u] + 4 <= g.n) {
                    if (e.residual) res[u] = load4(rp);
                    if (e.bias) bias[u] = load4(bp);
                } else {
                    float* rf = &res[u].x;
                    float* bf = &bias[u].x;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col[u] + j < g.n) {
                            if (e.residual) rf[j] = to_f32(rp[j]);
                            if (e.bias) bf[j] = to_f32(bp[j]);
                        }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row[u] >= g.m || col[u] >= g.n) continue;
            float4 z;
            if (S > 1) {
                z = ld_cluster_f4(pbase + at[u], rank);
                for (int s = 1; s < S; ++s) {
                    const float4 v = ld_cluster_f4(pbase + at[u], (rank + s) & (S - 1));
                    z.x += v.x;
                    z.y += v.y;
                    z.z += v.z;
                    z.w += v.w;
                }
            } else {
                z = *reinterpret_cast<const float4*>(reinterpret_cast<const char*>(part) + at[u]);
            }
            const bool whole = col[u] + 4 <= g.n;
            if (PARTS) z = make_float4(z.x * scale, z.y * scale, z.z * scale, z.w * scale);
            if (products > 1) {
                z.x = finite_or_retake<T>(g, row[u], col[u], z.x);
                if (col[u] + 1 < g.n) z.y = finite_or_retake<T>(g, row[u], col[u] + 1, z.y);
                if (col[u] + 2 < g.n) z.z = finite_or_retake<T>(g, row[u], col[u] + 2, z.z);
                if (col[u] + 3 < g.n) z.w = finite_or_retake<T>(g, row[u], col[u] + 3, z.w);
            }
            z.x += bias[u].x;
            z.y += bias[u].y;
            z.z += bias[u].z;
            z.w += bias[u].w;
            auto put = [&](void* out, long long ld, const float4& v) {
                T* p = static_cast<T*>(out) + row[u] * ld + col[u];
                if (g.vec && whole) {
                    store4(p, v);
                } else {
                    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col[u] + j < g.n) p[j] = from_f32<T>(f[j]);
                }
            };
            if (e.pre) put(e.pre, e.ldp, z);
            float4 y = z;
            if (e.act == FG_ACT_GELU && FAST) {
                gelu2(y.x, y.y);
                gelu2(y.z, y.w);
            } else if (e.act != FG_ACT_NONE) {
                y = make_float4(activate<FAST>(z.x, e.act), activate<FAST>(z.y, e.act), activate<FAST>(z.z, e.act),
                                activate<FAST>(z.w, e.act));
            }
            y.x += res[u].x;
            y.y += res[u].y;
            y.z += res[u].z;
            y.w += res[u].w;
            put(e.y, e.ldy, y);
        }
    }
    if (S > 1) cluster_sync();  // a peer may still read this CTA's partial tile
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
template <class T, int BN>
struct PairOf {
    static constexpr int B = BN / 2 * GT_K * 2, STAGE = GP_A + B, STAGES = sizeof(T) == 4 ? 3 : 5;
    static constexpr int BUF = sizeof(T) == 4 ? 2 * GP_BUF : GP_BUF;
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

template <int ACT>
__device__ __forceinline__ void activate_all(float (&v)[2][32]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            if (ACT == FG_ACT_GELU) {
                gelu2(v[h][j], v[h][j + 1]);
            } else {
                v[h][j] = activate<true>(v[h][j], ACT);
                v[h][j + 1] = activate<true>(v[h][j + 1], ACT);
            }
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

template <class T>
__device__ __forceinline__ void add_bias(float (&v)[2][32], const unsigned char* b) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; j += 8) add8<T>(&v[h][j], *reinterpret_cast<const uint4*>(b + (32 * h + j) * 2));
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
// needs: they pass row by row between memory and the buffer.  PARTS: A in two parts.
template <class T, int BN, bool DIRECT, bool PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GP_NT, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap ty, const __grid_constant__ CUtensorMap tp,
                     const __grid_constant__ CUtensorMap tr, const __grid_constant__ TcArgs g) {
    using P = PairOf<T, BN>;
    constexpr int GP_STAGES = P::STAGES;
    static_assert(sizeof(T) == 2 || BN == 256, "float32 takes 256 columns");
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t full[GP_STAGES], empty[GP_STAGES], acc_full[2], acc_empty[2], res_full[GP_EPI];
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail, s_odd;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank();
    unsigned char *ring = dsmem, *bufs = ring + GP_STAGES * P::STAGE, *biases = bufs + GP_EPI * P::BUF;
    const int pairs = (int)(gridDim.x >> 1), items = g.mt * g.nt * g.split;
    auto k_begin = [&](int part) { return (int)((long long)g.kt * part / g.split); };
    constexpr int chunk = sizeof(T) == 4 ? GP_CHUNK : 1 << 30;
    constexpr int products = sizeof(T) == 4 ? 6 : PARTS ? 2 : 1;
    constexpr float scale = PartsOf<T>::hi;

    if (warp == 2 && tc::elect_one()) {
        tc::prefetch_map(&ta);
        tc::prefetch_map(&tb);
        if (!DIRECT) {
            tc::prefetch_map(&ty);
            if (g.e.pre) tc::prefetch_map(&tp);
            if (g.e.residual) tc::prefetch_map(&tr);
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
        for (int w = 0; w < GP_EPI; ++w) tc::mbar_init(&res_full[w], 1);
        tc::fence_mbar_init();
    }
    if (tid == 0 && (tc::smem_u32(dsmem) & 1023)) s_fail = 1;  // swizzled tiles start on 1,024 bytes
    if (warp == 1) tc::tmem_alloc_pair(&tmem_slot, 2 * BN);
    tc::fence_before_sync();
    __syncthreads();
    cluster_sync();  // the peer's barriers are ready too
    tc::fence_after_sync();
    const uint32_t taddr = tmem_slot;
    volatile int* fail = &s_fail;

    if (warp == 0) {
        if (tc::elect_one()) {  // ---- TMA producer (each CTA its own halves)
            int i = 0;
            bool ok = true;
            for (int w = blockIdx.x >> 1; w < items && ok; w += pairs) {
                const int t = w / g.split, sp = w - t * g.split, k1 = k_begin(sp + 1);
                const int m0 = t / g.nt * 2 * GT_M + rank * GT_M, n0 = t % g.nt * BN + rank * (BN / 2);
                auto load = [&](int kb, int product) {
                    const int st = i % GP_STAGES, k = kb * GT_K;
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
        const bool ahead = sizeof(T) == 2 && e.residual && !e.pre;  // residuals a tile ahead (DIRECT: during its products)
        if (!DIRECT && ahead && item < items && tc::elect_one()) fetch_residual(item);
        if constexpr (sizeof(T) == 4) {
            // Chunks of k are added to the sums in shared memory, a lane its own row, in
            // two halves of 32 columns; the last one is followed by the epilogue proper,
            // one step after the other: six products a K block hide it.
            for (; item < items; item += step) {
                const int t = item / g.split, sp = item - t * g.split, k1 = k_begin(sp + 1);
                const int col = t % g.nt * BN + part * 64, m0 = t / g.nt * 2 * GT_M + tr_rows;
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
                        tc::tmem_ld_32x32(taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(acc * BN + part * 64 + 32 * h), v);
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
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
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
    cluster_sync();  // no CTA leaves while its peer still reads its memory
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
        const int m0 = t / g.nt * 2 * GT_M + rank * GT_M, n0 = t % g.nt * BN;
        for (int i = tid; i < GT_M * BN; i += GP_NT) {
            const int row = m0 + i / BN, col = n0 + i % BN;
            if (row >= g.m || col >= g.n) continue;
            const float y = to_f32(__ldcg(mark + row * ld + col));
            if (y != y) epilogue_store<T>(e, row, col, retake<T>(g, row, col));
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

// Operand of `rows` rows (unit stride along k: [rows][k], else [k][rows]), in
// `planes` planes `plane` elements apart.
static int operand_map(CUtensorMap* m, int dtype, const void* p, long long rows, long long k, long long ld, bool mn,
                       int box_rows, int planes, long long plane) {
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3] = {(cuuint64_t)(mn ? rows : k), (cuuint64_t)(mn ? k : rows), (cuuint64_t)planes};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)(mn ? GT_K : box_rows), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, dtype == FG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
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

bool tc_gemm_fits(const void* a, const void* b, const GemmShape& g) {
    const long long lda = g.ak == 1 ? g.am : g.ak, ldb = g.bk == 1 ? g.bn : g.bk;
    return aligned(a, 16) && aligned(b, 16) && lda % 8 == 0 && ldb % 8 == 0 && g.k > 0 && g.m < (1ll << 31) - 512 &&
           g.n < (1ll << 31) - 512 && g.k < (1ll << 31) - 512;
}

template <class T, int BN>
static int launch_split(int dtype, const void* a, const void* b, const GemmShape& s, TcArgs g, cudaStream_t st) {
    CUtensorMap ta, tb;
    int rc = operand_map(&ta, dtype, a, s.m, s.k, g.a_mn ? s.ak : s.am, g.a_mn, GT_M, a_planes(g), g.a_plane);
    if (!rc) rc = operand_map(&tb, dtype, b, s.n, s.k, g.b_mn ? s.bk : s.bn, g.b_mn, BN, b_planes(g), g.b_plane);
    if (rc) return rc;
    g.idesc = instr_desc(dtype, GT_M, BN, g.a_mn, g.b_mn);
    g.nt = (g.n + BN - 1) / BN;
    const long long ctas = (long long)g.mt * g.nt * g.split;
    FG_REQUIRE(ctas <= 0x7fffffffll, "%d x %d outputs: too many tiles", g.m, g.n);
    auto kernel = &gemm_split_kernel<T, BN, false>;
    if constexpr (sizeof(T) == 2)
        if (g.products == 2) kernel = &gemm_split_kernel<T, BN, true>;
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

// Matrix [rows][n] for the epilogue's TMA: boxes of 32 rows of 128 bytes.
static int tile_map(CUtensorMap* m, int dtype, const void* p, long long rows, long long n, long long ld) {
    if (!p) return FG_OK;  // the kernel does not touch it
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int es = dtype_size(dtype);
    cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * es};
    cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType t = dtype == FG_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : dtype == FG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = enc(m, t, 2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FG_OK;
}

template <class T, int BN>
static int launch_pair(int dtype, const void* a, const void* b, const GemmShape& s, TcArgs g, void* ws, cudaStream_t st) {
    CUtensorMap ta, tb, ty = {}, tp = {}, tr = {};
    const Epilogue& e = g.e;
    const long long ld = (s.n + 3) / 4 * 4;
    g.mt = (g.m + 2 * GT_M - 1) / (2 * GT_M);
    g.nt = (g.n + BN - 1) / BN;
    g.m_pad = g.mt * 2 * GT_M;
    int rc = operand_map(&ta, dtype, a, s.m, s.k, g.a_mn ? s.ak : s.am, g.a_mn, GT_M, a_planes(g), g.a_plane);
    if (!rc) rc = operand_map(&tb, dtype, b, s.n, s.k, g.b_mn ? s.bk : s.bn, g.b_mn, BN / 2, b_planes(g), g.b_plane);
    if (g.split > 1) {
        if (!rc) rc = tile_map(&ty, FG_DTYPE_F32, ws, (long long)g.split * g.m_pad, ld, ld);
    } else if (!g.direct) {
        if (!rc) rc = tile_map(&ty, dtype, e.y, s.m, s.n, e.ldy);
        if (!rc) rc = tile_map(&tp, dtype, e.pre, s.m, s.n, e.ldp);
        if (!rc) rc = tile_map(&tr, dtype, e.residual, s.m, s.n, e.ldr);
    }
    if (rc) return rc;
    g.idesc = instr_desc(dtype, 2 * GT_M, BN, g.a_mn, g.b_mn);
    const long long items = (long long)g.mt * g.nt * g.split;
    FG_REQUIRE(items <= 0x3fffffffll && (long long)g.split * g.m_pad <= 0x7fffffffll, "%d x %d outputs: too many tiles", g.m,
               g.n);
    const bool direct = g.direct && g.split == 1;
    auto kernel = direct ? &gemm_pair_kernel<T, BN, true, false> : &gemm_pair_kernel<T, BN, false, false>;
    if constexpr (sizeof(T) == 2)
        if (g.products == 2) kernel = direct ? &gemm_pair_kernel<T, BN, true, true> : &gemm_pair_kernel<T, BN, false, true>;
    FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), PairOf<T, BN>::SMEM));
    const int pairs = std::max(1, device_attr(cudaDevAttrMultiProcessorCount) / 2);
    TcArgs k = g;
    if (g.split > 1) k.e.bias = k.e.residual = k.e.pre = nullptr;  // finish_kernel's
    kernel<<<2 * (unsigned)std::min<long long>(items, pairs), GP_NT, PairOf<T, BN>::SMEM, st>>>(ta, tb, ty, tp, tr, k);
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

static TcPlan tc_plan_of(const GemmShape& s, int products, bool direct) {
    const int sms = std::max(2, device_attr(cudaDevAttrMultiProcessorCount));
    const int kt = (int)((s.k + GT_K - 1) / GT_K) * products;
    auto waves = [](long long tiles, int slots) { return (double)((tiles + slots - 1) / slots); };
    TcPlan best{false, 256, 1, 0};
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
        if (products == 6 && bn == 128) break;
        const long long tiles = m2 * ((s.n + bn - 1) / bn);
        // 16-bit sums run over GT_RUN K blocks at most: parts go on past 32, and past a full
        // GPU, until they are that short (in 64 bits: kb may be 2^25)
        auto too_long = [&](int parts) { return products < 6 && kb > (long long)GT_RUN * parts; };
        for (int sp = 1; sp <= 32 || too_long(sp / 2); sp *= 2) {
            if (direct && sp > 1) break;
            if (sp > 1 && (sp > kb / 2 || (tiles * sp > sms && kb <= (long long)GT_RUN * (sp / 2)))) break;
            if (too_long(sp)) continue;
            const size_t ws = sp > 1 ? (size_t)sp * m2 * 2 * GT_M * ((s.n + 3) / 4 * 4) * 4 : 0;
            const double epi = bn == 256 ? 2.0 : 1.0, main = (kt + sp - 1) / sp * (bn == 256 ? 0.39 : 0.34);
            const double rows = direct ? (bn == 256 ? 14.0 : 8.0) : 0.0;
            offer(6.0 + waves(tiles * sp, sms / 2) * (std::max(main, epi) + rows) + epi + (sp > 1 ? 3.0 + 1.5e-6 * ws / 6.0 : 0.0),
                  TcPlan{true, bn, sp, ws});
        }
    }
    for (int bn : {256, 128, 64}) {
        const long long tiles = m1 * ((s.n + bn - 1) / bn);
        for (int sp : {1, 2, 4, 8}) {
            if (sp > kb || (direct && sp > 1)) break;
            // the sums' length: 512 k for each of float32's 512 / bn accumulators
            if (kb > (products < 6 ? GT_RUN : GP_CHUNK * 512 / bn) * sp && kb > 3) continue;
            const int slots = sp == 1 ? sms : sp == 2 ? sms / 2 : std::max(1, sp == 4 ? sms * 32 / 148 : sms * 14 / 148);
            const double main = (kt + sp - 1) / sp * (bn == 256 ? 0.43 : bn == 128 ? 0.30 : 0.21);
            const double rows = direct ? 0.055 * bn : 0.0;
            offer(5.0 + waves(tiles, slots) * (main + 2.0 + 0.02 * bn / sp + rows) + (sp == 8 ? 0.7 : 0.0), TcPlan{false, bn, sp, 0});
        }
    }
    return best;
}

// Outputs that go row by row cost a wave 8 or 14 us more with pairs, less with small
// tiles (1777 x 101 -> 333 bf16: 27 us with pairs, 12 in tiles of 64 columns).  Only
// tiles whose sums are not split are chosen anew: those add in one order whichever
// kernel takes them, so that a result does not depend on where it is written.
static TcPlan tc_plan(const GemmShape& s, int products, bool direct) {
    const TcPlan p = tc_plan_of(s, products, false);
    return direct && p.split == 1 ? tc_plan_of(s, products, true) : p;
}

size_t tc_gemm_workspace(int products, const GemmShape& s) {
    return s.k > 0 ? tc_plan(s, products, false).ws : 0;
}

int tc_gemm(int dtype, const void* a, long long a_plane, const void* b, long long b_plane, const GemmShape& s,
            const Epilogue& e, void* ws, cudaStream_t st) {
    TcArgs g{};
    g.m = (int)s.m;
    g.n = (int)s.n;
    g.kt = (int)((s.k + GT_K - 1) / GT_K);
    g.mt = (int)((s.m + GT_M - 1) / GT_M);
    g.a_mn = s.ak != 1;
    g.b_mn = s.bk != 1;
    g.products = tc_products(dtype, a_plane != 0);
    g.f = s;
    g.fa = a;
    g.fb = b;
    g.a_plane = a_planes(g) == 1 ? 8 : a_plane;  // one plane: any multiple of 16 bytes
    g.b_plane = b_planes(g) == 1 ? 8 : b_plane;
    g.e = e;
    const int es = dtype_size(dtype);
    auto lies = [&](const void* p, long long ld, int n) { return !p || (aligned(p, n) && ld * es % n == 0); };
    g.vec = lies(e.y, e.ldy, 4 * es) && lies(e.bias, 0, 4 * es) && lies(e.pre, e.ldp, 4 * es) && lies(e.residual, e.ldr, 4 * es);
    g.direct = !(lies(e.y, e.ldy, 16) && lies(e.bias, 0, 16) && lies(e.pre, e.ldp, 16) && lies(e.residual, e.ldr, 16));
    const TcPlan p = tc_plan(s, g.products, g.direct);
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

}  // namespace fg
