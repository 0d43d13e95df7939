// linear_tc.cu -- the linear layer's products on the 5th-generation tensor cores:
// C(m, n) = sum over k of A(m, k) B(n, k), 16-bit operands, fp32 accumulators in
// TMEM.  Either operand may have unit stride along k (K-major: x and w of the
// forward pass, dz of dx = dz w) or along its rows (MN-major: w of dx, both
// operands of dw = dz^T x), so no pass over memory transposes anything.
#include <algorithm>

#include "linear.cuh"
#include "tc_common.cuh"

namespace fg {

constexpr int GT_M = 128;          // UMMA M: rows of a tile, TMEM lanes
constexpr int GT_K = 64;           // elements of a K block: one 128-byte swizzle row
constexpr int GT_NT = 64 + 256;    // TMA warp, MMA warp, 8 epilogue warps
constexpr int GT_RING = 192 * 1024;

struct TcArgs {
    int kt, mt, nt;     // K blocks, row tiles, column tiles
    int m, n;
    int a_mn, b_mn;
    int split;          // CTAs of a cluster that share a tile's K range
    int vec;            // outputs, residual and bias allow 4-column accesses
    uint32_t idesc;
    Epilogue e;
};

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

template <class T>
__device__ __forceinline__ void store4(T* p, float4 f) {
    T v[4] = {from_f32<T>(f.x), from_f32<T>(f.y), from_f32<T>(f.z), from_f32<T>(f.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

// One tile of 128 x BN per cluster, its K blocks divided over the cluster's
// CTAs.  Each CTA's partial tile goes from TMEM to its shared memory (where the
// operand ring was); then each CTA adds one slice of the columns over the
// cluster, in rank order, and finishes it.
template <class T, int BN>
__global__ void __launch_bounds__(GT_NT, 1)
    gemm_split_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const TcArgs g) {
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
        tc::tmem_alloc(&tmem_slot, BN);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t taddr = tmem_slot;
    volatile int* fail = &s_fail;

    if (warp == 0) {
        if (lane == 0) {  // ---- TMA producer
            int i = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb, ++i) {
                const int st = i % Ring::N;
                if (!(ok = tc::mbar_wait_or_fail(&empty[st], ((i / Ring::N) & 1) ^ 1, fail))) break;
                unsigned char *sa = ring + st * Ring::STAGE, *sb = sa + Ring::A;
                tc::mbar_arrive_expect_tx(&full[st], Ring::STAGE);
                if (g.a_mn) {
                    for (int c = 0; c < GT_M / 64; ++c)
                        tc::tma_load_2d(sa + c * 8192, &ta, &full[st], m0 + c * 64, kb * GT_K);
                } else {
                    tc::tma_load_2d(sa, &ta, &full[st], kb * GT_K, m0);
                }
                if (g.b_mn) {
                    for (int c = 0; c < BN / 64; ++c)
                        tc::tma_load_2d(sb + c * 8192, &tb, &full[st], n0 + c * 64, kb * GT_K);
                } else {
                    tc::tma_load_2d(sb, &tb, &full[st], kb * GT_K, n0);
                }
            }
            if (!ok)  // copies in flight land before the block ends
                for (int j = i > Ring::N ? i - Ring::N : 0; j < i; ++j)
                    tc::mbar_wait(&full[j % Ring::N], (j / Ring::N) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {  // ---- MMA issuer
            bool ok = true;
            int i = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++i) {
                const int st = i % Ring::N;
                if (!(ok = tc::mbar_wait_or_fail(&full[st], (i / Ring::N) & 1, fail))) break;
                tc::fence_after_sync();
                const unsigned char *sa = ring + st * Ring::STAGE, *sb = sa + Ring::A;
                const uint64_t da = g.a_mn ? tc::desc_mnmajor_sw128(sa, 8192) : tc::desc_kmajor_sw128(sa);
                const uint64_t db = g.b_mn ? tc::desc_mnmajor_sw128(sb, 8192) : tc::desc_kmajor_sw128(sb);
                const uint32_t ka = g.a_mn ? 128 : 2, kbs = g.b_mn ? 128 : 2;  // 16 k, in 16-byte units
#pragma unroll
                for (int kk = 0; kk < GT_K / 16; ++kk)
                    tc::umma_bf16(taddr, da + ka * kk, db + kbs * kk, g.idesc, (i | kk) != 0);
                tc::umma_commit(&empty[st]);
            }
            if (ok) tc::umma_commit(&acc_full);
        }
    } else {  // ---- epilogue warps: TMEM -> partial tile in shared memory
        const int q4 = warp & 3, half = (warp - 2) >> 2;
        const bool ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&acc_full, 0, fail));
        tc::fence_after_sync();
        float* row = part + (q4 * 32 + lane) * LDP;
#pragma unroll 1
        for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
            float v[32];
            tc::tmem_ld_32x32(taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)c, v);
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
        tc::tmem_dealloc(taddr, BN);
    }

    const int slice = BN / S, per_row = slice / 4;
    const uint32_t pbase = tc::smem_u32(part);
    for (int i = tid; i < GT_M * per_row; i += GT_NT) {
        const int r = i / per_row, c = rank * slice + (i - r * per_row) * 4;
        const int row = m0 + r, col = n0 + c;
        if (row >= g.m || col >= g.n) continue;
        const uint32_t at = pbase + (uint32_t)(r * LDP + c) * 4;
        float4 z = *reinterpret_cast<const float4*>(part + r * LDP + c);
        if (S > 1) {
            z = ld_cluster_f4(at, 0);
            for (int s = 1; s < S; ++s) {
                const float4 v = ld_cluster_f4(at, s);
                z.x += v.x;
                z.y += v.y;
                z.z += v.z;
                z.w += v.w;
            }
        }
        if (g.vec && col + 4 <= g.n) {
            const Epilogue& e = g.e;
            if (e.bias) {
                const float4 b = load4(static_cast<const T*>(e.bias) + col);
                z.x += b.x;
                z.y += b.y;
                z.z += b.z;
                z.w += b.w;
            }
            if (e.pre) store4(static_cast<T*>(e.pre) + row * e.ldp + col, z);
            float4 y = make_float4(activate(z.x, e.act), activate(z.y, e.act), activate(z.z, e.act),
                                   activate(z.w, e.act));
            if (e.residual) {
                const float4 b = load4(static_cast<const T*>(e.residual) + row * e.ldr + col);
                y.x += b.x;
                y.y += b.y;
                y.z += b.z;
                y.w += b.w;
            }
            store4(static_cast<T*>(e.y) + row * e.ldy + col, y);
        } else {
            const float v[4] = {z.x, z.y, z.z, z.w};
            for (int j = 0; j < 4 && col + j < g.n; ++j) epilogue_store<T>(g.e, row, col + j, v[j]);
        }
    }
    if (S > 1) cluster_sync();  // a peer may still read this CTA's partial tile
}

// ---- host side ---------------------------------------------------------------

// Operand of `rows` rows (unit stride along k: [rows][k], else [k][rows]).
static int operand_map(CUtensorMap* m, int dtype, const void* p, long long rows, long long k, long long ld, bool mn,
                       int box_rows) {
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[2] = {(cuuint64_t)(mn ? rows : k), (cuuint64_t)(mn ? k : rows)};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)(mn ? GT_K : box_rows)};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(m, dtype == FG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FG_OK;
}

// Instruction descriptor, kind::f16: f32 accumulators, M = 128.
static uint32_t instr_desc(int dtype, int n, bool a_mn, bool b_mn) {
    const uint32_t t = dtype == FG_DTYPE_BF16 ? 1 : 0;
    return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(GT_M >> 4) << 24);
}

bool tc_gemm_fits(const void* a, const void* b, const GemmShape& g) {
    const long long lda = g.ak == 1 ? g.am : g.ak, ldb = g.bk == 1 ? g.bn : g.bk;
    return aligned(a, 16) && aligned(b, 16) && lda % 8 == 0 && ldb % 8 == 0 && g.k > 0 && g.m < (1ll << 31) - 512 &&
           g.n < (1ll << 31) - 512 && g.k < (1ll << 31) - 512;
}

template <class T, int BN>
static int launch_split(int dtype, const void* a, const void* b, const GemmShape& s, TcArgs g, cudaStream_t st) {
    CUtensorMap ta, tb;
    int rc = operand_map(&ta, dtype, a, s.m, s.k, g.a_mn ? s.ak : s.am, g.a_mn, GT_M);
    if (!rc) rc = operand_map(&tb, dtype, b, s.n, s.k, g.b_mn ? s.bk : s.bn, g.b_mn, BN);
    if (rc) return rc;
    g.idesc = instr_desc(dtype, BN, g.a_mn, g.b_mn);
    g.nt = (g.n + BN - 1) / BN;
    const long long ctas = (long long)g.mt * g.nt * g.split;
    FG_REQUIRE(ctas <= 0x7fffffffll, "%d x %d outputs: too many tiles", g.m, g.n);
    auto kernel = &gemm_split_kernel<T, BN>;
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

int tc_gemm(int dtype, const void* a, const void* b, const GemmShape& s, const Epilogue& e, cudaStream_t st) {
    TcArgs g{};
    g.m = (int)s.m;
    g.n = (int)s.n;
    g.kt = (int)((s.k + GT_K - 1) / GT_K);
    g.mt = (int)((s.m + GT_M - 1) / GT_M);
    g.a_mn = s.ak != 1;
    g.b_mn = s.bk != 1;
    g.e = e;
    g.vec = aligned(e.y, 8) && e.ldy % 4 == 0 && (!e.bias || aligned(e.bias, 8)) &&
            (!e.pre || (aligned(e.pre, 8) && e.ldp % 4 == 0)) &&
            (!e.residual || (aligned(e.residual, 8) && e.ldr % 4 == 0));
    // The tile width and the split that finish first by this estimate of SM cycles:
    // a K block's MMAs, the tile's start and end, and the exchange of a split tile.
    const int sms = std::max(1, device_attr(cudaDevAttrMultiProcessorCount));
    int best_n = 256;
    double best = 1e300;
    for (int bn : {256, 128, 64}) {
        const long long tiles = (long long)g.mt * ((g.n + bn - 1) / bn);
        const double block = bn == 256 ? 520 : bn == 128 ? 280 : 200;
        for (int sp : {1, 2, 4, 8}) {
            if (sp > g.kt) break;
            const double waves = (double)((tiles * sp + sms - 1) / sms);
            const double cost = waves * ((g.kt + sp - 1) / sp * block + 3000 + 12 * bn) + (sp > 1 ? 1000 + 100 * sp : 0);
            if (cost < best) {
                best = cost;
                best_n = bn;
                g.split = sp;
            }
        }
    }
#define FG_SPLIT(T)                                                       \
    (best_n == 256   ? launch_split<T, 256>(dtype, a, b, s, g, st)        \
     : best_n == 128 ? launch_split<T, 128>(dtype, a, b, s, g, st)        \
                     : launch_split<T, 64>(dtype, a, b, s, g, st))
    return dtype == FG_DTYPE_F16 ? FG_SPLIT(__half) : FG_SPLIT(__nv_bfloat16);
#undef FG_SPLIT
}

}  // namespace fg
