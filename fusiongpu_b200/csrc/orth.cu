// orth.cu -- the orthogonal factor of a matrix, approached by a polynomial iteration.
//
//   X = G / (|G|_F + eps);  a number of times  A = X X^T,  B = b A + c A^2,  X = a X + B X
//
// (from the smaller side: for more rows than columns A = X^T X and X = a X + X B, without
// a transposition in memory: the operands' layouts say which index runs along k).  Each
// step maps the singular values s to a s + b s^3 + c s^5 and leaves the singular vectors.
//
// Matrices between the products are held as two float16 planes, x = h + 2^-11 l, 22 bits
// of the significand or 2^-36, and a product is the three plane products that reach 2^-22
// of it, with fp32 sums: the iteration multiplies what an operand's rounding leaves by up
// to a^steps, and with one float16 plane the result was off by 2.4e-3 of its norm, with
// one bfloat16 plane by 1.8e-2, with two by 6e-7 (float32 throughout: 2e-6).  Singular
// values stay of order one, so that float16's range holds them.
#include <algorithm>
#include <type_traits>

#include "adapter_common.cuh"
#include "tc_common.cuh"

namespace fg {

constexpr int OT_M = 128, OT_K = 64, OT_NT = 64 + 256;
constexpr int OT_RING = 192 * 1024;
constexpr int LOW_SHIFT = 11;  // h + 2^-11 l
constexpr int ORTH_RUN = 8;    // K blocks (512 k) that an accumulator sums before the next one is taken, where TMEM allows

__device__ __forceinline__ void planes_of(float v, __half& h, __half& l) {
    h = __float2half_rn(v);
    const float f = __half2float(h);
    l = fabsf(f) <= 65504.0f ? __float2half_rn((v - f) * (float)(1 << LOW_SHIFT)) : __float2half_rn(0.0f);
}
__device__ __forceinline__ float value_of(__half h, __half l) {
    return fmaf(__half2float(l), 1.0f / (1 << LOW_SHIFT), __half2float(h));
}

// ---- |G|_F and the first X ----------------------------------------------------------
//
// Squares are added in 64 bits, in an order that depends on the shape alone: a block sums
// every ORTH_PARTS-th run of 1,024 elements, and each block of the second launch adds the
// partial sums again.  Both are bound by memory.
constexpr int ORTH_PARTS = 128, OI_NT = 256, OI_RUN = 1024;

struct OrthIn {
    const void* g;
    double* part;  // [batch][ORTH_PARTS]
    __half* x;     // planes [2][batch][rows][ld]; NULL: `out` instead
    void* out;
    long long rows, row_stride, batch_stride, ld;
    int cols, batch, parts;
    float eps;
};

template <class T>
__global__ void __launch_bounds__(OI_NT) orth_norm_kernel(const OrthIn g) {
    __shared__ double s[OI_NT / 32];
    const T* p = static_cast<const T*>(g.g) + blockIdx.y * g.batch_stride;
    const long long n = g.rows * g.cols;
    double sum = 0.0;
    for (long long r = (long long)blockIdx.x * OI_RUN; r < n; r += (long long)g.parts * OI_RUN) {
#pragma unroll
        for (int k = 0; k < OI_RUN / OI_NT; ++k) {
            const long long i = r + k * OI_NT + threadIdx.x;
            if (i < n) {
                const long long row = i / g.cols;
                const double v = (double)to_f32(p[row * g.row_stride + (i - row * g.cols)]);
                sum = fma(v, v, sum);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < OI_NT / 32; ++w) sum += s[w];
        g.part[blockIdx.y * ORTH_PARTS + blockIdx.x] = sum;
    }
}

template <class T>
__global__ void __launch_bounds__(OI_NT) orth_scale_kernel(const OrthIn g) {
    __shared__ double s;
    if (threadIdx.x < 32) {
        double sum = 0.0;
        for (int i = threadIdx.x; i < g.parts; i += 32) sum += g.part[blockIdx.y * ORTH_PARTS + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) s = 1.0 / (sqrt(sum) + (double)g.eps);
    }
    __syncthreads();
    const double inv = s;
    const T* p = static_cast<const T*>(g.g) + blockIdx.y * g.batch_stride;
    const long long plane = (long long)g.batch * g.rows * g.ld;
    for (long long i = blockIdx.x * (long long)OI_NT + threadIdx.x; i < g.rows * g.ld; i += (long long)gridDim.x * OI_NT) {
        const long long row = i / g.ld;
        const int col = (int)(i - row * g.ld);
        const float v = col < g.cols ? (float)((double)to_f32(p[row * g.row_stride + col]) * inv) : 0.0f;
        if (g.x) {
            __half h, l;
            planes_of(v, h, l);
            __half* x = g.x + blockIdx.y * g.rows * g.ld + i;
            x[0] = h;
            x[plane] = l;
        } else if (col < g.cols) {
            static_cast<T*>(g.out)[(blockIdx.y * g.rows + row) * g.cols + col] = from_f32<T>(v);
        }
    }
}

// ---- products ------------------------------------------------------------------------
//
// D(m, n) = alpha C(m, n) + beta (sum over k of P(m, k) Q(n, k)): a 128 x BN tile a
// cluster, its K blocks divided over the cluster's CTAs, partial tiles added through
// distributed shared memory, as the linear layer's products of few tiles are.
struct OrthArgs {
    int kt, mt, nt, m, n;
    int p_mn, q_mn;       // the operand's unit stride is along its rows
    int split, batch;
    float alpha, beta;
    const __half* c;      // planes, NULL: none
    __half* d;            // planes, NULL: `out`
    void* out;
    long long ldc, ldd, ldo;       // row strides
    long long c_plane, d_plane;    // from a plane to the next; a matrix to the next: m * ld
    uint32_t idesc;
};

template <int BN>
struct OrthRing {
    static constexpr int A = OT_M * OT_K * 2, B = BN * OT_K * 2, STAGE = A + B;
    static constexpr int N = OT_RING / STAGE > 8 ? 8 : OT_RING / STAGE;
};

__device__ __forceinline__ uint32_t orth_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void orth_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float4 orth_peer(uint32_t a, uint32_t rank) {
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

// Planes of the i-th of three plane products: l h, h l, h h.
__device__ __forceinline__ int orth_plane_p(int i) { return i == 0; }
__device__ __forceinline__ int orth_plane_q(int i) { return i == 1; }

template <class T, int BN>
__global__ void __launch_bounds__(OT_NT, 1)
    orth_product_kernel(const __grid_constant__ CUtensorMap tp, const __grid_constant__ CUtensorMap tq, const __grid_constant__ OrthArgs g) {
    using Ring = OrthRing<BN>;
    constexpr int LDP = BN + 4, NA = 512 / BN;
    static_assert(OT_M * LDP * 4 <= Ring::N * Ring::STAGE, "the partial tile fits the ring");
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t full[Ring::N], empty[Ring::N], acc_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* ring = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~static_cast<uintptr_t>(1023));
    float* part = reinterpret_cast<float*>(ring);
    const int S = g.split, rank = S > 1 ? (int)orth_rank() : 0;
    const int tile = (int)(blockIdx.x / (unsigned)S), b = tile / (g.mt * g.nt), t = tile - b * (g.mt * g.nt);
    const int m0 = t / g.nt * OT_M, n0 = t % g.nt * BN;
    const int kb0 = (int)((long long)g.kt * rank / S), kb1 = (int)((long long)g.kt * (rank + 1) / S);
    const int share = max(ORTH_RUN, (kb1 - kb0 + NA - 1) / NA), shares = (kb1 - kb0 + share - 1) / share;

    if (warp == 2 && tc::elect_one()) {
        tc::prefetch_map(&tp);
        tc::prefetch_map(&tq);
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
        tc::tmem_alloc(&tmem_slot, 512);
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
            for (int c0 = kb0; c0 < kb1 && ok; c0 += share)
                for (int q = 0; q < 3 && ok; ++q)
                    for (int kb = c0; kb < min(c0 + share, kb1); ++kb) {
                        const int st = i % Ring::N, k = kb * OT_K;
                        ok = tc::mbar_wait_or_fail(&empty[st], ((i / Ring::N) & 1) ^ 1, fail);
                        if (!ok) break;
                        unsigned char *sa = ring + st * Ring::STAGE, *sb = sa + Ring::A;
                        tc::mbar_arrive_expect_tx(&full[st], Ring::STAGE);
                        const int zp = orth_plane_p(q) * g.batch + b, zq = orth_plane_q(q) * g.batch + b;
                        if (g.p_mn) {
                            for (int c = 0; c < OT_M / 64; ++c) tc::tma_load_3d(sa + c * 8192, &tp, &full[st], m0 + c * 64, k, zp);
                        } else {
                            tc::tma_load_3d(sa, &tp, &full[st], k, m0, zp);
                        }
                        if (g.q_mn) {
                            for (int c = 0; c < BN / 64; ++c) tc::tma_load_3d(sb + c * 8192, &tq, &full[st], n0 + c * 64, k, zq);
                        } else {
                            tc::tma_load_3d(sb, &tq, &full[st], k, n0, zq);
                        }
                        ++i;
                    }
            if (!ok)  // copies in flight land before the block ends
                for (int j = i > Ring::N ? i - Ring::N : 0; j < i; ++j) tc::mbar_wait(&full[j % Ring::N], (j / Ring::N) & 1);
        }
    } else if (warp == 1) {
        // ---- MMA issuer: the warp stays together, one elected lane issues
        bool ok = true;
        int i = 0;
        const uint64_t da0 = g.p_mn ? tc::desc_mnmajor_sw128(ring, 8192) : tc::desc_kmajor_sw128(ring);
        const uint64_t db0 = g.q_mn ? tc::desc_mnmajor_sw128(ring + Ring::A, 8192) : tc::desc_kmajor_sw128(ring + Ring::A);
        const uint32_t ka = g.p_mn ? 128 : 2, kbs = g.q_mn ? 128 : 2;  // 16 k, in 16-byte units
        for (int c0 = kb0, acc = 0; c0 < kb1 && ok; c0 += share, ++acc) {
            const int n = (min(c0 + share, kb1) - c0) * 3;
            for (int u = 0; u < n; ++u, ++i) {
                const int st = i % Ring::N;
                ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&full[st], (i / Ring::N) & 1, fail));
                if (!ok) break;
                tc::fence_after_sync();
                const uint64_t da = da0 + st * (Ring::STAGE / 16), db = db0 + st * (Ring::STAGE / 16);
                if (tc::elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < OT_K / 16; ++kk) {
                        const uint32_t d = taddr + (uint32_t)(acc * BN);
                        if (kk == 0 && 3 * u == 2 * n)  // the products of l are done: on to h h
                            tc::umma_shifted<LOW_SHIFT>(d, da, db, g.idesc);
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
                    ok ? make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]) : make_float4(NAN, NAN, NAN, NAN);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (S > 1) orth_cluster_sync();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(taddr, 512);
    }

    const int slice = BN / S, per_row = slice / 4;
    const uint32_t pbase = tc::smem_u32(part);
    for (int i = tid; i < OT_M * per_row; i += OT_NT) {
        const int r = i / per_row, cc = rank * slice + (i - r * per_row) * 4, row = m0 + r, col = n0 + cc;
        if (row >= g.m || col >= g.n) continue;
        const uint32_t at = (uint32_t)(r * LDP + cc) * 4;
        // planes have rows of a multiple of 8 elements, zeros past the last column
        alignas(8) __half ch[4], cl[4];
        if (g.c) {
            const __half* p = g.c + ((long long)b * g.m + row) * g.ldc + col;
            *reinterpret_cast<uint2*>(ch) = *reinterpret_cast<const uint2*>(p);
            *reinterpret_cast<uint2*>(cl) = *reinterpret_cast<const uint2*>(p + g.c_plane);
        }
        float4 z = S > 1 ? orth_peer(pbase + at, rank) : *reinterpret_cast<const float4*>(reinterpret_cast<const char*>(part) + at);
        for (int s = 1; s < S; ++s) {
            const float4 v = orth_peer(pbase + at, (rank + s) & (S - 1));
            z.x += v.x;
            z.y += v.y;
            z.z += v.z;
            z.w += v.w;
        }
        float v[4] = {z.x * g.beta, z.y * g.beta, z.z * g.beta, z.w * g.beta};
        if (g.c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(g.alpha, value_of(ch[j], cl[j]), v[j]);
        }
        if (g.d) {
            alignas(8) __half h[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) planes_of(col + j < g.n ? v[j] : 0.0f, h[j], l[j]);
            __half* p = g.d + ((long long)b * g.m + row) * g.ldd + col;
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
            *reinterpret_cast<uint2*>(p + g.d_plane) = *reinterpret_cast<const uint2*>(l);
        } else {
            T* p = static_cast<T*>(g.out) + ((long long)b * g.m + row) * g.ldo + col;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < g.n) p[j] = from_f32<T>(v[j]);
        }
    }
    if (S > 1) orth_cluster_sync();  // a peer may still read this CTA's partial tile
}

// ---- host side -----------------------------------------------------------------------

// Planes [2][batch][rows][ld] as an operand of `lead` rows, its k along the memory's rows
// (lead == rows) or across them (mn).
static int orth_map(CUtensorMap* m, const __half* p, int batch, long long rows, int cols, long long ld, bool mn, int box_rows) {
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch * 2};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(rows * ld) * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)(mn ? OT_K : box_rows), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(p), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FG_OK;
}

struct OrthPlan {
    int bn, split;
};

// The tile width and split that finish first by the linear layer's estimate for products
// of few tiles (microseconds; three products a K block).
static OrthPlan orth_plan(long long m, long long n, long long k, int batch) {
    const int sms = std::max(2, device_attr(cudaDevAttrMultiProcessorCount)), kb = (int)((k + OT_K - 1) / OT_K);
    OrthPlan best{128, 1};
    double least = 1e300;
    for (int bn : {256, 128, 64}) {
        const long long tiles = (m + OT_M - 1) / OT_M * ((n + bn - 1) / bn) * batch;
        for (int sp : {1, 2, 4, 8}) {
            if (sp > kb) break;
            const int slots = sp == 1 ? sms : sp == 2 ? sms / 2 : std::max(1, sp == 4 ? sms * 32 / 148 : sms * 14 / 148);
            const double main = (kb + sp - 1) / sp * 3 * (bn == 256 ? 0.43 : bn == 128 ? 0.30 : 0.21);
            const double cost = (double)((tiles + slots - 1) / slots) * (main + 2.0 + 0.02 * bn / sp) + (sp == 8 ? 0.7 : 0.0);
            if (cost < least) {
                least = cost;
                best = OrthPlan{bn, sp};
            }
        }
    }
    return best;
}

struct OrthOperand {
    const __half* p;
    long long rows;  // as it lies
    int cols;
    long long ld;
    bool mn;
};

template <class T, int BN>
static int launch_product(const OrthOperand& p, const OrthOperand& q, OrthArgs g, cudaStream_t s) {
    CUtensorMap tp, tq;
    int rc = orth_map(&tp, p.p, g.batch, p.rows, p.cols, p.ld, p.mn, OT_M);
    if (!rc) rc = orth_map(&tq, q.p, g.batch, q.rows, q.cols, q.ld, q.mn, BN);
    if (rc) return rc;
    g.p_mn = p.mn;
    g.q_mn = q.mn;
    g.mt = (g.m + OT_M - 1) / OT_M;
    g.nt = (g.n + BN - 1) / BN;
    // kind::f16: f16 operands, f32 accumulators
    g.idesc = (1u << 4) | ((uint32_t)p.mn << 15) | ((uint32_t)q.mn << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(OT_M >> 4) << 24);
    const long long ctas = (long long)g.mt * g.nt * g.batch * g.split;
    FG_REQUIRE(ctas <= 0x7fffffffll, "too many tiles");
    auto kernel = &orth_product_kernel<T, BN>;
    const int smem = OrthRing<BN>::N * OrthRing<BN>::STAGE + 1024;
    FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(OT_NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = g.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tp, tq, g));
    return FG_OK;
}

template <class T>
static int product(const OrthOperand& p, const OrthOperand& q, OrthArgs g, long long k, cudaStream_t s) {
    const OrthPlan plan = orth_plan(g.m, g.n, k, g.batch);
    g.split = plan.split;
    g.kt = (int)((k + OT_K - 1) / OT_K);
    return plan.bn == 256   ? launch_product<T, 256>(p, q, g, s)
           : plan.bn == 128 ? launch_product<T, 128>(p, q, g, s)
                            : launch_product<T, 64>(p, q, g, s);
}

struct OrthWs {
    __half *x[2], *a, *b;
    double* part;
};

static long long orth_ld(long long cols) { return (cols + 7) / 8 * 8; }

static size_t orth_carve(const fg_orthogonalize_params* p, void* ws, size_t bytes, OrthWs& w) {
    Carve c(ws, bytes);
    w = OrthWs{};
    const size_t side = std::min(p->rows, p->cols), batch = p->batch;
    w.part = c.take<double>(batch * ORTH_PARTS);
    if (p->steps > 0) {
        for (int k = 0; k < 2; ++k)
            if (k == 0 || p->steps > 1) w.x[k] = c.take<__half>(2 * batch * p->rows * orth_ld(p->cols));
        w.a = c.take<__half>(2 * batch * side * orth_ld(side));
        w.b = c.take<__half>(2 * batch * side * orth_ld(side));
    }
    return c.used;
}

constexpr int ORTH_DIM = 32768, ORTH_BATCH = 65535;

static int orth_check(const fg_orthogonalize_params* p) {
    FG_REQUIRE(p, "null params");
    FG_REQUIRE(p->batch >= 0 && p->rows >= 1 && p->cols >= 1, "bad matrix shape");
    if (p->batch > ORTH_BATCH || p->rows > ORTH_DIM || p->cols > ORTH_DIM)
        return fail(FG_ERR_UNSUPPORTED, "a batch above %d or a dimension above %d", ORTH_BATCH, ORTH_DIM);
    FG_REQUIRE(float_dtype(p->dtype), "unknown dtype %d", p->dtype);
    FG_REQUIRE(p->steps >= 0 && p->steps <= 100, "steps must be 0 .. 100");
    FG_REQUIRE(p->eps >= 0.0f && p->eps < INFINITY, "eps must be finite and not negative");
    for (float c : {p->a, p->b, p->c}) FG_REQUIRE(fabsf(c) <= 16.0f, "coefficients must be within 16");
    FG_REQUIRE(p->row_stride == 0 || p->row_stride >= p->cols, "row stride below the row length");
    FG_REQUIRE(p->batch_stride >= 0, "negative batch stride");
    return FG_OK;
}

template <class T>
static int orthogonalize(const fg_orthogonalize_params* p, const void* g, void* out, const OrthWs& w, cudaStream_t s) {
    const int rows = p->rows, cols = p->cols, batch = p->batch, side = std::min(rows, cols), far = std::max(rows, cols);
    const long long ldx = orth_ld(cols), lda = orth_ld(side), n = (long long)rows * cols;
    OrthIn in{};
    in.g = g;
    in.part = w.part;
    in.x = w.x[0];
    in.out = out;
    in.rows = rows;
    in.cols = cols;
    in.row_stride = p->row_stride ? p->row_stride : cols;
    in.batch_stride = p->batch_stride ? p->batch_stride : rows * in.row_stride;
    in.ld = ldx;
    in.batch = batch;
    in.eps = p->eps;
    in.parts = (int)std::min<long long>(ORTH_PARTS, (n + OI_RUN - 1) / OI_RUN);
    orth_norm_kernel<T><<<dim3(in.parts, batch), OI_NT, 0, s>>>(in);
    int rc = check_launch("orth_norm_kernel");
    if (rc) return rc;
    const int blocks = (int)std::min<long long>((rows * ldx + OI_NT - 1) / OI_NT, 1024);
    orth_scale_kernel<T><<<dim3(blocks, batch), OI_NT, 0, s>>>(in);
    if ((rc = check_launch("orth_scale_kernel"))) return rc;
    const bool tall = rows > cols;
    const long long x_plane = (long long)batch * rows * ldx, a_plane = (long long)batch * side * lda;
    for (int k = 0; k < p->steps; ++k) {
        const __half* x = w.x[k & 1];
        const bool last = k + 1 == p->steps;
        OrthArgs a{};  // A = X X^T
        a.m = a.n = side;
        a.batch = batch;
        a.beta = 1.0f;
        a.d = w.a;
        a.ldd = lda;
        a.d_plane = a_plane;
        const OrthOperand xs{x, rows, cols, ldx, tall};
        if ((rc = product<T>(xs, xs, a, far, s))) return rc;
        a.alpha = p->b;  // B = b A + c A A
        a.beta = p->c;
        a.c = w.a;
        a.ldc = lda;
        a.c_plane = a_plane;
        a.d = w.b;
        const OrthOperand as{w.a, side, side, lda, false}, bs{w.b, side, side, lda, false};
        if ((rc = product<T>(as, as, a, side, s))) return rc;
        OrthArgs d{};  // X = a X + B X, or a X + X B
        d.m = rows;
        d.n = cols;
        d.batch = batch;
        d.alpha = p->a;
        d.beta = 1.0f;
        d.c = x;
        d.ldc = ldx;
        d.c_plane = x_plane;
        d.d = last ? nullptr : w.x[(k + 1) & 1];
        d.ldd = ldx;
        d.d_plane = x_plane;
        d.out = out;
        d.ldo = cols;
        const OrthOperand xk{x, rows, cols, ldx, !tall};
        if ((rc = tall ? product<T>(xk, bs, d, side, s) : product<T>(bs, xk, d, side, s))) return rc;
    }
    return FG_OK;
}

}  // namespace fg

using namespace fg;

extern "C" {

int fg_orthogonalize_workspace_size(const fg_orthogonalize_params* params, size_t* bytes) {
    return c_entry([&]() -> int {
        FG_REQUIRE(bytes, "null bytes");
        const int rc = orth_check(params);
        if (rc) return rc;
        OrthWs w;
        *bytes = orth_carve(params, nullptr, 0, w);
        return FG_OK;
    });
}

int fg_orthogonalize(const fg_orthogonalize_params* params, const void* g, void* out, void* workspace, size_t workspace_bytes,
                     void* stream) {
    return c_entry([&]() -> int {
        int rc = orth_check(params);
        if (rc) return rc;
        if (params->batch == 0) return FG_OK;
        FG_REQUIRE(g && out, "null buffer");
        OrthWs w;
        if ((rc = adapter_ws(workspace, workspace_bytes, orth_carve(params, nullptr, 0, w)))) return rc;
        orth_carve(params, workspace, workspace_bytes, w);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return params->dtype == FG_DTYPE_F32   ? orthogonalize<float>(params, g, out, w, s)
               : params->dtype == FG_DTYPE_F16 ? orthogonalize<__half>(params, g, out, w, s)
                                               : orthogonalize<__nv_bfloat16>(params, g, out, w, s);
    });
}

}  // extern "C"
