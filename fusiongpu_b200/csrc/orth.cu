// orth.cu -- the orthogonal factor of a matrix, approached by a polynomial iteration.
//
//   X = G / (|G|_F + eps);  a number of times  A = X X^T,  B = b A + c A^2,  X = a X + B X
//
// (K. Jordan and others, "Muon: An optimizer for hidden layers in neural networks", 2024,
// whose coefficients are the default; from the smaller side: for more rows than columns A =
// X^T X and X = a X + X B, without a transposition in memory: the operands' layouts say which
// index runs along k).  Each step maps the singular values s to a s + b s^3 + c s^5 and
// leaves the singular vectors.
//
// Matrices between the products are held as two float16 planes, x = h + 2^-11 l, 22 bits
// of the significand or 2^-36, and a product is the three plane products that reach 2^-22
// of it, with fp32 sums: the iteration multiplies what an operand's rounding leaves by up
// to a^steps, and with one float16 plane the result was off by 2.4e-3 of its norm, with
// one bfloat16 plane by 1.8e-2, with two by 1.1e-6 to 2.4e-6 (float32 throughout: 1.2e-6 to
// 3.5e-6; four of 2048 x 1024 1.1e-6 and 3.1e-6).  Singular values stay of order one, so
// that float16's range holds them.
//
// The tensor cores cut their sums, always towards zero: 1,024 k in one accumulator, and a I
// as part of Y in X = Y X (or the completed square c (A + b / 2c)^2, which spares B's
// addend), left 1.4e-5 of float32 results.  So a X and b A are added behind the products,
// and sums are taken from the accumulators after ORTH_RUN blocks of 64 k and added in
// fp32.
#include <algorithm>
#include <type_traits>

#include "adapter_common.cuh"
#include "packed.cuh"
#include "tc_common.cuh"

namespace fg {

constexpr int OT_M = 128, OT_K = 64;
constexpr int LOW_SHIFT = 11;  // h + 2^-11 l
constexpr int ORTH_RUN = 2;    // K blocks (128 k) that an accumulator sums

// Two values, on the instructions for two.  What is past float16's range becomes NaN.
__device__ __forceinline__ uint64_t both(float c) { return pair2(c, c); }
__device__ __forceinline__ void planes_of(uint64_t v, __half2& h, __half2& l) {
    constexpr float up = 1 << LOW_SHIFT;
    float a, b;
    unpair2(v, a, b);
    h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    unpair2(fma2(pair2(f.x, f.y), both(-up), mul2(v, both(up))), a, b);  // exact
    l = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void planes_of(float v0, float v1, __half2& h, __half2& l) { planes_of(pair2(v0, v1), h, l); }
__device__ __forceinline__ uint64_t value_of(__half2 h, __half2 l) {
    const float2 a = __half22float2(h), b = __half22float2(l);
    return fma2(pair2(b.x, b.y), both(1.0f / (1 << LOW_SHIFT)), pair2(a.x, a.y));
}

// ---- |G|_F and the first X ----------------------------------------------------------
//
// Squares are added in 64 bits, in an order that depends on the shape alone: a warp takes
// runs of OI_COLS columns of a row, every so many of them; the blocks of the second
// launch add the blocks' sums again.  Both are bound by memory.
constexpr int ORTH_PARTS = 592, OI_NT = 256, OI_WARPS = OI_NT / 32, OI_COLS = 1024;

struct OrthIn {
    const void* g;
    double* part;  // [batch][ORTH_PARTS]
    __half* x;     // [batch][2 planes][rows][ld]; NULL: `out` instead
    void* out;
    long long row_stride, batch_stride, ld;
    int rows, cols, batch, parts, runs;  // runs of a row
    int wide;                            // G's rows start on 16 bytes
    float eps;
};

// VEC elements of a row from column c on, zeros behind its end.
template <class T, int VEC>
__device__ __forceinline__ void orth_load(T (&v)[VEC], const T* row, int c, int cols, int wide) {
    if (wide && c + VEC <= cols) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(row + c);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = c + i < cols ? row[c + i] : from_f32<T>(0.0f);
    }
}

template <class T>
__global__ void __launch_bounds__(OI_NT) orth_norm_kernel(const OrthIn g) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ double s[OI_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* p = static_cast<const T*>(g.g) + blockIdx.y * g.batch_stride;
    const int items = g.rows * g.runs;  // at most 2^15 rows of 32 runs
    double sum = 0.0;
    for (int i = blockIdx.x * OI_WARPS + warp; i < items; i += g.parts * OI_WARPS) {
        const int row = i / g.runs, c0 = (i - row * g.runs) * OI_COLS, c1 = min(c0 + OI_COLS, g.cols);
        const T* r = p + row * g.row_stride;
#pragma unroll 4
        for (int c = c0 + lane * VEC; c < c1; c += 32 * VEC) {
            alignas(16) T v[VEC];
            orth_load<T, VEC>(v, r, c, c1, g.wide);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const double d = (double)to_f32(v[j]);
                sum = fma(d, d, sum);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < OI_WARPS; ++w) sum += s[w];
        g.part[blockIdx.y * ORTH_PARTS + blockIdx.x] = sum;
    }
}

template <class T>
__global__ void __launch_bounds__(OI_NT) orth_scale_kernel(const OrthIn g) {
    constexpr int VEC = 8;  // of a plane's 16 bytes
    constexpr int IN = 16 / sizeof(T);
    __shared__ double s[OI_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double sum = 0.0;
    for (int i = threadIdx.x; i < g.parts; i += OI_NT) sum += g.part[blockIdx.y * ORTH_PARTS + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s[warp] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < OI_WARPS; ++w) sum += s[w];
    const double inv = 1.0 / (sqrt(sum) + (double)g.eps);
    const T* p = static_cast<const T*>(g.g) + blockIdx.y * g.batch_stride;
    const long long plane = g.rows * g.ld;
    const int items = g.rows * g.runs;
    for (int i = blockIdx.x * OI_WARPS + warp; i < items; i += gridDim.x * OI_WARPS) {
        const int row = i / g.runs, c0 = (i - row * g.runs) * OI_COLS, c1 = min(c0 + OI_COLS, g.cols);
        const T* r = p + row * g.row_stride;
        for (int c = c0 + lane * VEC; c < c1; c += 32 * VEC) {
            alignas(16) T v[VEC / IN][IN];
#pragma unroll
            for (int k = 0; k < VEC / IN; ++k) orth_load<T, IN>(v[k], r, c + k * IN, c1, g.wide);
            float f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = (float)((double)to_f32(v[j / IN][j % IN]) * inv);
            if (g.x) {
                alignas(16) __half h[VEC], l[VEC];
#pragma unroll
                for (int j = 0; j < VEC; j += 2)
                    planes_of(f[j], f[j + 1], *reinterpret_cast<__half2*>(h + j), *reinterpret_cast<__half2*>(l + j));
                __half* x = g.x + 2 * blockIdx.y * plane + row * g.ld + c;
                *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(h);
                *reinterpret_cast<uint4*>(x + plane) = *reinterpret_cast<const uint4*>(l);
            } else {
                T* o = static_cast<T*>(g.out) + ((long long)blockIdx.y * g.rows + row) * g.cols + c;
                for (int j = 0; j < VEC; ++j)
                    if (c + j < c1) o[j] = from_f32<T>(f[j]);
            }
        }
    }
}

// ---- products ------------------------------------------------------------------------
//
// D(m, n) = beta (sum over k of P(m, k) Q(n, k)) + alpha C(m, n).  A 128 x BN tile a
// cluster, its K blocks divided over the cluster's CTAs, partial tiles added through
// distributed shared memory.  A stage of the ring holds both planes of both operands for
// 64 k, which three products share: h h' into one accumulator, h l' and l h' into
// another, that counts 2^-11 of it.  The epilogue warps take the first one's sums into
// registers after each run; the next run's products of l come first, behind which that
// hides.
//
// SYM: D is symmetric.  Tiles above the diagonal are left out; an element below it is
// written to both its places.
//
// The products of one call follow one another by a few microseconds each, so a kernel
// starts while the one before it ends (griddepcontrol): barriers, tensor memory and
// tensor maps are ready when that one's results are.
struct OrthArgs {
    int kt, mt, nt, m, n, tiles;  // tiles of a matrix
    int p_mn, q_mn;               // the operand's unit stride is along its rows
    int split;
    int sym, vec;                 // vec: `out` allows 4-column stores
    float alpha, beta;
    const __half* c;              // NULL: none
    __half* d;                    // NULL: `out`
    void* out;                    // [batch][m][n]
    long long ldc, ldd;
    uint32_t idesc;
};

// DEEP: twice the stages, for products whose blocks have an SM each.
template <int BN, bool DEEP>
struct OrthRing {
    static constexpr int A = 2 * OT_M * OT_K * 2, B = 2 * BN * OT_K * 2, STAGE = A + B;
    static constexpr int N = BN == 128 ? 3 : DEEP ? 4 : 2;       // 2: two blocks to an SM
    static constexpr int COLS = 2 * BN;                          // of TMEM: h h', and the others
    // warps that empty the accumulators; threads: a block with the SM to itself has eight more
    // warps for its finish
    static constexpr int WARPS = 8, NT = BN == 64 && DEEP ? 576 : 320;
};

template <class T, int BN, bool SPLIT, bool DEEP>
__global__ void __launch_bounds__(OrthRing<BN, DEEP>::NT, BN == 64 && !DEEP ? 2 : 1)
    orth_product_kernel(const __grid_constant__ CUtensorMap tp, const __grid_constant__ CUtensorMap tq, const __grid_constant__ OrthArgs g) {
    using Ring = OrthRing<BN, DEEP>;
    constexpr int NT = Ring::NT, LDP = BN + 4;  // partial row: 4 floats of padding keep 16-byte stores off each other's banks
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t full[Ring::N], empty[Ring::N], acc_full, acc_empty;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* ring = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~static_cast<uintptr_t>(1023));
    float* part = reinterpret_cast<float*>(ring);
    const int S = SPLIT ? g.split : 1, rank = SPLIT ? (int)tc::cluster_rank() : 0;
    const int tile = (int)(blockIdx.x / (unsigned)S), b = tile / g.tiles;
    int t = tile - b * g.tiles, mi = 0;
    if (g.sym) {  // row tiles hold the column tiles up to the diagonal
        for (int in_row; t >= (in_row = min(g.nt, ((mi + 1) * OT_M + BN - 1) / BN)); ++mi) t -= in_row;
    } else {
        mi = t / g.nt;
        t -= mi * g.nt;
    }
    const int m0 = mi * OT_M, n0 = t * BN;
    const int kb0 = (int)((long long)g.kt * rank / S), kb1 = (int)((long long)g.kt * (rank + 1) / S);
    const int runs = (kb1 - kb0 + ORTH_RUN - 1) / ORTH_RUN;

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
        tc::mbar_init(&acc_empty, Ring::WARPS);
        tc::fence_mbar_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&tmem_slot, Ring::COLS);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t taddr = tmem_slot;
    volatile int* fail = &s_fail;
    // the next kernel's blocks may come: this block holds its tensor memory
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the last kernel's results are in memory

    // The finishing pass: W columns a position, two positions a thread and round, their
    // addends a round ahead, the first one's before the products.  A cluster's exchange waits
    // for distributed shared memory (a tile of 128 x 64, four CTAs, finished in 2 us), of which
    // a round asks for three peers at once; alone, instructions count, and 16-byte stores (with
    // 16 warps 1.1 us, with ten 1.5; four positions a thread are no faster).
    constexpr int W = SPLIT ? 4 : 8, U = 2;
    using Wide = typename std::conditional<W == 8, uint4, uint2>::type;
    const int slice = BN / S, shift = __ffs(slice / W) - 1;  // columns, and the logarithm of a row's positions
    const long long c_plane = g.m * g.ldc, d_plane = g.m * g.ldd;
    auto place = [&](int i, int& r, int& c) {
        r = i >> shift;
        c = (i - (r << shift)) * W;
        return r < OT_M && m0 + r < g.m && n0 + rank * slice + c < g.n;
    };
    Wide next_h[U], next_l[U];
    auto addends = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int r, c;
            if (!g.c || !place(i0 + u * NT, r, c)) continue;
            const __half* p = g.c + 2 * b * c_plane + (m0 + r) * g.ldc + n0 + rank * slice + c;  // rows hold a multiple of 8 elements
            next_h[u] = *reinterpret_cast<const Wide*>(p);
            next_l[u] = *reinterpret_cast<const Wide*>(p + c_plane);
        }
    };
    int lost = 0;
    if (warp > 0) addends(tid);  // the producer's behind its work: its fence waits for loads

    if (warp == 0) {
        if (tc::elect_one()) {  // ---- TMA producer
            asm volatile("fence.proxy.async.global;" ::: "memory");  // operands written by ordinary stores
            bool ok = true;
            int i = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++i) {
                const int st = i % Ring::N, k = kb * OT_K;
                ok = tc::mbar_wait_or_fail(&empty[st], ((i / Ring::N) & 1) ^ 1, fail);
                if (!ok) break;
                unsigned char *sa = ring + st * Ring::STAGE, *sb = sa + Ring::A;
                tc::mbar_arrive_expect_tx(&full[st], Ring::STAGE);
                if (g.p_mn) {
                    for (int c = 0; c < OT_M / 64; ++c) tc::tma_load_3d(sa + c * 16384, &tp, &full[st], m0 + c * 64, k, 2 * b);
                } else {
                    tc::tma_load_3d(sa, &tp, &full[st], k, m0, 2 * b);
                }
                if (g.q_mn) {
                    for (int c = 0; c < BN / 64; ++c) tc::tma_load_3d(sb + c * 16384, &tq, &full[st], n0 + c * 64, k, 2 * b);
                } else {
                    tc::tma_load_3d(sb, &tq, &full[st], k, n0, 2 * b);
                }
            }
            if (!ok)  // copies in flight land before the block ends
                for (int j = i > Ring::N ? i - Ring::N : 0; j < i; ++j) tc::mbar_wait(&full[j % Ring::N], (j / Ring::N) & 1);
        }
        __syncwarp();
        addends(tid);
    } else if (warp == 1) {
        // ---- MMA issuer: the warp stays together, one elected lane issues
        bool ok = true;
        // planes lie one behind the other: whole (K-major), or in each chunk of 64 rows
        const uint32_t pa = (g.p_mn ? 8192 : OT_M * 128) / 16, pb = (g.q_mn ? 8192 : BN * 128) / 16;
        const uint64_t da0 = g.p_mn ? tc::desc_mnmajor_sw128(ring, 16384) : tc::desc_kmajor_sw128(ring);
        const uint64_t db0 = g.q_mn ? tc::desc_mnmajor_sw128(ring + Ring::A, 16384) : tc::desc_kmajor_sw128(ring + Ring::A);
        const uint32_t ka = g.p_mn ? 128 : 2, kq = g.q_mn ? 128 : 2;  // 16 k, in 16-byte units
        for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
            const int st = i % Ring::N;
            ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&full[st], (i / Ring::N) & 1, fail));
            if (!ok) break;
            tc::fence_after_sync();
            const uint64_t da = da0 + st * (Ring::STAGE / 16), db = db0 + st * (Ring::STAGE / 16);
            const bool run = i % ORTH_RUN == 0;
            if (tc::elect_one()) {
#pragma unroll
                for (int kk = 0; kk < OT_K / 16; ++kk) {
                    tc::umma_bf16(taddr, da + ka * kk, db + kq * kk + pb, g.idesc, (i | kk) != 0);
                    tc::umma_bf16(taddr, da + ka * kk + pa, db + kq * kk, g.idesc, 1);
                }
            }
            __syncwarp();
            if (run && i > 0) {  // the last run's sums have been taken
                ok = __all_sync(0xffffffffu, tc::mbar_wait_or_fail(&acc_empty, (i / ORTH_RUN - 1) & 1, fail));
                if (!ok) break;
                tc::fence_after_sync();
            }
            if (tc::elect_one()) {
#pragma unroll
                for (int kk = 0; kk < OT_K / 16; ++kk)
                    tc::umma_bf16(taddr + BN, da + ka * kk, db + kq * kk, g.idesc, !run || kk != 0);
                tc::umma_commit(&empty[st]);
                if (kb + 1 == kb1 || (i + 1) % ORTH_RUN == 0) tc::umma_commit(&acc_full);
            }
            __syncwarp();
        }
    } else if (warp < 2 + Ring::WARPS) {  // ---- epilogue warps: TMEM -> partial tile in shared memory
        constexpr int COLUMNS = BN / (Ring::WARPS / 4), G = COLUMNS / 32;  // of a warp
        const int q4 = warp & 3, c0 = ((warp - 2) >> 2) * COLUMNS;
        float* row = part + (q4 * 32 + lane) * LDP;
        const uint32_t src = taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)c0;
        bool ok = true;
        float sum[G][32];
        for (int r = 0; r < runs; ++r) {
            ok = tc::mbar_wait_warp(&acc_full, r & 1, fail) && ok;
            tc::fence_after_sync();
#pragma unroll
            for (int c = 0; c < G; ++c) {
                float v[32];
                tc::tmem_ld_32x32(src + (uint32_t)(BN + 32 * c), v);
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[c][j] = r ? sum[c][j] + v[j] : v[j];
            }
            tc::fence_before_sync();
            __syncwarp();
            if (tc::elect_one()) tc::mbar_arrive(&acc_empty);
        }
#pragma unroll
        for (int c = 0; c < G; ++c) {
            float v[32];
            tc::tmem_ld_32x32(src + (uint32_t)(32 * c), v);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = fmaf(v[j], 1.0f / (1 << LOW_SHIFT), sum[c][j]);
#pragma unroll
            for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<float4*>(row + c0 + 32 * c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
        lost = !ok;
        tc::fence_before_sync();
    }
    if (__syncthreads_or(lost)) {  // a wait that ran out leaves NaN, not a plausible number, once no copy is under way to the ring
        for (int i = tid; i < OT_M * LDP; i += NT) part[i] = NAN;
        __syncthreads();
    }
    if (SPLIT) tc::cluster_sync();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(taddr, Ring::COLS);
    }

    static_assert((OT_M * LDP + OT_M * BN) * 4 <= Ring::N * Ring::STAGE, "the tile, and for SYM its transposed copy, fit the ring");
    uint32_t* turned = reinterpret_cast<uint32_t*>(part + OT_M * LDP);  // SYM: the slice transposed, h and l in one word,
    auto turn = [](int c, int r) { return c * OT_M + ((r + c / W * 4) & (OT_M - 1)); };  // turned on by 4 rows every W columns
    const uint32_t pbase = tc::smem_u32(part);
    for (int i0 = tid; i0 < OT_M << shift; i0 += U * NT) {
        int r[U], cc[U];
        bool in[U];
        alignas(16) float v[U][W];
        Wide ch[U], cl[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ch[u] = next_h[u];
            cl[u] = next_l[u];
            in[u] = place(i0 + u * NT, r[u], cc[u]);
            if (!in[u]) continue;
            const float* own = part + r[u] * LDP + rank * slice + cc[u];
#pragma unroll
            for (int j = 0; j < W; j += 4) *reinterpret_cast<float4*>(&v[u][j]) = *reinterpret_cast<const float4*>(own + j);
        }
        addends(i0 + U * NT);
        if constexpr (SPLIT) {
            for (int s0 = 1; s0 < S; s0 += 3) {
                float4 x[U][3];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int s = 0; s < 3; ++s)
                        if (in[u] && s0 + s < S)
                            x[u][s] = tc::ld_cluster_f4(pbase + (uint32_t)(r[u] * LDP + rank * slice + cc[u]) * 4, (rank + s0 + s) & (S - 1));
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int s = 0; s < 3; ++s)
                        if (in[u] && s0 + s < S) {
                            v[u][0] += x[u][s].x;
                            v[u][1] += x[u][s].y;
                            v[u][2] += x[u][s].z;
                            v[u][3] += x[u][s].w;
                        }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!in[u]) continue;
            const int row = m0 + r[u], col = n0 + rank * slice + cc[u];
            uint64_t z[W / 2];
#pragma unroll
            for (int j = 0; j < W / 2; ++j) z[j] = mul2(pair2(v[u][2 * j], v[u][2 * j + 1]), both(g.beta));
            if (g.c) {
#pragma unroll
                for (int j = 0; j < W / 2; ++j)
                    z[j] = fma2(both(g.alpha), value_of(reinterpret_cast<const __half2*>(&ch[u])[j], reinterpret_cast<const __half2*>(&cl[u])[j]), z[j]);
            }
            if (g.d) {
                alignas(16) __half h[W], l[W];
#pragma unroll
                for (int j = 0; j < W; j += 2) planes_of(z[j / 2], *reinterpret_cast<__half2*>(h + j), *reinterpret_cast<__half2*>(l + j));
                __half* p = g.d + 2 * b * d_plane + row * g.ldd + col;
                if (!g.sym || col + W - 1 <= row) {  // elements past the last column lie in the row's padding
                    *reinterpret_cast<Wide*>(p) = *reinterpret_cast<const Wide*>(h);
                    *reinterpret_cast<Wide*>(p + d_plane) = *reinterpret_cast<const Wide*>(l);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (col + j <= row) {
                            p[j] = h[j];
                            p[d_plane + j] = l[j];
                        }
                }
                if (g.sym) {
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        turned[turn(cc[u] + j, r[u])] = (uint32_t)__half_as_ushort(h[j]) | (uint32_t)__half_as_ushort(l[j]) << 16;
                }
            } else {
                T* p = static_cast<T*>(g.out) + ((long long)b * g.m + row) * g.n + col;
#pragma unroll
                for (int j = 0; j < W; j += 2) unpair2(z[j / 2], v[u][j], v[u][j + 1]);
#pragma unroll
                for (int k = 0; k < W; k += 4) {
                    if (g.vec && col + k < g.n) {
                        alignas(16) T o[4] = {from_f32<T>(v[u][k]), from_f32<T>(v[u][k + 1]), from_f32<T>(v[u][k + 2]), from_f32<T>(v[u][k + 3])};
                        if constexpr (sizeof(T) == 4)
                            *reinterpret_cast<uint4*>(p + k) = *reinterpret_cast<const uint4*>(o);
                        else
                            *reinterpret_cast<uint2*>(p + k) = *reinterpret_cast<const uint2*>(o);
                    } else {
#pragma unroll
                        for (int j = k; j < k + 4; ++j)
                            if (col + j < g.n) p[j] = from_f32<T>(v[u][j]);
                    }
                }
            }
        }
    }
    if (SPLIT) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // this block has read its peers' partial tiles: nothing of its own to show them
    if (g.sym) {  // a lane takes four rows, which become neighbouring columns; what is past the last one lies in the padding
        __syncthreads();
        for (int i = tid; i < slice * (OT_M / 4); i += NT) {
            const int c = i / (OT_M / 4), r = i % (OT_M / 4) * 4, row = m0 + r, col = n0 + rank * slice + c;
            if (col > row + 3 || col >= g.n || row >= g.m) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(turned + turn(c, r));
            const uint2 h = make_uint2(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.z, x.w, 0x5410));
            const uint2 l = make_uint2(__byte_perm(x.x, x.y, 0x7632), __byte_perm(x.z, x.w, 0x7632));
            __half* p = g.d + 2 * b * d_plane + col * g.ldd + row;
            if (col <= row) {
                *reinterpret_cast<uint2*>(p) = h;
                *reinterpret_cast<uint2*>(p + d_plane) = l;
            } else {  // on the diagonal
                const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 1; j < 4; ++j)
                    if (row + j >= col) {
                        p[j] = __ushort_as_half((unsigned short)v[j]);
                        p[d_plane + j] = __ushort_as_half((unsigned short)(v[j] >> 16));
                    }
            }
        }
    }
    if (SPLIT) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // a peer may still read this CTA's partial tile
}

// ---- up to 128 on the smaller side: the whole iteration in one launch --------------------
//
// A block holds 256 columns of X (rows, where they lie that way) in shared memory as the
// tensor cores read them: chunks of 64 columns, 128 rows of 128 bytes, 128-byte swizzle, a
// row of X an index of the smaller side.  The same chunk is a K-major operand of X X^T and
// an MN-major one of B X.  A product's epilogue writes the next one's operand in place.
//
// Up to 256 on the longer side one block does; up to 2,048 a cluster of two, four or eight,
// whose parts of A meet in the workspace (L2 carries them faster than distributed shared
// memory): each block adds a slice of them and writes its planes, of which all take a
// copy.  B is worked out by every block for itself, B X is its own.  Bound by the chain of
// three products and three epilogues a step, 9.4 us for 128 x 256 in one block (products
// 2.0, 1.2 and 1.9).
constexpr int OS_NT = 512, OS_SIDE = 128, OS_FAR = 256, OS_CHUNK = 128 * 128, OS_MOST = 8;  // OS_FAR: of a block; blocks
constexpr int OS_X = 4 * OS_CHUNK, OS_Y = 2 * OS_CHUNK;  // bytes of a plane
constexpr int OS_SMEM = 2 * OS_X + 2 * OS_Y + 1024;

struct OrthSmall {
    const void* g;
    void* out;
    long long row_stride, batch_stride;
    int rows, cols, steps, wide, split;  // wide: G's rows start on 16 bytes; split: blocks a matrix
    float a, b, c, eps;
    double* sums;         // split > 1: [batch][split]
    float4* part;         // [batch][split][columns of A / 4][128]
    unsigned char* image; // [batch][2 planes of Y]
};

static_assert(OS_SIDE * OS_SIDE / 4 / OS_NT == OS_MOST, "pieces of A that a thread adds");
__device__ __forceinline__ float4 os_add(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

__device__ __forceinline__ uint32_t os_at(int row, int col) {  // byte of 8 elements from col on
    return (uint32_t)((col >> 6) * OS_CHUNK + row * 128 + (((col & 63) * 2) ^ ((row & 7) << 4)));
}

template <class T>
__global__ void __launch_bounds__(OS_NT, 1) orth_small_kernel(const OrthSmall g) {
    extern __shared__ __align__(1024) unsigned char dsmem[];
    __shared__ __align__(8) uint64_t done, copied;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_fail;
    __shared__ double s_sum[OS_NT / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* xs = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* ys = xs + 2 * OS_X;
    const bool tall = g.rows > g.cols;
    const int S = g.split, rank = S > 1 ? (int)tc::cluster_rank() : 0, matrix = (int)(blockIdx.x / (unsigned)S);
    const int side = tall ? g.cols : g.rows, whole = tall ? g.rows : g.cols, chunks_of_all = (whole + 63) / 64;
    const int chunk0 = chunks_of_all * rank / S, f0 = chunk0 * 64;  // this block's part of the longer side
    const int sc = (side + 63) / 64, fc = chunks_of_all * (rank + 1) / S - chunk0, far = min(whole - f0, fc * 64);
    const T* in = static_cast<const T*>(g.g) + matrix * g.batch_stride + (tall ? f0 * g.row_stride : (long long)f0);

    if (tid == 0) {
        s_fail = 0;
        tc::mbar_init(&done, 1);
        tc::mbar_init(&copied, 1);
        tc::fence_mbar_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&tmem_slot, 512);
        tc::tmem_relinquish();
    }
    // G is read once, 64 elements a thread: |G|_F, then the planes of X
    constexpr int PIECES = OS_SIDE * OS_FAR / 8 / OS_NT;
    const int pieces = OS_SIDE * fc * 8;  // eight elements of an index of the smaller side
    auto piece_of = [&](int k, int& r, int& c) {
        const int i = k * OS_NT + tid;
        r = tall ? i & (OS_SIDE - 1) : i / (fc * 8);  // neighbouring lanes on neighbouring columns of memory
        c = (tall ? i / OS_SIDE : i % (fc * 8)) * 8;
        return i < pieces;
    };
    float v[PIECES][8];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        int r, c;
        const bool in_x = piece_of(k, r, c) && r < side;
        if (!tall && g.wide && in_x && c + 8 <= far) {
            alignas(16) T t[8];
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                reinterpret_cast<uint4*>(t)[j] = reinterpret_cast<const uint4*>(in + r * g.row_stride + c)[j];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = to_f32(t[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[k][j] = in_x && c + j < far ? to_f32(in[tall ? (c + j) * g.row_stride + r : r * g.row_stride + c + j]) : 0.0f;
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fma((double)v[k][j], (double)v[k][j], sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t taddr = tmem_slot;
    volatile int* fail = &s_fail;
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < OS_NT / 32; ++w) sum += s_sum[w];
    if (S > 1) {
        if (tid == 0) g.sums[matrix * S + rank] = sum;
        tc::cluster_sync();
        sum = 0.0;
        for (int r = 0; r < S; ++r) sum += __ldcg(g.sums + matrix * S + r);
    }
    const double inv = 1.0 / (sqrt(sum) + (double)g.eps);
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        int r, c;
        if (!piece_of(k, r, c)) continue;
        alignas(16) __half h[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2)
            planes_of((float)((double)v[k][j] * inv), (float)((double)v[k][j + 1] * inv), *reinterpret_cast<__half2*>(h + j),
                      *reinterpret_cast<__half2*>(l + j));
        const uint32_t at = os_at(r, c);
        *reinterpret_cast<uint4*>(xs + at) = *reinterpret_cast<const uint4*>(h);
        *reinterpret_cast<uint4*>(xs + OS_X + at) = *reinterpret_cast<const uint4*>(l);
    }

    const uint32_t idesc = (1u << 4) | ((uint32_t)(OT_M >> 4) << 24);  // f16 operands, f32 accumulators
    const int q4 = warp & 3, part = warp >> 2;                         // lanes of TMEM, columns
    uint32_t phase = 0;
    bool ok = true;
    // A wait that another warp's failure ended early is taken again by itself: neither products
    // nor copies are left under way at the block's end, and what was waited for in vain is NaN.
    auto landed = [&](uint64_t* bar, uint32_t parity) {
        if (tc::mbar_wait_warp(bar, parity, fail)) return true;
        tc::mbar_wait(bar, parity);
        __syncwarp();
        return false;
    };
    // h h' of columns [0, n) and, 256 on, h l' + l h', over `chunks` of 64 k; with `two`, the
    // second half of the chunks into columns from 128 on
    auto multiply = [&](const unsigned char* p, uint32_t p_low, const unsigned char* q, uint32_t q_low, bool q_mn, int n, int chunks, bool two) {
        tc::fence_proxy_async();  // operands written by ordinary stores
        tc::fence_before_sync();
        __syncthreads();
        tc::fence_after_sync();
        if (warp == 0) {
            const uint64_t dp = tc::desc_kmajor_sw128(p), dq = q_mn ? tc::desc_mnmajor_sw128(q, OS_CHUNK) : tc::desc_kmajor_sw128(q);
            const uint32_t id = idesc | ((uint32_t)q_mn << 16) | ((uint32_t)(n >> 3) << 17);
            if (tc::elect_one()) {
                for (int c = 0; c < chunks; ++c)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t a = dp + c * (OS_CHUNK / 16) + 2 * kk;
                        const uint64_t b = dq + (q_mn ? c * (64 * 128 / 16) + 128 * kk : c * (OS_CHUNK / 16) + 2 * kk);
                        const int later = two && 2 * c >= chunks, first = later ? (chunks + 1) / 2 : 0;
                        tc::umma_bf16(taddr + 128 * later, a, b, id, c > first || kk != 0);
                        tc::umma_bf16(taddr + 256, a, b + q_low / 16, id, (c | kk) != 0);
                        tc::umma_bf16(taddr + 256, a + p_low / 16, b, id, 1);
                    }
                tc::umma_commit(&done);
            }
            __syncwarp();
        }
        ok = landed(&done, phase) && ok;
        phase ^= 1;
        tc::fence_after_sync();
    };
    // 32 columns of a product from column c on, this lane's row
    auto take = [&](float (&v)[32], int c, bool two) {
        float x[32];
        const uint32_t src = taddr + ((uint32_t)(q4 * 32) << 16) + (uint32_t)c;
        tc::tmem_ld_32x32_nowait(src, v);
        tc::tmem_ld_32x32_nowait(src + 256, x);
        tc::tmem_ld_wait(v);
        tc::tmem_ld_wait(x);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = ok ? fmaf(x[j], 1.0f / (1 << LOW_SHIFT), v[j]) : NAN;
        if (two) {
            tc::tmem_ld_32x32(src + 128, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += x[j];
        }
    };
    // v = scale v + w times the matrix's own columns from c on
    auto add = [&](float (&v)[32], float scale, float w, const unsigned char* from, uint32_t low, int row, int c) {
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
            alignas(16) __half2 h[4], l[4];
            const uint32_t at = os_at(row, c + j);
            *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(from + at);
            *reinterpret_cast<uint4*>(l) = *reinterpret_cast<const uint4*>(from + low + at);
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                unpair2(fma2(pair2(v[j + k], v[j + k + 1]), both(scale), mul2(both(w), value_of(h[k / 2], l[k / 2]))), v[j + k], v[j + k + 1]);
        }
    };
    auto put = [&](unsigned char* to, uint32_t low, const float (&v)[32], int row, int c) {
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
            alignas(16) __half h[8], l[8];
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                planes_of(v[j + k], v[j + k + 1], *reinterpret_cast<__half2*>(h + k), *reinterpret_cast<__half2*>(l + k));
            const uint32_t at = os_at(row, c + j);
            *reinterpret_cast<uint4*>(to + at) = *reinterpret_cast<const uint4*>(h);
            *reinterpret_cast<uint4*>(to + low + at) = *reinterpret_cast<const uint4*>(l);
        }
    };
    const int row = q4 * 32 + lane;
    T* out = static_cast<T*>(g.out) + (long long)matrix * g.rows * g.cols + (tall ? (long long)f0 * side : (long long)f0);
    // the result: tall, neighbouring lanes on neighbouring columns; else through shared memory,
    // eight elements where their own planes were: the first four in h's place, then l's
    auto store = [&](const float (&v)[32], int c) {
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
            if (tall) {
#pragma unroll
                for (int k = j; k < j + 8; ++k)
                    if (row < side && c + k < far) out[(long long)(c + k) * side + row] = from_f32<T>(v[k]);
            } else {
                const uint32_t at = os_at(row, c + j);
                *reinterpret_cast<float4*>(xs + at) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                *reinterpret_cast<float4*>(xs + OS_X + at) = make_float4(v[j + 4], v[j + 5], v[j + 6], v[j + 7]);
            }
        }
    };
    float4* parts = g.part + (size_t)matrix * S * sc * 16 * OS_SIDE;
    unsigned char* image = g.image + (size_t)matrix * 2 * OS_Y;
#pragma unroll 1
    for (int step = 0; step < g.steps; ++step) {
        float v[32];
        const int c0 = part * 32;
        multiply(xs, OS_X, xs, OS_X, false, sc * 64, fc, fc > 1);
        if (c0 < sc * 64) {
            take(v, c0, fc > 1);
            if (g.c == 0.0f) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= g.b;
            }
            if (S == 1) {
                put(ys, OS_Y, v, row, c0);
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                    parts[(rank * sc * 16 + (c0 + j) / 4) * OS_SIDE + row] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            }
        }
        if (S > 1) {
            tc::cluster_sync();
            // eight pieces of four columns a thread at most, all asked for at once
            const int pieces = sc * 16 * OS_SIDE, per = pieces / S, loads = (per + OS_NT - 1) / OS_NT * S;
            float4 p[OS_MOST];
#pragma unroll
            for (int k = 0; k < OS_MOST; ++k)
                if (k < loads && tid < per) p[k] = __ldcg(parts + (k & (S - 1)) * pieces + rank * per + k / S * OS_NT + tid);
#pragma unroll
            for (int k = 0; k < OS_MOST; ++k) {
                if (k >= loads || tid >= per) break;
                if ((k & (S - 1)) != 0) p[k] = os_add(p[k - 1], p[k]);  // the blocks' in their order
                if (((k + 1) & (S - 1)) != 0) continue;
                alignas(8) __half h[4], l[4];
                planes_of(p[k].x, p[k].y, *reinterpret_cast<__half2*>(h), *reinterpret_cast<__half2*>(l));
                planes_of(p[k].z, p[k].w, *reinterpret_cast<__half2*>(h + 2), *reinterpret_cast<__half2*>(l + 2));
                const int i = rank * per + k / S * OS_NT + tid, col = i / OS_SIDE * 4;
                unsigned char* at = image + os_at(i & (OS_SIDE - 1), col & ~7) + (col & 4) * 2;
                *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(h);
                *reinterpret_cast<uint2*>(at + OS_Y) = *reinterpret_cast<const uint2*>(l);
            }
            tc::cluster_sync();
            if (tid == 0) {
                asm volatile("fence.proxy.async.global;" ::: "memory");  // written by ordinary stores
                tc::mbar_arrive_expect_tx(&copied, 2 * sc * OS_CHUNK);
                for (int k = 0; k < 2 * sc; ++k) {
                    const int at = (k & 1) * OS_Y + (k >> 1) * OS_CHUNK;
                    tc::bulk_load(ys + at, image + at, OS_CHUNK, &copied);
                }
            }
            ok = landed(&copied, step & 1) && ok;
        }
        if (g.c != 0.0f) {
            multiply(ys, OS_Y, ys, OS_Y, false, sc * 64, sc, sc > 1);
            if (c0 < sc * 64) {
                take(v, c0, sc > 1);
                add(v, g.c, g.b, ys, OS_Y, row, c0);
                put(ys, OS_Y, v, row, c0);
            }
        }
        multiply(ys, OS_Y, xs, OS_X, true, fc * 64, sc, false);
#pragma unroll 1
        for (int c = c0; c < fc * 64; c += 128) {
            take(v, c, false);
            add(v, 1.0f, g.a, xs, OS_X, row, c);
            if (step + 1 < g.steps)
                put(xs, OS_X, v, row, c);
            else
                store(v, c);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == 1) tc::tmem_dealloc(taddr, 512);
    if (!tall)
        for (int r = warp; r < side; r += OS_NT / 32)
            for (int c = lane; c < far; c += 32)
                out[(long long)r * whole + c] = from_f32<T>(*reinterpret_cast<const float*>(xs + (c & 4 ? OS_X : 0) + os_at(r, c & ~7) + (c & 3) * 4));
}

// ---- host side -----------------------------------------------------------------------

// Matrices [batch][2 planes][rows][ld] as an operand: boxes of 64 columns of memory, both
// planes; mn: its k runs across the rows.
static int orth_map(CUtensorMap* m, const __half* p, int batch, long long rows, int cols, long long ld, bool mn, int box_rows) {
    tc::EncodeTiledFn enc = tc::encode_fn();
    if (!enc) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch * 2};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(rows * ld) * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)(mn ? OT_K : box_rows), 2};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(p), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FG_OK;
}

struct OrthPlan {
    int bn, split;
    bool deep;
};

static long long orth_tiles(long long m, long long n, int bn, bool sym) {
    const long long mt = (m + OT_M - 1) / OT_M, nt = (n + bn - 1) / bn;
    if (!sym) return mt * nt;
    long long t = 0;
    for (long long i = 0; i < mt; ++i) t += std::min(nt, ((i + 1) * OT_M + bn - 1) / bn);
    return t;
}

// The tile width and split that finish first by this estimate, in microseconds: a K block
// takes 0.75 in tiles of 64 columns, of which two blocks share an SM, 0.45 in such tiles with
// the SM and twice the stages to themselves, 0.7 in tiles of 128; what follows the products 3
// (4 with neighbours on their SMs), 2.5 and 3.7; and an exchange over the cluster, by what
// each CTA has left to finish, 1.8 of two, and of four 0.5 where results go to two places
// (SYM), else 2; with the SM to itself 0.2 and none, else 0.9 and 1.1.  Measured for 130 x 130
// to four of 2048 x 1024, each product with each choice: within 1.6 us of the best one.
// (Tiles of 256 columns, whose accumulators fill TMEM, took 95 us where these take 77: 2048 x
// 1024 from the right, four matrices.)
static OrthPlan orth_plan(long long m, long long n, long long k, int batch, bool sym) {
    const int sms = std::max(2, device_attr(cudaDevAttrMultiProcessorCount)), kb = (int)((k + OT_K - 1) / OT_K);
    OrthPlan best{128, 1, false};
    double least = 1e300;
    for (const OrthPlan& way : {OrthPlan{128, 1, false}, OrthPlan{64, 1, false}, OrthPlan{64, 1, true}}) {
        const long long tiles = orth_tiles(m, n, way.bn, sym) * batch;
        for (int sp : {1, 2, 4, 8}) {
            if (sp > kb) break;
            int slots = sp == 1 ? sms : sp == 2 ? sms / 2 : std::max(1, sp == 4 ? sms * 32 / 148 : sms * 14 / 148);
            if (way.bn == 64 && !way.deep) slots *= 2;
            const double exchange = sp == 1 ? 0.0 : sp == 8 ? 4.0 : way.deep ? (sp == 2 ? (sym ? 0.2 : 0.9) : sym ? 0.0 : 1.1)
                                                                             : (sp == 2 ? 1.8 : sym ? 0.5 : 2.0);
            const double each = (kb + sp - 1) / sp * (way.bn == 128 ? 0.7 : way.deep ? 0.45 : 0.75) +
                                (way.bn == 128 ? 3.7 : way.deep ? 2.5 : tiles * sp > sms ? 4.0 : 3.0) + exchange;
            const double cost = (double)((tiles + slots - 1) / slots) * each;
            if (cost < least) {
                least = cost;
                best = OrthPlan{way.bn, sp, way.deep};
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

// A product ready to launch: a step's are the last step's but for the buffers of X, so they
// are made once a call (each tensor map takes the host a microsecond).
struct OrthProduct {
    CUtensorMap tp, tq;
    OrthArgs g;
    OrthPlan plan;
    unsigned ctas;
};

static int make_product(const OrthOperand& p, const OrthOperand& q, const OrthArgs& args, long long k, int batch, OrthProduct& o) {
    o.plan = orth_plan(args.m, args.n, k, batch, args.sym);
    const int bn = o.plan.bn;
    int rc = orth_map(&o.tp, p.p, batch, p.rows, p.cols, p.ld, p.mn, OT_M);
    if (!rc) rc = orth_map(&o.tq, q.p, batch, q.rows, q.cols, q.ld, q.mn, bn);
    if (rc) return rc;
    OrthArgs& g = o.g;
    g = args;
    g.split = o.plan.split;
    g.kt = (int)((k + OT_K - 1) / OT_K);
    g.p_mn = p.mn;
    g.q_mn = q.mn;
    g.mt = (g.m + OT_M - 1) / OT_M;
    g.nt = (g.n + bn - 1) / bn;
    g.tiles = (int)orth_tiles(g.m, g.n, bn, g.sym);
    // kind::f16: f16 operands, f32 accumulators
    g.idesc = (1u << 4) | ((uint32_t)p.mn << 15) | ((uint32_t)q.mn << 16) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(OT_M >> 4) << 24);
    const long long ctas = (long long)g.tiles * batch * g.split;
    FG_REQUIRE(ctas <= 0x7fffffffll, "too many tiles");
    o.ctas = (unsigned)ctas;
    return FG_OK;
}

template <class T, int BN, bool DEEP>
static int launch_product(const OrthProduct& o, cudaStream_t s) {
    auto kernel = o.plan.split > 1 ? &orth_product_kernel<T, BN, true, DEEP> : &orth_product_kernel<T, BN, false, DEEP>;
    const int smem = OrthRing<BN, DEEP>::N * OrthRing<BN, DEEP>::STAGE + 1024;
    FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(o.ctas);
    cfg.blockDim = dim3(OrthRing<BN, DEEP>::NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = o.plan.split;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = o.plan.split > 1 ? 2 : 1;
    FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, o.tp, o.tq, o.g));
    return FG_OK;
}

template <class T>
static int product(const OrthProduct& o, cudaStream_t s) {
    return o.plan.bn == 128 ? launch_product<T, 128, false>(o, s)
           : o.plan.deep    ? launch_product<T, 64, true>(o, s)
                            : launch_product<T, 64, false>(o, s);
}

struct OrthWs {
    __half *x[2], *a, *b;
    double* part;
    float4* parts;
    unsigned char* image;
};

static long long orth_ld(long long cols) { return (cols + 7) / 8 * 8; }

// Blocks a matrix for the one launch above, or 0: it does not fit, or so many matrices take
// more than two rounds of clusters (74, 32 and 14 of two, four and eight blocks run at once),
// where the products one by one are as fast.
static int orth_small(const fg_orthogonalize_params* p) {
    const int far = std::max(p->rows, p->cols);
    if (p->steps == 0 || std::min(p->rows, p->cols) > OS_SIDE || far > OS_FAR * OS_MOST) return 0;
    int split = 1;
    while (far > OS_FAR * split) split *= 2;
    const int sms = std::max(2, device_attr(cudaDevAttrMultiProcessorCount));
    const int slots = split == 2 ? sms / 2 : std::max(1, split == 4 ? sms * 32 / 148 : sms * 14 / 148);
    return split == 1 || p->batch <= 2 * slots ? split : 0;
}

static size_t orth_carve(const fg_orthogonalize_params* p, void* ws, size_t bytes, OrthWs& w) {
    Carve c(ws, bytes);
    w = OrthWs{};
    const size_t side = std::min(p->rows, p->cols), batch = p->batch;
    if (const int split = orth_small(p)) {
        if (split == 1) return 0;
        w.part = c.take<double>(batch * split);
        w.parts = c.take<float4>(batch * split * ((side + 63) / 64) * 16 * OS_SIDE);
        w.image = c.take<unsigned char>(batch * 2 * OS_Y);
        return c.used;
    }
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
    const long long ldx = orth_ld(cols), lda = orth_ld(side);
    const long long row_stride = p->row_stride ? p->row_stride : cols, batch_stride = p->batch_stride ? p->batch_stride : rows * row_stride;
    const int es = sizeof(T);
    const bool wide = aligned(g, 16) && row_stride * es % 16 == 0 && (batch == 1 || batch_stride * es % 16 == 0);
    if (const int split = orth_small(p)) {
        FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(&orth_small_kernel<T>), OS_SMEM));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)batch * split);
        cfg.blockDim = dim3(OS_NT);
        cfg.dynamicSmemBytes = OS_SMEM;
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = split;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, &orth_small_kernel<T>,
                                       OrthSmall{g, out, row_stride, batch_stride, rows, cols, p->steps, wide, split, p->a, p->b, p->c,
                                                 p->eps, w.part, w.parts, w.image}));
        return FG_OK;
    }
    OrthIn in{};
    in.g = g;
    in.part = w.part;
    in.x = w.x[0];
    in.out = out;
    in.rows = rows;
    in.cols = cols;
    in.row_stride = row_stride;
    in.batch_stride = batch_stride;
    in.ld = ldx;
    in.batch = batch;
    in.eps = p->eps;
    in.runs = (cols + OI_COLS - 1) / OI_COLS;
    in.parts = (int)std::min<long long>(ORTH_PARTS, ((long long)rows * in.runs + OI_WARPS - 1) / OI_WARPS);
    in.wide = wide;
    orth_norm_kernel<T><<<dim3(in.parts, batch), OI_NT, 0, s>>>(in);
    int rc = check_launch("orth_norm_kernel");
    if (rc) return rc;
    orth_scale_kernel<T><<<dim3(in.parts, batch), OI_NT, 0, s>>>(in);
    if ((rc = check_launch("orth_scale_kernel"))) return rc;
    if (p->steps == 0) return FG_OK;
    const bool tall = rows > cols;
    OrthProduct first[2], second, third[2];  // by the buffer that X lies in
    const OrthOperand as{w.a, side, side, lda, false}, bs{p->c == 0.0f ? w.a : w.b, side, side, lda, false};
    for (int k = 0; k < std::min(2, p->steps); ++k) {
        OrthArgs a{};  // A = X X^T, or without c already B = b A
        a.m = a.n = side;
        a.sym = 1;
        a.beta = p->c == 0.0f ? p->b : 1.0f;
        a.d = w.a;
        a.ldd = lda;
        const OrthOperand xs{w.x[k], rows, cols, ldx, tall};
        if ((rc = make_product(xs, xs, a, far, batch, first[k]))) return rc;
        OrthArgs d{};  // X = a X + B X, or a X + X B
        d.m = rows;
        d.n = cols;
        d.alpha = p->a;
        d.beta = 1.0f;
        d.c = w.x[k];
        d.ldc = ldx;
        d.d = w.x[k ^ 1];
        d.ldd = ldx;
        d.out = out;
        d.vec = cols % 4 == 0 && aligned(out, 4 * es);
        const OrthOperand xk{w.x[k], rows, cols, ldx, !tall};
        if ((rc = make_product(tall ? xk : bs, tall ? bs : xk, d, side, batch, third[k]))) return rc;
    }
    if (p->c != 0.0f) {  // B = b A + c A A
        OrthArgs a{};
        a.m = a.n = side;
        a.sym = 1;
        a.alpha = p->b;
        a.beta = p->c;
        a.c = w.a;
        a.ldc = lda;
        a.d = w.b;
        a.ldd = lda;
        if ((rc = make_product(as, as, a, side, batch, second))) return rc;
    }
    for (int k = 0; k < p->steps; ++k) {
        if ((rc = product<T>(first[k & 1], s))) return rc;
        if (p->c != 0.0f && (rc = product<T>(second, s))) return rc;
        if (k + 1 == p->steps) third[k & 1].g.d = nullptr;  // to `out`
        if ((rc = product<T>(third[k & 1], s))) return rc;
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
