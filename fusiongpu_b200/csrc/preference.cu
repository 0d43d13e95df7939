// preference.cu -- paired preference loss over an index's raw vectors.
//
// Policy pi(d | q) = softmax over documents of the search score s(q, d); in a
// ratio of two documents of one query the normaliser cancels, so the log ratio
// of pair (d+, d-) against the reference query r is, with u = q - r,
//   inner product:  z = beta u . (d+ - d-)
//   squared L2:     z = 2 beta u . (d+ - d-)         (the norms cancel)
// and without a reference u = q, for L2 u = q - (d+ + d-) / 2.  The product
// with the difference is taken as written, which loses nothing to cancellation
// of four large scores.  loss = (1-e) softplus(-z) + e softplus(z), d loss / d z =
// e - sigmoid(-z), dz / dq = k beta (d+ - d-).
//
// Bound by memory: two document rows a pair, gathered from anywhere in the base,
// each read once -- the difference stays in registers until the loss's derivative
// is known, then joins the query's gradient.  A block takes one query; each group
// of G threads (8, 32, 128 or 512, by the row's length) takes every (threads / G)-th
// pair and keeps u and its share of the gradient in registers, the rows of its next
// pair being loaded meanwhile; at the end the block adds the groups' shares in their
// order.  Rows of 256 columns to 3 KB go to the second kernel below.  Measured: 10,000
// queries of 16 pairs, documents of 128 f32 72 us (2.3 TB/s), of 768 f16 179 us (2.7
// TB/s, second kernel), 32 queries of 10 pairs of 128 bytes 5.5 us.
#include <algorithm>

#include "adapter_common.cuh"
#include "packed.cuh"
#include "tc_common.cuh"

namespace fg {

constexpr int PREF_MAX_DIM = 16384;

struct PrefArgs {
    const void *q, *ref, *base;
    const int64_t* offsets;
    const int32_t *pos, *neg;
    const float* weights;
    float *losses, *margins;
    void* dq;
    long long nbase, n_pairs, ldq, ldr, lddq;
    int nq, dim, l2, dtype;
    int wide, qwide;  // document rows and query rows start on 16-byte boundaries
    float k, smooth;  // k = beta (IP) or 2 beta (L2)
};

template <class B, int VEC>
struct Piece {
    B v[VEC];
};

template <class B, int VEC>
__device__ __forceinline__ void load_piece(Piece<B, VEC>& c, const B* p, int wide) {
    constexpr int BYTES = VEC * sizeof(B);
    if (BYTES == 16 && wide) {
        uint4 u;
        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                     : "l"(p));
        *reinterpret_cast<uint4*>(c.v) = u;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) c.v[i] = p[i];
    }
}

template <int G>
__device__ __forceinline__ float pref_group_sum(float v, float* s) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (G <= 32) return v;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) v += s[w];
    return v;
}

// Loss of margin z, and d loss / d z times k: the factor of w (d+ - d-) in the gradient.
__device__ __forceinline__ float pair_value(const PrefArgs& g, float z) {
    // (1 - e) max(-z, 0) + e max(z, 0), one of them: no infinity less another at infinite margins
    const float line = z < 0.0f ? (g.smooth - 1.0f) * z : g.smooth > 0.0f ? g.smooth * z : 0.0f;
    return line + log1pf(expf(-fabsf(z)));
}
__device__ __forceinline__ float pair_slope(const PrefArgs& g, float z) {
    const float e = expf(-fabsf(z));
    return (g.smooth - __fdividef(z >= 0.0f ? e : 1.0f, 1.0f + e)) * g.k;  // smooth - sigmoid(-z)
}

// Pairs before the first query's and after the last one's are masked ones: 0, by `nt`
// threads of the blocks that hold these queries.
__device__ __forceinline__ void mask_outside(const PrefArgs& g, long long i, long long p0, long long p1, int tid, int nt) {
    auto clear = [&](long long from, long long to) {
        for (long long p = from + tid; p < to; p += nt) {
            g.losses[p] = 0.0f;
            if (g.margins) g.margins[p] = 0.0f;
        }
    };
    if (i == 0) clear(0, p0);
    if (i == g.nq - 1) clear(p1, g.n_pairs);
}

// VEC elements of a query row.
template <class T, int VEC>
__device__ __forceinline__ void load_query(float* f, const T* p, int wide) {
    alignas(16) T v[VEC];
    constexpr int BYTES = VEC * sizeof(T);
    if (wide && BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if (wide && BYTES == 8) {
        *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f32(v[i]);
}

template <class T, class B, int VEC, int NCH, int G>
__global__ void __launch_bounds__(512) preference_kernel(const PrefArgs g) {
    constexpr int E = NCH * VEC;
    constexpr bool AHEAD = E <= 24;  // registers for the next pair's rows
    const int GROUPS = G >= 128 ? 1 : blockDim.x / G;
    extern __shared__ float sm[];  // GROUPS > 1: one gradient row per group
    __shared__ float s[16];
    const int gl = threadIdx.x % G, group = threadIdx.x / G;
    const bool mid = g.l2 && !g.ref;
    struct Pair {
        Piece<B, VEC> a[NCH], b[NCH];
        float w;
        bool fine;
    };
    struct Ids {
        int a, b;
        float w;
    };
    for (long long i = blockIdx.x; i < g.nq; i += gridDim.x) {
        const long long p0 = min(max((long long)g.offsets[i], 0ll), g.n_pairs);
        const long long p1 = min(max((long long)g.offsets[i + 1], p0), g.n_pairs);
        mask_outside(g, i, p0, p1, threadIdx.x, blockDim.x);
        auto ids_of = [&](long long p) {
            Ids d = {-1, -1, 1.0f};
            if (p < p1) {
                d.a = g.pos[p];
                d.b = g.neg[p];
                if (g.weights) d.w = g.weights[p];
            }
            return d;
        };
        auto fetch = [&](Pair& x, const Ids& d) {
            x.fine = d.a >= 0 && d.a < g.nbase && d.b >= 0 && d.b < g.nbase;
            if (!x.fine) return;
            x.w = d.w;
            const B* up = static_cast<const B*>(g.base) + (long long)d.a * g.dim;
            const B* dn = static_cast<const B*>(g.base) + (long long)d.b * g.dim;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int j = (c * G + gl) * VEC;
                if (j < g.dim) {
                    load_piece<B, VEC>(x.a[c], up + j, g.wide);
                    load_piece<B, VEC>(x.b[c], dn + j, g.wide);
                }
            }
        };
        Pair cur, next;
        Ids ids = ids_of(p0 + group);
        if (AHEAD) {
            fetch(next, ids);
            ids = ids_of(p0 + group + GROUPS);
        }
        const T* q = static_cast<const T*>(g.q) + i * g.ldq;
        const T* r = g.ref ? static_cast<const T*>(g.ref) + i * g.ldr : nullptr;
        float u[E], acc[E];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int j = (c * G + gl) * VEC;
            float x[VEC], y[VEC];
            if (j < g.dim) {
                load_query<T, VEC>(x, q + j, g.qwide);
                if (r) load_query<T, VEC>(y, r + j, g.qwide);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                u[c * VEC + e] = j < g.dim ? x[e] - (r ? y[e] : 0.0f) : 0.0f;
                acc[c * VEC + e] = 0.0f;
            }
        }
        // every group of a warp stays in the loop as long as one of its pairs exists
        const int first = G > 32 ? group : group - (threadIdx.x % 32) / G;
        for (long long p = p0 + group, w0 = p0 + first; w0 < p1; p += GROUPS, w0 += GROUPS) {
            if (AHEAD) {
                cur = next;
                fetch(next, ids);
                ids = ids_of(p + 2 * GROUPS);
            } else {
                fetch(cur, ids);
                ids = ids_of(p + GROUPS);
            }
            float t = 0.0f;
            if (cur.fine) {
#pragma unroll
                for (int c = 0; c < NCH; ++c)
                    if ((c * G + gl) * VEC < g.dim) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float x = to_f32(cur.a[c].v[e]), y = to_f32(cur.b[c].v[e]);
                            t = fmaf(mid ? u[c * VEC + e] - 0.5f * (x + y) : u[c * VEC + e], x - y, t);
                        }
                    }
            }
            const float z = pref_group_sum<G>(t, s) * g.k;
            if (cur.fine) {
                if (gl == 0) {
                    g.losses[p] = pair_value(g, z);
                    if (g.margins) g.margins[p] = z;
                }
                const float coef = pair_slope(g, z) * cur.w;
#pragma unroll
                for (int c = 0; c < NCH; ++c)
                    if ((c * G + gl) * VEC < g.dim) {
#pragma unroll
                        for (int x = 0; x < VEC; ++x)
                            acc[c * VEC + x] = fmaf(coef, to_f32(cur.a[c].v[x]) - to_f32(cur.b[c].v[x]), acc[c * VEC + x]);
                    }
            } else if (gl == 0 && p < p1) {
                g.losses[p] = 0.0f;
                if (g.margins) g.margins[p] = 0.0f;
            }
        }
        if (!g.dq) continue;
        T* dq = static_cast<T*>(g.dq) + i * g.lddq;
        if (G >= 128) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int j = (c * G + gl) * VEC + e;
                    if (j < g.dim) dq[j] = from_f32<T>(acc[c * VEC + e]);
                }
        } else {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int j = (c * G + gl) * VEC + e;
                    if (j < g.dim) sm[group * g.dim + j] = acc[c * VEC + e];
                }
            __syncthreads();
            for (int j = threadIdx.x; j < g.dim; j += blockDim.x) {
                float v = 0.0f;
                for (int w = 0; w < GROUPS; ++w) v += sm[w * g.dim + j];
                dq[j] = from_f32<T>(v);
            }
            __syncthreads();
        }
    }
}

// Rows of 256 columns to 3 KB on 16-byte boundaries: a fifth warp brings them
// into a ring in shared memory by bulk copies, as many pairs ahead as the ring holds
// and on into the block's next query, which it asks into L2 before (204 us without, 179
// with), so the latency of ids and rows is paid once; a
// warp takes every fourth pair of a query.  With the copies off the warps' hands the
// instructions a pair takes bound it next: the producer's lanes issue half a ring at
// once, the arithmetic is packed in pairs of columns, and a lane writes the loss of one
// pair in 32.  Each warp has slots of its own: were a slot shared, a warp could ask for
// its next phase before the last one had come, and a phase's parity cannot tell the two
// apart.
constexpr int PS_WARPS = 4;
constexpr int PS_RING = 36 * 1024;
constexpr int PS_STAGES = 16;

// Position in a warp's slots, and the parity of its phase.
struct RingAt {
    int slot;
    uint32_t phase;
    __device__ __forceinline__ void step(int by, int slots) {  // by <= slots
        slot += by;
        if (slot >= slots) {
            slot -= slots;
            phase ^= 1;
        }
    }
};

// Columns 2k and 2k + 1 of a 16-byte piece as floats.
template <class B>
__device__ __forceinline__ uint64_t columns(const uint32_t (&w)[4], int k);
template <>
__device__ __forceinline__ uint64_t columns<float>(const uint32_t (&w)[4], int k) {
    return pair2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
}
template <>
__device__ __forceinline__ uint64_t columns<__half>(const uint32_t (&w)[4], int k) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    return pair2(f.x, f.y);
}
template <>
__device__ __forceinline__ uint64_t columns<__nv_bfloat16>(const uint32_t (&w)[4], int k) {
    return pair2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint64_t columns<uint8_t>(const uint32_t (&w)[4], int k) {
    // 2^23 + byte as a float's bits, less 2^23
    const uint32_t x = __byte_perm(w[k / 2], 0x4b000000u, (k & 1) ? 0x7542 : 0x7540);
    const uint32_t y = __byte_perm(w[k / 2], 0x4b000000u, (k & 1) ? 0x7543 : 0x7541);
    return add2(pair2(__uint_as_float(x), __uint_as_float(y)), pair2(-8388608.0f, -8388608.0f));
}

// Element j of a query row of `dtype`, VEC of them from an aligned row.
template <int VEC>
__device__ __forceinline__ void query_columns(float* f, const void* p, int dtype, long long j, int wide) {
    if (dtype == FG_DTYPE_F32)
        load_query<float, VEC>(f, static_cast<const float*>(p) + j, wide);
    else if (dtype == FG_DTYPE_F16)
        load_query<__half, VEC>(f, static_cast<const __half*>(p) + j, wide);
    else
        load_query<__nv_bfloat16, VEC>(f, static_cast<const __nv_bfloat16*>(p) + j, wide);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// MID: squared L2 without a reference, u = q - (d+ + d-) / 2.
template <class B, int NCH, bool MID>
__global__ void __launch_bounds__((PS_WARPS + 1) * 32, NCH * 16 / sizeof(B) <= 16 ? 4 : 3)
    preference_stream_kernel(const PrefArgs g, int slots, int per_block) {
    constexpr int VEC = 16 / sizeof(B), E = NCH * VEC;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ __align__(8) uint64_t full[PS_STAGES], empty[PS_STAGES];
    __shared__ float s_w[PS_STAGES];
    __shared__ int s_fine[PS_STAGES], s_issued[PS_STAGES], s_fail;  // s_issued: parity of the slot's last copies, or -1
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = g.dim * (int)sizeof(B);
    float* part = reinterpret_cast<float*>(ring + (size_t)PS_WARPS * slots * 2 * row);  // the warps' gradients
    volatile int* fail = &s_fail;
    if (tid == 0) {
        s_fail = 0;
        for (int k = 0; k < PS_WARPS * slots; ++k) {
            tc::mbar_init(&full[k], 1);
            tc::mbar_init(&empty[k], 1);
            s_issued[k] = -1;
        }
        tc::fence_mbar_init();
    }
    __syncthreads();
    const long long i0 = (long long)blockIdx.x * per_block, i1 = min(i0 + per_block, (long long)g.nq);
    auto first_of = [&](long long i) { return min(max((long long)g.offsets[i], 0ll), g.n_pairs); };
    if (warp == PS_WARPS) {  // ---- producer: lane l the l-th pair of a batch
        // lane l brings pairs for warp l % 4: the next free slot but l / 4 of that warp
        const int depth = (slots + 1) / 2, batch = PS_WARPS * depth, w0 = (lane % PS_WARPS) * slots;
        RingAt at = {lane < batch ? lane / PS_WARPS : 0, 1};  // the slots start empty
        bool ok = true;
        const int size = g.dtype == FG_DTYPE_F32 ? 4 : 2;
        for (long long i = i0; i < i1 && ok; ++i) {
            for (int j = lane * 128; j < g.dim * size; j += 32 * 128) {  // the query comes to L2 meanwhile
                prefetch_l2(static_cast<const char*>(g.q) + i * g.ldq * size + j);
                if (g.ref) prefetch_l2(static_cast<const char*>(g.ref) + i * g.ldr * size + j);
            }
            const long long p0 = first_of(i), p1 = max(first_of(i + 1), p0);
            for (long long base = p0; base < p1; base += batch) {
                const long long p = base + lane;
                const int n = (int)min((long long)batch, p1 - base);
                bool good = true;
                if (lane < n) {
                    const int a = g.pos[p], b = g.neg[p];
                    const float w = g.weights ? g.weights[p] : 1.0f;
                    const bool fine = a >= 0 && a < g.nbase && b >= 0 && b < g.nbase;
                    const int st = w0 + at.slot;
                    good = tc::mbar_wait_or_fail(&empty[st], at.phase, fail);
                    if (good) {
                        s_w[st] = w;
                        s_fine[st] = fine;
                        if (fine) {
                            unsigned char* dst = ring + st * 2 * row;
                            tc::mbar_arrive_expect_tx(&full[st], 2 * row);
                            tc::bulk_load(dst, static_cast<const B*>(g.base) + (long long)a * g.dim, row, &full[st]);
                            tc::bulk_load(dst + row, static_cast<const B*>(g.base) + (long long)b * g.dim, row, &full[st]);
                            s_issued[st] = (int)(at.phase ^ 1);
                        } else {
                            tc::mbar_arrive(&full[st]);
                        }
                    }
                }
                ok = __all_sync(0xffffffffu, good);
                if (!ok) break;
                at.step((n - lane % PS_WARPS + PS_WARPS - 1) / PS_WARPS, slots);  // this warp's share of the n
            }
        }
        if (!ok && lane < PS_WARPS * slots && s_issued[lane] >= 0)  // copies in flight land before the block ends
            tc::mbar_wait(&full[lane], (uint32_t)s_issued[lane]);
        return;
    }
    RingAt at = {0, 0};
    const uint64_t minus = pair2(-1.0f, -1.0f), half = pair2(-0.5f, -0.5f);
    for (long long i = i0; i < i1; ++i) {
        const long long p0 = first_of(i), p1 = max(first_of(i + 1), p0);
        mask_outside(g, i, p0, p1, tid, PS_WARPS * 32);
        uint64_t u[E / 2], acc[E / 2];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int j = (c * 32 + lane) * VEC;
            float x[VEC], y[VEC];
            if (j < g.dim) {
                query_columns<VEC>(x, g.q, g.dtype, i * g.ldq + j, g.qwide);
                if (g.ref) query_columns<VEC>(y, g.ref, g.dtype, i * g.ldr + j, g.qwide);
            }
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const bool have = j < g.dim;
                u[(c * VEC + e) / 2] = pair2(have ? x[e] - (g.ref ? y[e] : 0.0f) : 0.0f,
                                             have ? x[e + 1] - (g.ref ? y[e + 1] : 0.0f) : 0.0f);
                acc[(c * VEC + e) / 2] = 0;
            }
        }
        float zk = 0.0f;  // margin of this warp's pairs: lane l the l-th of 32
        int kept = 0, masked = 0;
        auto write = [&](long long p_last) {  // losses of the `kept` pairs that end at p_last
            const long long p = p_last - (long long)(kept - 1 - lane) * PS_WARPS;
            if (lane < kept) {
                const float z = masked ? 0.0f : zk;
                g.losses[p] = masked ? 0.0f : pair_value(g, z);
                if (g.margins) g.margins[p] = z;
            }
            kept = 0;
        };
        long long p = p0 + warp;
        for (; p < p1; p += PS_WARPS) {
            const int st = warp * slots + at.slot;
            const bool ok = tc::mbar_wait_warp(&full[st], at.phase, fail);
            const bool fine = s_fine[st];
            const float wt = s_w[st];
            uint64_t d[E / 2], t[2] = {0, 0};
            if (fine) {
                const B *up = reinterpret_cast<const B*>(ring + st * 2 * row), *dn = up + g.dim;
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    const int j = (c * 32 + lane) * VEC;
                    if (j < g.dim) {
                        uint32_t a[4], b[4];
                        *reinterpret_cast<uint4*>(a) = *reinterpret_cast<const uint4*>(up + j);
                        *reinterpret_cast<uint4*>(b) = *reinterpret_cast<const uint4*>(dn + j);
#pragma unroll
                        for (int e = 0; e < VEC / 2; ++e) {
                            const int k = c * VEC / 2 + e;
                            const uint64_t x = columns<B>(a, e), y = columns<B>(b, e);
                            d[k] = fma2(y, minus, x);
                            t[k & 1] = fma2(MID ? fma2(add2(x, y), half, u[k]) : u[k], d[k], t[k & 1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&empty[st]);
            at.step(1, slots);
            float t0, t1;
            unpair2(add2(t[0], t[1]), t0, t1);
            float z = warp_sum(t0 + t1) * g.k;
            if (!ok) z = NAN;  // a wait that ran out leaves NaN, not a plausible number
            if (lane == kept) {
                zk = z;
                masked = !fine && ok;
            }
            if (++kept == 32) write(p);
            if (fine || !ok) {
                const float coef = pair_slope(g, z) * wt;
                const uint64_t c2 = pair2(coef, coef);
#pragma unroll
                for (int c = 0; c < NCH; ++c)
                    if ((c * 32 + lane) * VEC < g.dim) {
#pragma unroll
                        for (int k = c * VEC / 2; k < (c + 1) * VEC / 2; ++k) acc[k] = fma2(c2, ok ? d[k] : minus, acc[k]);
                    }
            }
        }
        if (kept) write(p - PS_WARPS);
        if (!g.dq) continue;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int j = (c * 32 + lane) * VEC;
            if (j < g.dim) {
#pragma unroll
                for (int k = c * VEC / 2; k < (c + 1) * VEC / 2; k += 2)
                    *reinterpret_cast<ulonglong2*>(part + warp * g.dim + j + 2 * k - c * VEC) =
                        make_ulonglong2(acc[k], acc[k + 1]);
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        for (int j = tid; j < g.dim; j += PS_WARPS * 32) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < PS_WARPS; ++w) v += part[w * g.dim + j];
            const long long at_j = i * g.lddq + j;
            if (g.dtype == FG_DTYPE_F32)
                static_cast<float*>(g.dq)[at_j] = v;
            else if (g.dtype == FG_DTYPE_F16)
                static_cast<__half*>(g.dq)[at_j] = from_f32<__half>(v);
            else
                static_cast<__nv_bfloat16*>(g.dq)[at_j] = from_f32<__nv_bfloat16>(v);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
    }
}

template <class B, int NCH>
static int preference_stream(const PrefArgs& g, cudaStream_t s) {
    const int row = g.dim * (int)sizeof(B), slots = std::min(PS_STAGES, std::max(PS_WARPS, PS_RING / (2 * row))) / PS_WARPS;
    const int smem = PS_WARPS * slots * 2 * row + PS_WARPS * g.dim * (int)sizeof(float);
    auto kernel = g.l2 && !g.ref ? &preference_stream_kernel<B, NCH, true> : &preference_stream_kernel<B, NCH, false>;
    if (smem > 40 * 1024) FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(kernel), smem));
    // 32 blocks in turn on each SM even out queries of unlike length (10,000 queries of 16
    // pairs on average: 179 us, with 16 186, with 8 192, with 3 266)
    const int sms = std::max(1, device_attr(cudaDevAttrMultiProcessorCount));
    const int per_block = std::max(1, std::min(16, g.nq / (32 * sms)));
    kernel<<<(g.nq + per_block - 1) / per_block, (PS_WARPS + 1) * 32, smem, s>>>(g, slots, per_block);
    return check_launch("preference_stream_kernel");
}

template <class T, class B, int VEC, int NCH, int G>
static int preference_launch(const PrefArgs& g, cudaStream_t s) {
    // Four warps to a query; sixteen where there are few queries of many pairs each;
    // one where there are many queries of short rows (four groups of 8).
    const int sms = std::max(1, device_attr(cudaDevAttrMultiProcessorCount));
    const int nt = G >= 128 ? G : g.nq < 2 * sms && g.n_pairs / g.nq >= 64 ? 512 : G == 8 && g.nq >= 16 * sms ? 32 : 128;
    const int smem = G >= 128 ? 0 : nt / G * g.dim * (int)sizeof(float);
    if (smem > 40 * 1024)
        FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(&preference_kernel<T, B, VEC, NCH, G>), smem));
    preference_kernel<T, B, VEC, NCH, G><<<std::min(g.nq, 1 << 24), nt, smem, s>>>(g);
    return check_launch("preference_kernel");
}

template <class T, class B>
static int preference_shape(PrefArgs g, cudaStream_t s) {
    constexpr int V = 16 / sizeof(B);
    g.wide = aligned(g.base, 16);
    auto lies = [&](const void* p, long long ld) { return !p || (aligned(p, 16) && ld * sizeof(T) % 16 == 0); };
    g.qwide = g.dim % V == 0 && lies(g.q, g.ldq) && lies(g.ref, g.ldr);
    // Stream and register kernel at 10,000 queries of 16 pairs: f16 256 columns 110 and
    // 165 us, 768 179 and 448; u8 512 123 and 173; f32 128 101 and 72, 256 106 and 146,
    // 768 294 and 296, 1024 357 and 303.  Below 256 columns a warp's lanes have too few
    // to hide a pair's chain of steps; beyond 768 of f32 the ring holds too few pairs.
    const int row = g.dim * (int)sizeof(B);
    if (g.dim % V == 0 && g.wide && row >= 512 && g.dim >= 256 && g.dim <= 1024 && row <= 768 * 4) {
        if constexpr (V == 16) {
            return g.dim <= 512 ? preference_stream<B, 1>(g, s) : preference_stream<B, 2>(g, s);
        } else if constexpr (V == 8) {
            return g.dim <= 512   ? preference_stream<B, 2>(g, s)
                   : g.dim <= 768 ? preference_stream<B, 3>(g, s)
                                  : preference_stream<B, 4>(g, s);
        } else {
            return g.dim <= 256   ? preference_stream<B, 2>(g, s)
                   : g.dim <= 512 ? preference_stream<B, 4>(g, s)
                                  : preference_stream<B, 6>(g, s);
        }
    }
#define FG_PREF(VEC, NCH, G) \
    if (g.dim <= (VEC) * (NCH) * (G)) return preference_launch<T, B, VEC, NCH, G>(g, s)
    if (g.dim % V == 0) {
        if constexpr (V == 16) {
            FG_PREF(16, 1, 8);
            FG_PREF(16, 1, 32);
            FG_PREF(16, 2, 32);
            FG_PREF(16, 1, 128);
            FG_PREF(16, 2, 128);
            FG_PREF(16, 2, 512);
        } else if constexpr (V == 8) {
            FG_PREF(8, 2, 8);
            FG_PREF(8, 2, 32);
            FG_PREF(8, 3, 32);
            FG_PREF(8, 1, 128);
            FG_PREF(8, 2, 128);
            FG_PREF(8, 4, 128);
            FG_PREF(8, 4, 512);
        } else {
            FG_PREF(4, 4, 8);
            FG_PREF(4, 4, 32);
            FG_PREF(4, 2, 128);
            FG_PREF(4, 4, 128);
            FG_PREF(4, 8, 128);
            FG_PREF(4, 8, 512);
        }
    }
    FG_PREF(1, 16, 8);
    FG_PREF(1, 16, 32);
    FG_PREF(1, 8, 128);
    FG_PREF(1, 32, 128);
    return preference_launch<T, B, 1, 32, 512>(g, s);
#undef FG_PREF
}

template <class T>
static int preference_base(const PrefArgs& g, int base_dtype, cudaStream_t s) {
    switch (base_dtype) {
        case FG_DTYPE_F32: return preference_shape<T, float>(g, s);
        case FG_DTYPE_F16: return preference_shape<T, __half>(g, s);
        case FG_DTYPE_BF16: return preference_shape<T, __nv_bfloat16>(g, s);
        default: return preference_shape<T, uint8_t>(g, s);
    }
}

}  // namespace fg

using namespace fg;

extern "C" int fg_preference_loss(const fg_preference_params* p, const void* queries, const void* ref,
                                  const void* base, const int64_t* offsets, const int32_t* pos_ids,
                                  const int32_t* neg_ids, const float* weights, float* losses, float* margins,
                                  void* dq, void* stream) {
    return c_entry([&]() -> int {
        FG_REQUIRE(p, "null params");
        FG_REQUIRE(p->nq >= 0 && p->dim >= 1 && p->nbase >= 0 && p->n_pairs >= 0, "bad shape");
        FG_REQUIRE(float_dtype(p->dtype), "unknown dtype %d", p->dtype);
        FG_REQUIRE(float_dtype(p->base_dtype) || p->base_dtype == FG_DTYPE_U8, "unknown base_dtype %d",
                   p->base_dtype);
        FG_REQUIRE(p->metric == FG_METRIC_L2 || p->metric == FG_METRIC_IP, "unknown metric %d", p->metric);
        FG_REQUIRE(p->beta > 0.0f && p->beta <= FLT_MAX, "beta %g is not a positive number", (double)p->beta);
        FG_REQUIRE(p->label_smoothing >= 0.0f && p->label_smoothing <= 0.5f, "label_smoothing %g outside [0, 0.5]",
                   (double)p->label_smoothing);
        if (p->dim > PREF_MAX_DIM) return fail(FG_ERR_UNSUPPORTED, "dim %d > %d", p->dim, PREF_MAX_DIM);
        PrefArgs g{};
        g.ldq = p->query_stride ? p->query_stride : p->dim;
        g.ldr = p->ref_stride ? p->ref_stride : p->dim;
        g.lddq = p->dq_stride ? p->dq_stride : p->dim;
        FG_REQUIRE(g.ldq >= p->dim && g.ldr >= p->dim && g.lddq >= p->dim, "row stride below dim");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (p->nq == 0) {  // no query holds a pair
            if (losses && p->n_pairs) FG_CUDA_TRY(cudaMemsetAsync(losses, 0, p->n_pairs * sizeof(float), s));
            if (margins && p->n_pairs) FG_CUDA_TRY(cudaMemsetAsync(margins, 0, p->n_pairs * sizeof(float), s));
            return FG_OK;
        }
        FG_REQUIRE(queries && offsets, "null buffer");
        FG_REQUIRE(p->n_pairs == 0 || (pos_ids && neg_ids && losses), "null buffer");
        FG_REQUIRE(p->nbase == 0 || base, "null base");
        g.q = queries;
        g.ref = ref;
        g.base = base;
        g.offsets = offsets;
        g.pos = pos_ids;
        g.neg = neg_ids;
        g.weights = weights;
        g.losses = losses;
        g.margins = margins;
        g.dq = dq;
        g.nbase = p->nbase;
        g.n_pairs = p->n_pairs;
        g.nq = p->nq;
        g.dim = p->dim;
        g.dtype = p->dtype;
        g.l2 = p->metric == FG_METRIC_L2;
        g.k = (g.l2 ? 2.0f : 1.0f) * p->beta;
        g.smooth = p->label_smoothing;
        return p->dtype == FG_DTYPE_F32   ? preference_base<float>(g, p->base_dtype, s)
               : p->dtype == FG_DTYPE_F16 ? preference_base<__half>(g, p->base_dtype, s)
                                          : preference_base<__nv_bfloat16>(g, p->base_dtype, s);
    });
}
