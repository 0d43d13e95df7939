// preference.cu -- paired preference loss over an index's raw vectors.
//
// Policy pi(d | q) = softmax over documents of the search score s(q, d); in a
// ratio of two documents of one query the normaliser cancels, so the log ratio
// of pair (d+, d-) against the reference query r is, with u = q - r,
//   inner product:  z = beta u . (d+ - d-)
//   squared L2:     z = 2 beta u . (d+ - d-)         (the norms cancel)
// and without a reference u = q, for L2 u = q - (d+ + d-) / 2.  The product
// with the difference is taken as written, which loses nothing to cancellation
// of four large scores.  loss = softplus(-z) + e z [= (1-e) softplus(-z) +
// e softplus(z)], d loss / d z = e - sigmoid(-z), dz / dq = k beta (d+ - d-).
#include <algorithm>

#include "adapter_common.cuh"

namespace fg {

constexpr int PREF_MAX_DIM = 16384;
constexpr int PREF_NT = 128;

struct PrefArgs {
    const void *q, *ref, *base;
    const int64_t* offsets;
    const int32_t *pos, *neg;
    const float* weights;
    float *losses, *margins;
    void* dq;
    long long nbase, n_pairs, ldq, ldr, lddq;
    int nq, dim, l2;
    float k, smooth;  // k = beta (IP) or 2 beta (L2)
};

// Block per query; u and the gradient row in shared memory, one pair at a time.
template <class T, class B>
__global__ void __launch_bounds__(PREF_NT) preference_kernel(const PrefArgs g) {
    extern __shared__ float sm[];
    __shared__ float s[PREF_NT / 32];
    float *u = sm, *acc = sm + g.dim;
    for (long long i = blockIdx.x; i < g.nq; i += gridDim.x) {
        const T* q = static_cast<const T*>(g.q) + i * g.ldq;
        const T* r = g.ref ? static_cast<const T*>(g.ref) + i * g.ldr : nullptr;
        for (int j = threadIdx.x; j < g.dim; j += PREF_NT) {
            u[j] = to_f32(q[j]) - (r ? to_f32(r[j]) : 0.0f);
            acc[j] = 0.0f;
        }
        const long long p0 = min(max((long long)g.offsets[i], 0ll), g.n_pairs);
        const long long p1 = min(max((long long)g.offsets[i + 1], p0), g.n_pairs);
        for (long long p = p0; p < p1; ++p) {
            const int a = g.pos[p], b = g.neg[p];
            const bool fine = a >= 0 && a < g.nbase && b >= 0 && b < g.nbase;
            float z = 0.0f;
            if (fine) {
                const B* dp = static_cast<const B*>(g.base) + (long long)a * g.dim;
                const B* dn = static_cast<const B*>(g.base) + (long long)b * g.dim;
                const bool mid = g.l2 && !r;
                float t = 0.0f;
                for (int j = threadIdx.x; j < g.dim; j += PREF_NT) {
                    const float x = to_f32(dp[j]), y = to_f32(dn[j]);
                    t = fmaf(mid ? u[j] - 0.5f * (x + y) : u[j], x - y, t);
                }
                z = block_sum<PREF_NT>(t, s) * g.k;
                const float e = expf(-fabsf(z));
                const float sig = (z >= 0.0f ? e : 1.0f) / (1.0f + e);  // sigmoid(-z)
                const float coef = (g.smooth - sig) * (g.weights ? g.weights[p] : 1.0f) * g.k;
                if (threadIdx.x == 0) {
                    g.losses[p] = fmaxf(-z, 0.0f) + log1pf(e) + g.smooth * z;
                    if (g.margins) g.margins[p] = z;
                }
                if (g.dq)
                    for (int j = threadIdx.x; j < g.dim; j += PREF_NT)
                        acc[j] = fmaf(coef, to_f32(dp[j]) - to_f32(dn[j]), acc[j]);
            } else if (threadIdx.x == 0) {
                g.losses[p] = 0.0f;
                if (g.margins) g.margins[p] = 0.0f;
            }
        }
        if (g.dq)
            for (int j = threadIdx.x; j < g.dim; j += PREF_NT)
                (static_cast<T*>(g.dq) + i * g.lddq)[j] = from_f32<T>(acc[j]);
    }
}

template <class T, class B>
static int preference_launch(const PrefArgs& g, cudaStream_t s) {
    const int smem = 2 * g.dim * (int)sizeof(float);
    FG_CUDA_TRY(ensure_smem(reinterpret_cast<const void*>(&preference_kernel<T, B>), smem));
    preference_kernel<T, B><<<std::min(g.nq, 1 << 20), PREF_NT, smem, s>>>(g);
    return check_launch("preference_kernel");
}

template <class T>
static int preference_base(const PrefArgs& g, int base_dtype, cudaStream_t s) {
    switch (base_dtype) {
        case FG_DTYPE_F32: return preference_launch<T, float>(g, s);
        case FG_DTYPE_F16: return preference_launch<T, __half>(g, s);
        case FG_DTYPE_BF16: return preference_launch<T, __nv_bfloat16>(g, s);
        default: return preference_launch<T, uint8_t>(g, s);
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
        if (p->nq == 0) return FG_OK;
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
        g.l2 = p->metric == FG_METRIC_L2;
        g.k = (g.l2 ? 2.0f : 1.0f) * p->beta;
        g.smooth = p->label_smoothing;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return p->dtype == FG_DTYPE_F32   ? preference_base<float>(g, p->base_dtype, s)
               : p->dtype == FG_DTYPE_F16 ? preference_base<__half>(g, p->base_dtype, s)
                                          : preference_base<__nv_bfloat16>(g, p->base_dtype, s);
    });
}
