// score_kernels.hip -- lcrc_score (include/lcrc_pipeline.h): ln p of given classes, entropy and the k best classes of every
// row of logits or posteriors.
//     l(c) = x(c) or ln x(c);  m = max x (logits), 0 (posteriors);  e(c) = exp(x(c) - m) or x(c)
//     S = sum e, T = sum e * (l - m);  ln p(c) = (l(c) - m) - ln S;  entropy = ln S - T / S
#include <cmath>

#include "ops_dev.h"

namespace phnrec {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// rising with the value, -0 and +0 alike; NaN never reaches it in a row whose result counts
__device__ __forceinline__ unsigned ordered(float x)
{
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ unsigned long long make_key(float x, int c)
{
    return ((unsigned long long)ordered(x) << 32) | (0xffffffffu - (unsigned)c);
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V *slot, Op op)
{
    for (int d = 32; d >= 1; d >>= 1) v = op(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
    for (int w = 1; w < kThreads / 64; w++) v = op(v, slot[w]);
    return v;
}

// One workgroup per row.
template <typename X, bool PROBS>
__global__ __launch_bounds__(kThreads) void score_kernel(const lcrc_score_args a)
{
    __shared__ float fslot[kThreads / 64];
    __shared__ unsigned long long kslot[kThreads / 64];
    const size_t r = blockIdx.x;
    const X *x = static_cast<const X *>(a.x) + r * (size_t)a.ld;
    const int tid = threadIdx.x, cols = a.cols;
    const auto add = [](float p, float q) { return p + q; };

    float m = -INFINITY;
    bool bad = false;
    for (int c = tid; c < cols; c += kThreads) {
        const float v = to_f32(x[c]);
        bad = bad || !(v < INFINITY) || (PROBS && !(v >= 0.0f));
        m = fmaxf(m, v);
    }
    bad = __syncthreads_or(bad);
    m = PROBS ? 0.0f : block_reduce(m, fslot, [](float p, float q) { return fmaxf(p, q); });
    float S = 0.0f, T = 0.0f;
    if (m > -INFINITY)
        for (int c = tid; c < cols; c += kThreads) {
            const float v = to_f32(x[c]);
            const float e = PROBS ? v : expf(v - m);
            S += e;
            if (e > 0.0f) T += e * (PROBS ? logf(v) : v - m);
        }
    S = block_reduce(S, fslot, add);
    T = block_reduce(T, fslot, add);
    const float ln_s = logf(S);
    const auto ln_p = [&](float v) {
        if (bad) return (float)NAN;
        if (!(S > 0.0f)) return -INFINITY;
        return (PROBS ? logf(v) : v - m) - ln_s;
    };
    if (a.entropy && tid == 0) a.entropy[r] = bad ? NAN : S > 0.0f ? ln_s - T / S : 0.0f;
    if (a.logp && tid < a.n_labels) {
        const int c = a.labels[r * a.n_labels + tid];
        a.logp[r * a.n_labels + tid] = c < 0 ? 0.0f : c >= cols ? NAN : ln_p(to_f32(x[c]));
    }
    if (!a.top_index && !a.top_logp) return;
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.k; j++) {
        unsigned long long best = 0;
        for (int c = tid; c < cols; c += kThreads) {
            const unsigned long long key = make_key(to_f32(x[c]), c);
            if (key < last && key > best) best = key;
        }
        last = block_reduce(best, kslot, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        if (tid == 0) {
            const int c = (int)(0xffffffffu - (unsigned)last);
            if (a.top_index) a.top_index[r * a.k + j] = bad ? -1 : c;
            if (a.top_logp) a.top_logp[r * a.k + j] = bad ? NAN : ln_p(to_f32(x[c]));
        }
    }
}

}  // namespace

size_t score_workspace_bytes(int, int, int) { return 0; }

hipError_t score_launch(const lcrc_score_args &a, hipStream_t stream)
{
    const auto go = [&](auto x) {
        if (a.form == LCRC_SCORE_PROBS) score_kernel<decltype(x), true><<<a.rows, kThreads, 0, stream>>>(a);
        else score_kernel<decltype(x), false><<<a.rows, kThreads, 0, stream>>>(a);
    };
    if (a.type == LCRC_T_F32) go(float());
    else if (a.type == LCRC_T_F16) go(_Float16());
    else go(__bf16());
    return hipGetLastError();
}

}  // namespace phnrec
