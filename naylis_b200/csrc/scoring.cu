// Token log probabilities of logits rows: the log probability of a given token,
// the distribution's entropy, its top alternatives, and their gradient.
//
// With y = x / T, m = max y, Z = sum e^(y-m):
//   logprob(t) = y_t - m - ln Z,   H = ln Z - sum (y-m) e^(y-m) / Z
// and, for upstream gradients g (logprob), h (entropy), a_k (alternatives), with
// p_j = e^(y_j-m) / Z and G = g + sum a_k:
//   dx_j = (1/T) (g 1(j=t) + sum_k a_k 1(j=i_k) - p_j (G + h (ln p_j + H)))
// stats keeps (m, Z, ln Z, H) of each row in fp32 for the backward. A masked
// logit (-inf) has probability 0 and gradient 0; a row that holds a NaN or +inf,
// or nothing but -inf, has NaN everywhere, as its softmax has.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace mom {

namespace {

constexpr int kThreads = 256;
constexpr float kNaN = __builtin_nanf("");

template <int DT>
__device__ __forceinline__ float logit(const void *row, int64_t j) {
    using T = typename Elem<DT>::T;
    return Elem<DT>::load(static_cast<const T *>(row), j);
}

// A total order over (value descending, index ascending) as one unsigned key:
// greater key = earlier. -0 counts as 0, every NaN as greater than +inf.
__device__ __forceinline__ uint64_t rank_key(float x, int j) {
    uint32_t b = __float_as_uint(x + 0.0f);
    if (x != x) b = 0x7fffffffu;
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<uint64_t>(b) << 32) | (0xffffffffu - static_cast<uint32_t>(j));
}
__device__ __forceinline__ int rank_index(uint64_t key) {
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}

__device__ __forceinline__ float block_sum(float v, float *s) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) t += s[w];
    return t;
}
__device__ __forceinline__ float block_max(float v, float *s) {
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = s[0];
    for (int w = 1; w < kThreads / 32; ++w) t = fmaxf(t, s[w]);
    return t;
}

template <int DT>
__global__ void __launch_bounds__(kThreads)
logprobs_fwd_kernel(const void *__restrict__ logits, int64_t ld, const int64_t *__restrict__ targets, int64_t R, int V,
                    int64_t ignore, float inv_t, int top, float *__restrict__ logprob, float *__restrict__ entropy,
                    float *__restrict__ top_lp, int64_t *__restrict__ top_idx, float4 *__restrict__ stats) {
    __shared__ float s[kThreads / 32];
    __shared__ unsigned long long best;
    const int64_t r = blockIdx.x;
    const void *row = static_cast<const typename Elem<DT>::T *>(logits) + r * ld;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < V; j += kThreads) m = fmaxf(m, logit<DT>(row, j));
    m = block_max(m, s);
    float z = 0.0f, t = 0.0f;
    for (int j = threadIdx.x; j < V; j += kThreads) {
        const float y = (logit<DT>(row, j) - m) * inv_t, e = expf(y);
        z += e;
        t += e * fmaxf(y, -1e4f);      // 0 for a masked logit
    }
    z = block_sum(z, s);
    t = block_sum(t, s);
    const float lz = logf(z), H = lz - t / z;
    if (threadIdx.x == 0) {
        const int64_t tok = targets[r];
        float lp = 0.0f;
        if (tok != ignore) lp = tok >= 0 && tok < V ? (logit<DT>(row, tok) - m) * inv_t - lz : kNaN;
        logprob[r] = lp;
        entropy[r] = H;
        if (stats) stats[r] = make_float4(m, z, lz, H);
    }
    uint64_t below = ~0ull;
    for (int k = 0; k < top; ++k) {
        uint64_t mine = 0;
        for (int j = threadIdx.x; j < V; j += kThreads) {
            const uint64_t key = rank_key(logit<DT>(row, j), j);
            if (key < below && key > mine) mine = key;
        }
        __syncthreads();
        if (threadIdx.x == 0) best = 0;
        __syncthreads();
        atomicMax(&best, static_cast<unsigned long long>(mine));
        __syncthreads();
        below = best;
        if (threadIdx.x == 0) {
            const int j = rank_index(below);
            top_idx[r * top + k] = j;
            top_lp[r * top + k] = (logit<DT>(row, j) - m) * inv_t - lz;
        }
    }
}

template <int DT>
__global__ void __launch_bounds__(kThreads)
logprobs_bwd_kernel(const void *__restrict__ logits, int64_t ld, const int64_t *__restrict__ targets,
                    const float4 *__restrict__ stats, const int64_t *__restrict__ top_idx, int top,
                    const float *__restrict__ g_lp, const float *__restrict__ g_ent, const float *__restrict__ g_top,
                    int64_t R, int V, int64_t ignore, float inv_t, void *__restrict__ dlogits) {
    using T = typename Elem<DT>::T;
    const int64_t r = blockIdx.x;
    const void *row = static_cast<const T *>(logits) + r * ld;
    T *drow = static_cast<T *>(dlogits) + r * V;
    const float4 st = stats[r];
    const int64_t tok = targets[r];
    float g = g_lp && tok != ignore ? g_lp[r] : 0.0f;
    if (tok != ignore && (tok < 0 || tok >= V)) g = kNaN;
    const float h = g_ent ? g_ent[r] : 0.0f;
    float G = g;
    for (int k = 0; g_top && k < top; ++k) G += g_top[r * top + k];
    for (int j = threadIdx.x; j < V; j += kThreads) {
        const float y = (logit<DT>(row, j) - st.x) * inv_t, p = expf(y) / st.y;
        float d = -p * (G + h * (fmaxf(y, -1e4f) - st.z + st.w));
        if (j == tok) d += g;
        for (int k = 0; g_top && k < top; ++k)
            if (top_idx[r * top + k] == j) d += g_top[r * top + k];
        Elem<DT>::store(drow, j, d * inv_t);
    }
}

}  // namespace

cudaError_t launch_logprobs_fwd(const void *logits, int dt, int64_t ld, const int64_t *targets, int64_t R, int V,
                                int64_t ignore, float inv_t, int top, float *logprob, float *entropy, float *top_lp,
                                int64_t *top_idx, float *stats, cudaStream_t st) {
    auto go = [&](auto kernel) {
        kernel<<<static_cast<unsigned>(R), kThreads, 0, st>>>(logits, ld, targets, R, V, ignore, inv_t, top, logprob,
                                                              entropy, top_lp, top_idx,
                                                              reinterpret_cast<float4 *>(stats));
    };
    if (dt == MOM_BF16) go(logprobs_fwd_kernel<MOM_BF16>);
    else go(logprobs_fwd_kernel<MOM_F32>);
    count_launch();
    return cudaGetLastError();
}

cudaError_t launch_logprobs_bwd(const void *logits, int dt, int64_t ld, const int64_t *targets, const float *stats,
                                const int64_t *top_idx, int top, const float *g_lp, const float *g_ent,
                                const float *g_top, int64_t R, int V, int64_t ignore, float inv_t, void *dlogits,
                                cudaStream_t st) {
    auto go = [&](auto kernel) {
        kernel<<<static_cast<unsigned>(R), kThreads, 0, st>>>(logits, ld, targets,
                                                              reinterpret_cast<const float4 *>(stats), top_idx, top,
                                                              g_lp, g_ent, g_top, R, V, ignore, inv_t, dlogits);
    };
    if (dt == MOM_BF16) go(logprobs_bwd_kernel<MOM_BF16>);
    else go(logprobs_bwd_kernel<MOM_F32>);
    count_launch();
    return cudaGetLastError();
}

}  // namespace mom
