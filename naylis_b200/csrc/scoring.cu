// Token log probabilities of logits rows: the log probability of a given token,
// the distribution's entropy, its top alternatives, and their gradient.
//
// With y = x / T, m = max y, Z = sum e^(y-m):
//   logprob(t) = y_t - m - ln Z,   H = ln Z - sum (y-m) e^(y-m) / Z
// and, for upstream gradients g (logprob), h (entropy), a_k (alternatives), with
// p_j = e^(y_j-m) / Z and G = g + sum a_k:
//   dx_j = (1/T) (g 1(j=t) + sum_k a_k 1(j=i_k) - p_j (G + h (ln p_j + H)))
// stats keeps (m, Z, ln Z, H) of each row in fp32 for the backward (m: the reference
// that the sums are taken against, the maximum up to kSlack). A masked logit (-inf, or the
// type's lowest value next to ordinary ones) has probability 0 and gradient 0; a row that
// holds a NaN or +inf, or nothing but -inf, has NaN everywhere, as its softmax has.
//
// Bound by reading the logits (and, backward, writing their gradient). 16376 rows of
// 32000 in bf16, B200: forward 190 us, 5.5 TB/s (the special-function unit, one
// exponential an element, is 66 % busy), with 8 alternatives 247 us; backward 303 us,
// 6.9 TB/s. In fp32, 4096 rows of 32003: forward 89 us, 5.9 TB/s.
#include <algorithm>

#include "launch.h"
#include "tc_common.cuh"

namespace mom {

namespace {

constexpr float kNaN = __builtin_nanf("");
// Logits are summed as at least kFloor, which is below every reference that counts: the
// weight of a masked one is then 0, not 0 x inf. Rows whose maximum lies beyond kFar
// (nothing but masks of the type's lowest value, say) are summed by themselves.
constexpr float kFloor = -0x1.92p+99f;      // the bf16 nearest -1e30
constexpr float kFar = 1e29f;

template <int DT>
__device__ __forceinline__ float logit(const void *row, int64_t j) {
    using T = typename Elem<DT>::T;
    return Elem<DT>::load(static_cast<const T *>(row), j);
}

// A value's place in the order: -0 counts as 0, every NaN as greater than +inf; 0 is below all.
__device__ __forceinline__ uint32_t order_of(float x) {
    uint32_t b = __float_as_uint(x + 0.0f);
    if (x != x) b = 0x7fffffffu;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// (value descending, index ascending) as one key: greater = earlier.
__device__ __forceinline__ uint64_t rank_key(uint32_t order, uint32_t j) {
    return (static_cast<uint64_t>(order) << 32) | (0xffffffffu - j);
}
__device__ __forceinline__ int rank_index(uint64_t key) {
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}

// A row's 16-byte vectors, and the elements before the first and behind the last of them.
template <int DT>
struct RowSpan {
    using T = typename Elem<DT>::T;
    static constexpr int kVE = 16 / sizeof(T);
    const T *row;
    const uint4 *vec;
    int head, nvec, tail;
    __device__ __forceinline__ RowSpan(const void *base, int64_t offset, int V) {
        row = static_cast<const T *>(base) + offset;
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
        head = min(V, off ? (16 - off) / static_cast<int>(sizeof(T)) : 0);
        nvec = (V - head) / kVE;
        tail = V - head - nvec * kVE;
        vec = reinterpret_cast<const uint4 *>(row + head);
    }
    // index of the single element that thread t takes, or -1
    __device__ __forceinline__ int extra(int t) const {
        if (t < head) return t;
        return t - head < tail ? head + nvec * kVE + t - head : -1;
    }
    __device__ __forceinline__ int index(int v, int e) const { return head + v * kVE + e; }
};

template <int DT>
__device__ __forceinline__ void unpack(const uint4 &v, float (&x)[16 / sizeof(typename Elem<DT>::T)]) {
    const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == MOM_BF16) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
        } else {
            x[i] = __uint_as_float(a[i]);
        }
    }
}

// The same with values below kFloor (a masked logit's, -inf or the type's lowest, a NaN) raised to it.
template <int DT>
__device__ __forceinline__ void unpack_floor(const uint4 &v, float (&x)[16 / sizeof(typename Elem<DT>::T)]) {
    if constexpr (DT == MOM_BF16) {
        uint32_t a[4] = {v.x, v.y, v.z, v.w};
        const uint32_t floor2 = 0xf149f149u;      // kFloor, the bf16 nearest -1e30, twice
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("max.bf16x2 %0, %0, %1;\n" : "+r"(a[i]) : "r"(floor2));
        unpack<DT>(make_uint4(a[0], a[1], a[2], a[3]), x);
    } else {
        unpack<DT>(v, x);
#pragma unroll
        for (float &y : x) y = fmaxf(y, kFloor);
    }
}

// The greatest value of a vector, NaN if one is (bf16 pairs compared as they are).
template <int DT>
__device__ __forceinline__ float vec_max(const uint4 &v) {
    const uint32_t a[4] = {v.x, v.y, v.z, v.w};
    if constexpr (DT == MOM_BF16) {
        uint32_t m;
        asm("{\n .reg .b32 p, q;\n max.NaN.bf16x2 p, %1, %2;\n max.NaN.bf16x2 q, %3, %4;\n max.NaN.bf16x2 %0, p, q;\n}\n"
            : "=r"(m)
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]));
        return tc::fmax3_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u), -INFINITY);
    } else {
        return tc::fmax3_nan(__uint_as_float(a[0]), __uint_as_float(a[1]),
                             tc::fmax3_nan(__uint_as_float(a[2]), __uint_as_float(a[3]), -INFINITY));
    }
}

// One row per TPR threads (a warp, or a CTA). A thread streams its vectors once and
// sums e^(y-c) and e^(y-c) (y-c) against a reference c of its own, the maximum of its
// first kHold vectors, moved only when a later one passes it by more than kSlack (so
// the sums neither overflow nor lose digits); the row's threads rebase to the greatest
// reference at the end. A masked logit counts as kFloor, and a reference is no lower.
//
// Alternatives: the k-th greatest of the groups' maxima bounds the k-th greatest
// logit from below, so few elements reach it; the threads that hold them list them
// (reading their vectors again, from L2) and each is placed by counting the greater
// ones. Ties beyond the list's room (rows of equal logits) go through k rounds of a
// row maximum instead.
template <int TPR>
struct Team {
    static constexpr int kRows = TPR == 32 ? 4 : 1;           // rows of a CTA
    static constexpr int kThreads = TPR * kRows;
    static constexpr int kGroups = TPR == 512 ? 64 : 32;
    static constexpr int kLanes = TPR / kGroups, kShare = kGroups / kLanes;   // of a group; groups a lane compares
    static_assert(kShare % 4 == 0, "group maxima are read as 16-byte vectors");
    static constexpr int kList = TPR == 32 ? 320 : 768;       // >= 32 groups x 8 elements + head + tail
    static __device__ __forceinline__ void sync() {
        if constexpr (TPR == 32) __syncwarp();
        else __syncthreads();
    }
};

template <int TPR>
struct Scratch {
    uint32_t top[TPR / 32];            // the warps' maxima
    float2 sums[TPR / 32];
    alignas(16) uint32_t group[Team<TPR>::kGroups];
    uint32_t bound;                    // no alternative is below
    int count;
    unsigned long long best;
    uint64_t list[Team<TPR>::kList];
};

constexpr int kHold = 8;            // vectors of a thread in flight
constexpr float kSlack = 24.0f;     // log2

template <int DT, int TPR>
__global__ void __launch_bounds__(Team<TPR>::kThreads, 1024 / Team<TPR>::kThreads)
logprobs_fwd_kernel(const void *__restrict__ logits, int64_t ld, const int64_t *__restrict__ targets, int64_t R, int V,
                    int64_t ignore, float inv_t, int top, float *__restrict__ logprob, float *__restrict__ entropy,
                    float *__restrict__ top_lp, int64_t *__restrict__ top_idx, float4 *__restrict__ stats) {
    using Tm = Team<TPR>;
    constexpr int kVE = RowSpan<DT>::kVE;
    __shared__ Scratch<TPR> scratch[Tm::kRows];
    Scratch<TPR> &S = scratch[threadIdx.x / TPR];
    const int t = threadIdx.x % TPR, warp = t >> 5, lane = t & 31;
    const float c2 = inv_t * kLog2e;
    const int64_t step = static_cast<int64_t>(gridDim.x) * Tm::kRows;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * Tm::kRows + threadIdx.x / TPR; r < R; r += step) {
        const RowSpan<DT> row(logits, r * ld, V);
        const int64_t tok = targets[r];
        const int ex = row.extra(t);
        const float x_extra = ex >= 0 ? logit<DT>(row.row, ex) : -INFINITY;
        const float x_tok = tok >= 0 && tok < V ? logit<DT>(row.row, tok) : kNaN;
        // reference, s = sum 2^z and w = sum 2^z z with z = (x - ref) c2
        float ref = x_extra;
        uint64_t s2 = tc::f2(0.0f, 0.0f), w2 = s2, ref2 = s2;
        const uint64_t cc2 = tc::f2(c2, c2);
        auto rebase = [&](float to) {
            if (ref > -INFINITY) {
                const float delta = fmaxf((ref - to) * c2, -256.0f), f = tc::ex2(delta);      // f is 0 there
                w2 = tc::mul2(tc::fma2(tc::f2(delta, delta), s2, w2), tc::f2(f, f));
                s2 = tc::mul2(s2, tc::f2(f, f));
            }
            ref = to;
            ref2 = tc::f2(to, to);
        };
        auto add = [&](float xa, float xb) {      // xa, xb finite: at least kFloor
            // the difference first: it is exact near the reference, whatever that is. (x c2 - ref c2 in one step
            // leaves the rounding of ref c2 in every term, and so in ln Z: 4e-5 at logits of 1000.)
            const uint64_t z = tc::mul2(tc::sub2(tc::f2(xa, xb), ref2), cc2);
            const uint64_t e = tc::ex2_pair(z);
            s2 = tc::add2(s2, e);
            w2 = tc::fma2(e, z, w2);
        };
        if (x_extra > -INFINITY) {
            ref = -INFINITY;
            rebase(fmaxf(x_extra, kFloor));
            add(fmaxf(x_extra, kFloor), kFloor);
        }
        const float slack = kSlack / c2;
        // the batches' maxima, those of batch b, b + 4, ... in one: where the alternatives are looked for
        float bmax[4] = {x_extra, -INFINITY, -INFINITY, -INFINITY};
        int batch = 0;
        for (int v0 = t; v0 - t < row.nvec; v0 += kHold * TPR, ++batch) {
            uint4 d[kHold];
            constexpr uint32_t none = DT == MOM_BF16 ? 0xff80ff80u : 0xff800000u;      // -inf adds nothing
            const int held = (row.nvec - (v0 - t) + TPR - 1) / TPR;      // vectors that any thread has
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
                const int v = v0 + i * TPR;
                d[i] = make_uint4(none, none, none, none);
                if (v < row.nvec) d[i] = __ldg(row.vec + v);
            }
            float vm[kHold];
#pragma unroll
            for (int i = 0; i < kHold; ++i) vm[i] = vec_max<DT>(d[i]);
            vm[0] = tc::fmax3_nan(tc::fmax3_nan(vm[0], vm[1], vm[2]), tc::fmax3_nan(vm[3], vm[4], vm[5]),
                                  tc::fmax3_nan(vm[6], vm[7], vm[7]));
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if ((batch & 3) == q) bmax[q] = tc::fmax3_nan(bmax[q], bmax[q], vm[0]);
            if (vm[0] > ref + slack) rebase(fmaxf(vm[0], kFloor));
            auto sum = [&](const uint4 &q) {
                float x[kVE];
                unpack_floor<DT>(q, x);
#pragma unroll
                for (int e = 0; e < kVE; e += 2) add(x[e], x[e + 1]);
            };
            if (held > kHold / 2) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) sum(d[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kHold / 2; ++i) {
                    if (i >= held) break;
                    sum(d[i]);
                }
            }
        }
        const float m = tc::fmax3_nan(tc::fmax3_nan(bmax[0], bmax[1], bmax[2]), bmax[3], bmax[3]);
        const bool any = ex >= 0 || t < row.nvec;
        const uint32_t mine = any ? order_of(m) : 0u;
        uint32_t M_order = __reduce_max_sync(0xffffffffu, any ? order_of(ref) : 0u);
        const bool broken = __any_sync(0xffffffffu, any && !(m < INFINITY));      // a NaN or an infinite logit
        if (broken) M_order = 0xffffffffu;
        if constexpr (TPR > 32) {
            if (lane == 0) S.top[warp] = M_order;
            __syncthreads();
            M_order = __reduce_max_sync(0xffffffffu, lane < (TPR / 32) ? S.top[lane] : 0u);
        }
        float M = value_of(M_order);
        if (ref > -INFINITY && M < INFINITY) rebase(M);
        const float2 ss = tc::f2_split(s2), ww = tc::f2_split(w2);
        float s = ss.x + ss.y, w = ww.x + ww.y;
        if (fabsf(M) > kFar && fabsf(M) < INFINITY) {
            // a row of masks alone, or a logit whose distance from the floor is not finite: once more,
            // element by element, against the row's maximum
            M_order = __reduce_max_sync(0xffffffffu, mine);
            if constexpr (TPR > 32) {
                __syncthreads();      // S.top is read
                if (lane == 0) S.top[warp] = M_order;
                __syncthreads();
                M_order = __reduce_max_sync(0xffffffffu, lane < (TPR / 32) ? S.top[lane] : 0u);
            }
            M = value_of(M_order);
            s = w = 0.0f;
#pragma unroll 1
            for (int j = t; j < V; j += TPR) {
                const float z = (logit<DT>(row.row, j) - M) * c2, e = tc::ex2(z);
                if (e > 0.0f) {      // not 0 x inf
                    s += e;
                    w = fmaf(e, z, w);
                }
            }
        }
        if (!(M < INFINITY)) s = kNaN;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            w += __shfl_xor_sync(0xffffffffu, w, o);
        }
        if (top > 0) {
            uint32_t g = mine;
#pragma unroll
            for (int o = 1; o < TPR / Tm::kGroups; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
            if (t % (TPR / Tm::kGroups) == 0) S.group[t / (TPR / Tm::kGroups)] = g;
            if (t == 0) S.count = 0;
        }
        if constexpr (TPR > 32) {
            if (lane == 0) S.sums[warp] = make_float2(s, w);
        }
        Tm::sync();
        if constexpr (TPR > 32) {
            const float2 a = lane < (TPR / 32) ? S.sums[lane] : make_float2(0.0f, 0.0f);
            s = a.x;
            w = a.y;
#pragma unroll
            for (int o = (TPR / 32) / 2; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                w += __shfl_xor_sync(0xffffffffu, w, o);
            }
            s = __shfl_sync(0xffffffffu, s, 0);
            w = __shfl_sync(0xffffffffu, w, 0);
        }
        const float lz = logf(s), H = lz - w * kLn2 / s;
        if (t == 0) {
            logprob[r] = tok == ignore ? 0.0f : (x_tok - M) * inv_t - lz;
            entropy[r] = H;
            if (stats) stats[r] = make_float4(M, s, lz, H);
        }
        if (top == 0) {
            if constexpr (TPR > 32) __syncthreads();      // S is read
            continue;
        }
        // the group maximum that exactly top - 1 others are before, counted by the group's lanes
        {
            constexpr int kLanes = Tm::kLanes, kShare = Tm::kShare;
            const int gi = t / kLanes, q0 = t % kLanes * kShare;
            const uint32_t g = S.group[gi];
            int before = 0;
#pragma unroll
            for (int i = 0; i < kShare; i += 4) {
                const uint4 o = *reinterpret_cast<const uint4 *>(&S.group[q0 + i]);
                before += (o.x > g || (o.x == g && q0 + i < gi)) + (o.y > g || (o.y == g && q0 + i + 1 < gi)) +
                          (o.z > g || (o.z == g && q0 + i + 2 < gi)) + (o.w > g || (o.w == g && q0 + i + 3 < gi));
            }
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
            if (before == top - 1 && t % kLanes == 0) S.bound = g;
        }
        Tm::sync();
        const uint32_t bound = S.bound;
        // each element of this thread in turn
        auto each = [&](auto use) {
            if (ex >= 0) use(order_of(x_extra), ex);
            for (int v = t; v < row.nvec; v += TPR) {
                float x[kVE];
                unpack<DT>(__ldg(row.vec + v), x);
#pragma unroll
                for (int e = 0; e < kVE; ++e) use(order_of(x[e]), row.index(v, e));
            }
        };
        if (mine >= bound && any) {
            auto take = [&](uint32_t o, int j) {
                if (o >= bound) {
                    const int at = atomicAdd(&S.count, 1);
                    if (at < Tm::kList) S.list[at] = rank_key(o, j);
                }
            };
            if (ex >= 0) take(order_of(x_extra), ex);
            uint32_t hot = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) hot |= static_cast<uint32_t>(order_of(bmax[q]) >= bound) << q;
            batch = 0;
            for (int v0 = t; v0 < row.nvec; v0 += kHold * TPR, ++batch) {
                if (!(hot >> (batch & 3) & 1)) continue;
                uint32_t hits = 0;
#pragma unroll
                for (int i = 0; i < kHold; ++i)
                    if (v0 + i * TPR < row.nvec)
                        hits |= static_cast<uint32_t>(order_of(vec_max<DT>(__ldg(row.vec + v0 + i * TPR))) >= bound) << i;
                for (; hits; hits &= hits - 1) {
                    const int v = v0 + (__ffs(hits) - 1) * TPR;
                    float x[kVE];
                    unpack<DT>(__ldg(row.vec + v), x);
#pragma unroll
                    for (int e = 0; e < kVE; ++e) take(order_of(x[e]), row.index(v, e));
                }
            }
        }
        Tm::sync();
        const int n = S.count;
        auto put = [&](int k, uint64_t key) {
            top_idx[r * top + k] = rank_index(key);
            top_lp[r * top + k] = (value_of(static_cast<uint32_t>(key >> 32)) - M) * inv_t - lz;
        };
        if (n <= Tm::kList) {
            for (int i = t; i < n; i += TPR) {
                const uint64_t key = S.list[i];
                int before = 0;
                for (int q = 0; q < n; ++q) before += S.list[q] > key;
                if (before < top) put(before, key);
            }
        } else {
            uint64_t below = ~0ull;
            for (int k = 0; k < top; ++k) {
                uint64_t key = 0;
                each([&](uint32_t o, int j) {
                    const uint64_t c = rank_key(o, j);
                    if (c < below && c > key) key = c;
                });
                if (t == 0) S.best = 0;
                Tm::sync();
                atomicMax(&S.best, static_cast<unsigned long long>(key));
                Tm::sync();
                below = S.best;
                if (t == 0) put(k, below);
                Tm::sync();
            }
        }
        Tm::sync();
    }
}

constexpr int kBwdThreads = 256;
constexpr int kBwdVecs = 4;           // vectors of a thread
constexpr int kBwdSpan = kBwdThreads * kBwdVecs;

// One CTA per row and span of kBwdSpan vectors. The terms of single elements (the
// target's, the alternatives') are written over the row's once it stands: the sums
// stay in fp32 and are rounded once.
template <int DT>
__global__ void __launch_bounds__(kBwdThreads)
logprobs_bwd_kernel(const void *__restrict__ logits, int64_t ld, const int64_t *__restrict__ targets,
                    const float4 *__restrict__ stats, const int64_t *__restrict__ top_idx, int top,
                    const float *__restrict__ g_lp, const float *__restrict__ g_ent, const float *__restrict__ g_top,
                    int spans, int V, int64_t ignore, float inv_t, void *__restrict__ dlogits) {
    using T = typename Elem<DT>::T;
    constexpr int kVE = RowSpan<DT>::kVE;
    const int64_t r = blockIdx.x / spans;
    const int span = static_cast<int>(blockIdx.x % spans);
    const RowSpan<DT> row(logits, r * ld, V);
    T *drow = static_cast<T *>(dlogits) + r * V;
    // vectors only where both rows start alike
    const bool alike = ((reinterpret_cast<uintptr_t>(row.row) ^ reinterpret_cast<uintptr_t>(drow)) & 15) == 0;
    const int v0 = span * kBwdSpan + static_cast<int>(threadIdx.x);
    uint4 d[kBwdVecs];
    if (alike)
#pragma unroll
        for (int i = 0; i < kBwdVecs; ++i)
            if (v0 + i * kBwdThreads < row.nvec) d[i] = __ldcs(row.vec + v0 + i * kBwdThreads);
    const float4 st = stats[r];
    const int64_t tok = targets[r];
    float g = g_lp && tok != ignore ? g_lp[r] : 0.0f;
    if (g_lp && tok != ignore && (tok < 0 || tok >= V)) g = kNaN;      // its logprob is; the rest is not its concern
    const float h = g_ent ? g_ent[r] : 0.0f;
    float G = g;
    if (g_top)
        for (int k = 0; k < top; ++k) G += g_top[r * top + k];
    // p (G + h (ln p + H)) with ln p = y - ln Z and p = e^y / Z
    const float inv_z = 1.0f / st.y, base = G + h * (st.w - st.z), c2 = inv_t * kLog2e, hy = h * inv_t;
    const float far = -256.0f / c2;      // p is 0 from there on
    auto grad = [&](float x) {
        const float dx = fmaxf(x - st.x, far);
        const float p = tc::ex2(dx * c2) * inv_z;
        // a masked logit: 0 whatever the rest (p = 0 here, and hy dx is at most 178 h)
        return -p * fmaf(hy, dx, base) * inv_t;
    };
    if (alike) {
        uint4 *dvec = reinterpret_cast<uint4 *>(drow + row.head);
#pragma unroll
        for (int i = 0; i < kBwdVecs; ++i) {
            const int v = v0 + i * kBwdThreads;
            if (v >= row.nvec) break;
            float x[kVE];
            unpack<DT>(d[i], x);
            uint4 o;
            if constexpr (DT == MOM_BF16)
                o = make_uint4(pack_bf16x2(grad(x[0]), grad(x[1])), pack_bf16x2(grad(x[2]), grad(x[3])),
                               pack_bf16x2(grad(x[4]), grad(x[5])), pack_bf16x2(grad(x[6]), grad(x[7])));
            else
                o = make_uint4(__float_as_uint(grad(x[0])), __float_as_uint(grad(x[1])), __float_as_uint(grad(x[2])),
                               __float_as_uint(grad(x[3])));
            __stcs(dvec + v, o);
        }
        if (span == 0) {
            const int ex = row.extra(static_cast<int>(threadIdx.x));
            if (ex >= 0) Elem<DT>::store(drow, ex, grad(logit<DT>(row.row, ex)));
        }
    } else {
        const int j1 = min(V, (span + 1) * kBwdSpan * kVE);
        for (int j = span * kBwdSpan * kVE + static_cast<int>(threadIdx.x); j < j1; j += kBwdThreads)
            Elem<DT>::store(drow, j, grad(logit<DT>(row.row, j)));
    }
    // single elements of this CTA's span
    const int n = g_top ? top : 0;
    __syncthreads();
    const int k = static_cast<int>(threadIdx.x);
    if (k > n) return;
    const int64_t j = k < n ? top_idx[r * top + k] : tok;
    if (j < 0 || j >= V || (k == n && g == 0.0f)) return;
    const int owner = alike ? (j < row.head || j >= row.head + static_cast<int64_t>(row.nvec) * kVE
                                   ? 0
                                   : static_cast<int>((j - row.head) / (kBwdSpan * kVE)))
                            : static_cast<int>(j / (kBwdSpan * kVE));
    if (owner != span) return;
    float add = j == tok ? g : 0.0f;
    for (int q = 0; q < n; ++q)
        if (top_idx[r * top + q] == j) add += g_top[r * top + q];
    Elem<DT>::store(drow, j, fmaf(add, inv_t, grad(logit<DT>(row.row, j))));
}

}  // namespace

// A warp per row has nothing to wait for and costs the fewest instructions, a CTA has
// more of a row on its way. Measured (bf16, 5 alternatives, 16376 rows; warp / 128
// threads): 1000 elements 28 / 77 us, 6000 63 / 102, 12000 106 / 137, 32000 271 / 232.
// Few rows leave SMs idle and want more threads each (128 / 512 threads, kernel time):
// 148 rows of 32000 11.5 / 8.9 us, 400 rows 15 / 16.
cudaError_t launch_logprobs_fwd(const void *logits, int dt, int64_t ld, const int64_t *targets, int64_t R, int V,
                                int64_t ignore, float inv_t, int top, float *logprob, float *entropy, float *top_lp,
                                int64_t *top_idx, float *stats, cudaStream_t st) {
    auto go = [&](auto kernel, int threads, int rows) {
        const int64_t most = static_cast<int64_t>(device_sm_count()) * (1024 / threads);
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>((R + rows - 1) / rows, most));
        kernel<<<grid, threads, 0, st>>>(logits, ld, targets, R, V, ignore, inv_t, top, logprob, entropy, top_lp,
                                         top_idx, reinterpret_cast<float4 *>(stats));
        count_launch();
        return cudaGetLastError();
    };
    auto pick = [&](auto k32, auto k128, auto k512) {
        const int64_t bytes = static_cast<int64_t>(V) * (dt == MOM_BF16 ? 2 : 4), sms = device_sm_count();
        if (bytes > 16384 && R <= 2 * sms) return go(k512, 512, 1);
        return bytes <= 4096 || (bytes <= 32768 && R >= 16 * sms) ? go(k32, 128, 4) : go(k128, 128, 1);
    };
    if (dt == MOM_BF16)
        return pick(logprobs_fwd_kernel<MOM_BF16, 32>, logprobs_fwd_kernel<MOM_BF16, 128>,
                    logprobs_fwd_kernel<MOM_BF16, 512>);
    return pick(logprobs_fwd_kernel<MOM_F32, 32>, logprobs_fwd_kernel<MOM_F32, 128>, logprobs_fwd_kernel<MOM_F32, 512>);
}

cudaError_t launch_logprobs_bwd(const void *logits, int dt, int64_t ld, const int64_t *targets, const float *stats,
                                const int64_t *top_idx, int top, const float *g_lp, const float *g_ent,
                                const float *g_top, int64_t R, int V, int64_t ignore, float inv_t, void *dlogits,
                                cudaStream_t st) {
    const int per = kBwdSpan * (dt == MOM_BF16 ? 8 : 4);
    const int spans = (V + per - 1) / per;
    if (R * spans > INT32_MAX) return cudaErrorInvalidValue;
    auto go = [&](auto kernel) {
        kernel<<<static_cast<unsigned>(R * spans), kBwdThreads, 0, st>>>(
            logits, ld, targets, reinterpret_cast<const float4 *>(stats), top_idx, top, g_lp, g_ent, g_top, spans, V,
            ignore, inv_t, dlogits);
    };
    if (dt == MOM_BF16) go(logprobs_bwd_kernel<MOM_BF16>);
    else go(logprobs_bwd_kernel<MOM_F32>);
    count_launch();
    return cudaGetLastError();
}

}  // namespace mom
