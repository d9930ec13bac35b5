// Drafted tokens against the target's distribution: which of them stay, and the token
// that follows them.
//
// With p_j = softmax(x_j / T) of the target's row j and q_j the draft's (drafts without
// logits of their own: all of it on the draft d_j), and given numbers u in [0, 1):
//   draft j stays while u_j q_j(d_j) < p_j(d_j)  (the ones before it having stayed);
//   at the first that falls the token is drawn from max(p_j - q_j, 0), behind all drafts
//   from p_n: the least index i whose running sum exceeds u_K times the whole sum.
// (Leviathan, Kalman and Matias, 2023: the tokens are then distributed as the target's.)
// Greedy: a draft stays while it is the row's greatest logit (the lowest index of equals).
//
// A running sum over the vocabulary decides between neighbours, so everything behind the
// choice of the row is in 64 bits: exponentials, sums, the search. A draft's own test is a
// comparison of two numbers: the rows' sums for it are 32-bit, and where u q and p are within
// 2^-13 of one another, far above those sums' error, it is done again in 64 bits.
//
// One cluster takes a sequence, each of its warps a stretch of every row.
#include <algorithm>
#include <cfloat>

#include "logits.cuh"

namespace mom {

namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kMostCtas = 8;
constexpr int kHold = 4;            // vectors of a lane in flight

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The same place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ uint64_t ld_cluster(const void *p, int rank) {
    uint32_t at;
    uint64_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ double ld_cluster(const double *p, int rank) {
    return __longlong_as_double(static_cast<long long>(ld_cluster(static_cast<const void *>(p), rank)));
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct VerifyArgs {
    const void *logits, *draft;         // draft: null without the drafts' own
    int64_t ld_seq, ld_row, draft_ld_seq, draft_ld_row;
    const int64_t *drafts;
    const float *uniforms;
    const int32_t *draft_lens;          // null: all K
    int V, K, ctas;
    float c2;                           // log2(e) / T
    double inv_t;
    int64_t *tokens, *accepted;
};

enum Verdict { kFalls, kStays, kUnsure, kBroken };

// Greedy: a row's greatest logit, ties to the lowest index. Own: the drafts have logits.
template <int DT, bool Greedy, bool Own>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const __grid_constant__ VerifyArgs P) {
    using T = typename Elem<DT>::T;
    constexpr int kVE = RowSpan<DT>::kVE;
    constexpr int kRows = 2 * kMaxDrafts + 1;
    // of a row: the warps' greatest logit and sum (Greedy: rank key), then this CTA's
    __shared__ uint64_t s_warp[kWarps][Greedy ? kMaxDrafts + 1 : kRows], s_cta[Greedy ? kMaxDrafts + 1 : kRows];
    __shared__ float s_max[kRows];              // of the whole row
    __shared__ float s_sum[kRows];
    __shared__ int s_verdict[kMaxDrafts];
    __shared__ double s_part[2][kWarps];        // the warps' sums in 64 bits, for the target and the draft
    __shared__ double s_whole[2], s_left[kWarps], s_find[2];
    __shared__ int s_owner;
    const int b = static_cast<int>(blockIdx.y), me = static_cast<int>(blockIdx.x), ctas = P.ctas;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w = me * kWarps + warp, W = ctas * kWarps;      // of the cluster's warps
    const int given = P.draft_lens ? P.draft_lens[b] : P.K;
    const bool refused = given < 0 || given > P.K;
    const int n = refused ? 0 : given;
    const int rows = Greedy || !Own ? n + 1 : 2 * n + 1;      // the target's n + 1, then the draft's n
    const int64_t *drafts = P.drafts + static_cast<int64_t>(b) * P.K;
    auto place = [&](int r, const void *&base) {
        if (r <= n) {
            base = P.logits;
            return b * P.ld_seq + r * P.ld_row;
        }
        base = P.draft;
        return b * P.draft_ld_seq + (r - n - 1) * P.draft_ld_row;
    };

    // ---- every row's greatest logit and sum, a stretch of it to each warp
    for (int r = 0; r < rows; ++r) {
        const void *base;
        const int64_t off = place(r, base);
        const RowSpan<DT> row(base, off, P.V);
        const int v0 = static_cast<int>(static_cast<int64_t>(row.nvec) * w / W);
        const int v1 = static_cast<int>(static_cast<int64_t>(row.nvec) * (w + 1) / W);
        const int ex = w == 0 ? row.extra(lane) : -1;
        const float x_extra = ex >= 0 ? logit<DT>(row.row, ex) : -INFINITY;
        if constexpr (Greedy) {
            uint64_t best = ex >= 0 ? rank_key(order_of(x_extra), ex) : 0;
            for (int v = v0 + lane; v < v1; v += kHold * 32) {
                uint4 d[kHold];
#pragma unroll
                for (int i = 0; i < kHold; ++i)
                    if (v + 32 * i < v1) d[i] = __ldg(row.vec + v + 32 * i);
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    if (v + 32 * i >= v1 || order_of(vec_max<DT>(d[i])) < static_cast<uint32_t>(best >> 32)) continue;
                    float x[kVE];
                    unpack<DT>(d[i], x);
#pragma unroll
                    for (int e = 0; e < kVE; ++e)
                        best = max(best, rank_key(order_of(x[e]), row.index(v + 32 * i, e)));
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            if (lane == 0) s_warp[warp][r] = best;
        } else {
            float m = x_extra, ref = fmaxf(m, -FLT_MAX), s = ex >= 0 && x_extra > -INFINITY ? 1.0f : 0.0f;
            for (int v = v0 + lane; v < v1; v += kHold * 32) {
                uint4 d[kHold];
                constexpr uint32_t none = DT == MOM_BF16 ? 0xff80ff80u : 0xff800000u;      // -inf adds nothing
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    d[i] = make_uint4(none, none, none, none);
                    if (v + 32 * i < v1) d[i] = __ldg(row.vec + v + 32 * i);
                }
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kHold; ++i) top = tc::fmax3_nan(top, top, vec_max<DT>(d[i]));
                m = tc::fmax3_nan(m, m, top);
                if (top > ref) {
                    s *= tc::ex2((ref - top) * P.c2);
                    ref = top;
                }
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    float x[kVE], add = 0.0f;
                    unpack<DT>(d[i], x);
#pragma unroll
                    for (int e = 0; e < kVE; ++e) add += tc::ex2((x[e] - ref) * P.c2);
                    s += add;
                }
            }
            float to = m;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) to = tc::fmax3_nan(to, to, __shfl_xor_sync(0xffffffffu, to, o));
            s *= tc::ex2((ref - fmaxf(to, -FLT_MAX)) * P.c2);
            s = mom::warp_sum(s);
            if (lane == 0) s_warp[warp][r] = static_cast<uint64_t>(__float_as_uint(to)) << 32 | __float_as_uint(s);
        }
    }
    __syncthreads();
    auto join = [&](uint64_t a, uint64_t c) {      // of two stretches
        if constexpr (Greedy) return max(a, c);
        const float ma = __uint_as_float(static_cast<uint32_t>(a >> 32)), mc = __uint_as_float(static_cast<uint32_t>(c >> 32));
        const float m = tc::fmax3_nan(ma, ma, mc), ref = fmaxf(m, -FLT_MAX);
        const float s = __uint_as_float(static_cast<uint32_t>(a)) * tc::ex2((fmaxf(ma, -FLT_MAX) - ref) * P.c2) +
                        __uint_as_float(static_cast<uint32_t>(c)) * tc::ex2((fmaxf(mc, -FLT_MAX) - ref) * P.c2);
        return static_cast<uint64_t>(__float_as_uint(m)) << 32 | __float_as_uint(s);
    };
    for (int r = threadIdx.x; r < rows; r += kThreads) {
        uint64_t got = s_warp[0][r];
        for (int i = 1; i < kWarps; ++i) got = join(got, s_warp[i][r]);
        s_cta[r] = got;
    }
    cluster_sync();
    for (int r = threadIdx.x; r < rows; r += kThreads) {
        uint64_t got = ld_cluster(&s_cta[r], 0);
        for (int c = 1; c < ctas; ++c) got = join(got, ld_cluster(&s_cta[r], c));
        if constexpr (Greedy) {
            // the token, -1 for a row with a NaN
            s_warp[0][r] = static_cast<uint32_t>(got >> 32) == 0xffffffffu ? ~0ull : static_cast<uint64_t>(rank_index(got));
        } else {
            s_max[r] = __uint_as_float(static_cast<uint32_t>(got >> 32));
            s_sum[r] = __uint_as_float(static_cast<uint32_t>(got));
        }
    }
    __syncthreads();

    int64_t *tokens = P.tokens + static_cast<int64_t>(b) * (P.K + 1);
    auto finish = [&](int stay) {      // by the one CTA that knows the token: all but that
        for (int j = threadIdx.x; j <= P.K; j += kThreads)
            if (j != stay) tokens[j] = j < stay ? drafts[j] : -1;
        if (threadIdx.x == 0) P.accepted[b] = stay;
    };
    if constexpr (Greedy) {
        if (me == 0) {
            int stay = 0;
            while (stay < n && s_warp[0][stay] != ~0ull && drafts[stay] == static_cast<int64_t>(s_warp[0][stay])) ++stay;
            finish(stay);
            if (threadIdx.x == 0) tokens[stay] = refused ? -1 : static_cast<int64_t>(s_warp[0][stay]);
        }
        cluster_sync();      // nobody leaves while its part is read
        return;
    }

    // ---- 64 bits from here on: the terms of a row, the sums over the cluster
    const int e0 = static_cast<int>(static_cast<int64_t>(P.V) * w / W), e1 = static_cast<int>(static_cast<int64_t>(P.V) * (w + 1) / W);
    auto row_of = [&](int r) {
        const void *base;
        const int64_t off = place(r, base);
        return static_cast<const T *>(base) + off;
    };
    auto term = [&](const T *row, float top, int i) {      // e^((x - top) / T)
        return exp((static_cast<double>(Elem<DT>::load(row, i)) - static_cast<double>(top)) * P.inv_t);
    };
    // The sums of the target's row r (without its element `skip`) and, Own and r < n, of the draft's;
    // the stretches' in s_part.
    auto whole = [&](int r, int skip, bool both, double &zp, double &zq) {
        const T *p = row_of(r), *q = both ? row_of(n + 1 + r) : nullptr;
        const float mp = s_max[r], mq = both ? s_max[n + 1 + r] : 0.0f;
        double a = 0.0, c = 0.0;
#pragma unroll 4
        for (int i = e0 + lane; i < e1; i += 32) {
            if (i != skip) a += term(p, mp, i);
            if (both) c += term(q, mq, i);
        }
        a = warp_sum(a);
        if (both) c = warp_sum(c);
        if (lane == 0) s_part[0][warp] = a, s_part[1][warp] = c;
        __syncthreads();
        if (threadIdx.x < 2) {
            double s = 0.0;
            for (int i = 0; i < kWarps; ++i) s += s_part[threadIdx.x][i];
            s_whole[threadIdx.x] = s;
        }
        cluster_sync();
        zp = zq = 0.0;
        for (int c2 = 0; c2 < ctas; ++c2) {
            zp += ld_cluster(&s_whole[0], c2);
            if (both) zq += ld_cluster(&s_whole[1], c2);
        }
    };
    auto broken = [&](int r) { return !(s_max[r] < INFINITY) || s_max[r] == -INFINITY; };
    auto chance = [&](int r, int64_t d, double z) {      // of token d in row r
        return d >= 0 && d < P.V ? term(row_of(r), s_max[r], static_cast<int>(d)) / z : 0.0;
    };
    const float *u = P.uniforms + static_cast<int64_t>(b) * (P.K + 1);
    for (int j = threadIdx.x; j < n; j += kThreads) {
        int v = kBroken;
        const int64_t d = drafts[j];
        if (!broken(j) && !(Own && broken(n + 1 + j))) {
            const double p = chance(j, d, s_sum[j]);
            const double q = u[j] * (Own ? chance(n + 1 + j, d, s_sum[n + 1 + j]) : 1.0);
            v = d >= 0 && d < P.V && q < p ? kStays : kFalls;
            if (fabs(q - p) <= 0x1p-13 * fmax(fabs(q), p) && p > 0.0) v = kUnsure;
        }
        s_verdict[j] = v;
    }
    __syncthreads();
    // all of the cluster's threads come to the same verdicts
    int stay = 0, verdict = kStays;
    double zp = 0.0, zq = 0.0;
    for (; stay < n; ++stay) {
        verdict = s_verdict[stay];
        if (verdict == kUnsure) {
            whole(stay, -1, Own, zp, zq);
            const int64_t d = drafts[stay];
            const double q = u[stay] * (Own ? chance(n + 1 + stay, d, zq) : 1.0);
            verdict = q < chance(stay, d, zp) ? kStays : kFalls;
            cluster_sync();      // the sums are read
        }
        if (verdict != kStays) break;
    }
    if (refused || broken(stay) || verdict == kBroken) {
        if (me == 0) {
            finish(stay);
            if (threadIdx.x == 0) tokens[stay] = -1;
        }
        cluster_sync();
        return;
    }
    const bool fell = stay < n;
    const int64_t d = fell ? drafts[stay] : -1;
    const T *p = row_of(stay), *q = Own && fell ? row_of(n + 1 + stay) : nullptr;
    const float mp = s_max[stay], mq = q ? s_max[n + 1 + stay] : 0.0f;
    int skip = !Own && fell && d >= 0 && d < P.V ? static_cast<int>(d) : -1;
    bool both = q != nullptr;
    whole(stay, skip, both, zp, zq);
    double fp = 1.0, fq = 0.0;
    if (both) fp = 1.0 / zp, fq = 1.0 / zq;
    auto left = [&](int i) {      // what the token is drawn from
        double v = i == skip ? 0.0 : term(p, mp, i) * fp;
        if (both) v = fmax(v - term(q, mq, i) * fq, 0.0);
        return v;
    };
    if (both) {
        double a = 0.0;
#pragma unroll 4
        for (int i = e0 + lane; i < e1; i += 32) a += left(i);
        a = warp_sum(a);
        if (lane == 0) s_left[warp] = a;
    } else if (lane == 0) {
        s_left[warp] = s_part[0][warp];
    }
    cluster_sync();
    // where the running sum passes u times the whole: among the cluster's stretches
    auto find = [&]() {
        if (warp == 0) {
            // each lane takes neighbouring stretches
            constexpr int kPer = kMostCtas * kWarps / 32;
            const int per = (W + 31) / 32;
            double x[kPer], mine = 0.0;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = lane * per + k;
                x[k] = k < per && i < W ? ld_cluster(&s_left[i % kWarps], i / kWarps) : 0.0;
            }
#pragma unroll
            for (int k = 0; k < kPer; ++k) mine += x[k];
            double upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const double goal = u[P.K] * __shfl_sync(0xffffffffu, upto, 31);
            const uint32_t some = __ballot_sync(0xffffffffu, mine > 0.0);
            const uint32_t past = __ballot_sync(0xffffffffu, mine > 0.0 && upto > goal);
            if (lane == 0) s_owner = -1;
            __syncwarp();
            // u at or above 1, or its last bit: the last stretch with anything
            if (some && lane == (past ? __ffs(past) - 1 : 31 - __clz(some))) {
                double run = upto - mine;
                for (int k = 0; k < kPer; ++k) {
                    if (x[k] > 0.0) {
                        s_owner = lane * per + k;
                        s_find[0] = goal;
                        s_find[1] = run;
                        if (run + x[k] > goal) break;
                    }
                    run += x[k];
                }
            }
        }
        __syncthreads();
    };
    find();
    if (s_owner < 0) {
        // nothing is left (the draft's distribution is the target's): from the target's own
        skip = -1, both = false, fp = 1.0;
        cluster_sync();      // the sums are read
        double z0, z1;
        whole(stay, -1, false, z0, z1);
        if (lane == 0) s_left[warp] = s_part[0][warp];
        cluster_sync();
        find();
    }
    const int owner = s_owner;
    if (owner / kWarps == me) {
        finish(stay);
        if (owner % kWarps == warp) {
            // the owner's lanes take neighbouring elements each
            const int per = (e1 - e0 + 31) / 32, i0 = min(e0 + lane * per, e1), i1 = min(i0 + per, e1);
            double mine = 0.0;
            for (int i = i0; i < i1; ++i) mine += left(i);
            double upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const double goal = s_find[0];
            upto += s_find[1];
            const uint32_t some = __ballot_sync(0xffffffffu, mine > 0.0);
            uint32_t past = __ballot_sync(0xffffffffu, mine > 0.0 && upto > goal);
            if (!past) past = 1u << (31 - __clz(some));
            if (lane == __ffs(past) - 1) {
                double run = upto - mine;
                int at = -1;
                for (int i = i0; i < i1; ++i) {
                    const double x = left(i);
                    run += x;
                    if (x > 0.0) {
                        at = i;
                        if (run > goal) break;
                    }
                }
                tokens[stay] = at;
            }
        }
    }
    cluster_sync();      // nobody leaves while its sums are read
}

}  // namespace

cudaError_t launch_verify_drafts(const void *logits, int dt, int64_t ld_seq, int64_t ld_row, const void *draft,
                                 int64_t draft_ld_seq, int64_t draft_ld_row, const int64_t *drafts,
                                 const float *uniforms, const int32_t *draft_lens, int64_t B, int K, int V,
                                 double temperature, int64_t *tokens, int64_t *accepted, cudaStream_t st) {
    VerifyArgs p = {};
    p.logits = logits;
    p.draft = draft;
    p.ld_seq = ld_seq;
    p.ld_row = ld_row;
    p.draft_ld_seq = draft_ld_seq;
    p.draft_ld_row = draft_ld_row;
    p.drafts = drafts;
    p.uniforms = uniforms;
    p.draft_lens = draft_lens;
    p.V = V;
    p.K = K;
    const bool greedy = temperature == 0.0;
    p.inv_t = greedy ? 1.0 : 1.0 / temperature;
    p.c2 = static_cast<float>(p.inv_t * 1.4426950408889634);
    p.tokens = tokens;
    p.accepted = accepted;
    // as many CTAs a sequence as fit the GPU with those of all sequences
    p.ctas = kMostCtas;
    while (p.ctas > 1 && B * p.ctas > 2 * device_sm_count()) p.ctas /= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(p.ctas);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(p.ctas), static_cast<unsigned>(B));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    auto go = [&](auto kernel) { return cudaLaunchKernelEx(&cfg, kernel, p); };
    cudaError_t e;
    if (dt == MOM_BF16)
        e = greedy ? go(verify_kernel<MOM_BF16, true, false>)
                   : draft ? go(verify_kernel<MOM_BF16, false, true>) : go(verify_kernel<MOM_BF16, false, false>);
    else
        e = greedy ? go(verify_kernel<MOM_F32, true, false>)
                   : draft ? go(verify_kernel<MOM_F32, false, true>) : go(verify_kernel<MOM_F32, false, false>);
    count_launch();
    return e;
}

}  // namespace mom
