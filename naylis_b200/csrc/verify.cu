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
// comparison of two numbers: the rows' sums for it are 32-bit, and where u q and p are as near one
// another as those sums may be off, at least 2^-13, it is done again in 64 bits.
//
// One cluster takes a sequence. Its warps share the rows out for the 32-bit sums, each some
// contiguous part of one row at a time; in 64 bits each has a stretch of the vocabulary, whose
// exponentials it keeps in shared memory where they fit (the search then reads them).
// Rows of 32000, bf16: 1 sequence of 4 drafts 11 us, 48 of 4 22 us, 40 of 7 in fp32 17 us (drafts
// without logits), bound by the chain of phases (sums, decision, the row's terms, search), a barrier
// behind each; 256 of 7 greedily 25 us, 5.3 TB/s, by memory. Where the terms are not kept they are computed up to three
// times: 56 of 4 59 us, 256 of 4 237 us.
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "logits.cuh"

namespace mom {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kMostCtas = 16;      // of a cluster: 16 where there are few sequences and the device places them, else 8 at most
constexpr int kHold = 4;            // vectors of a lane in flight, twice
constexpr int kBatch = 8;           // elements of a lane in flight, of each row
constexpr int kRounds = 9;          // parts of rows that a warp takes, at most: all rows, one CTA
constexpr int kTableBits = 7, kTable = 1 << kTableBits;
constexpr int kMostKeep = 8300;     // doubles that a CTA keeps, for three CTAs an SM

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
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
    int keep;                           // elements of a CTA's stretch of a row that are kept, 0: none
    float c2;                           // log2(e) / T
    double near;                        // what two 32-bit sums may be off by, of themselves
    double scale;                       // kTable log2(e) / T
    int64_t *tokens, *accepted;
};

enum Verdict { kFalls, kStays, kUnsure, kBroken };

// e^(d s / kTable ln 2) for d <= 0 in 64 bits, by table and polynomial (Tang, 1989): d s is
// rounded to n, 2^(n mod kTable / kTable) comes from the table and the rest, within 1/2 of a
// kTable-th, from a polynomial of degree 4: 1e-15 of the result, and |d s| 2^-53 / kTable more.
__device__ __forceinline__ double exp_of(double d, double s, const double *table) {
    constexpr double kMagic = 6755399441055744.0;      // 1.5 2^52: the sum's low bits are the rounded number
    constexpr double kL = 0.69314718055994530942 / kTable;
    const double t = fma(d, s, kMagic), f = fma(d, s, kMagic - t);
    const int n = __double2loint(t);
    double p = fma(f, kL * kL * kL * kL / 24, kL * kL * kL / 6);
    p = fma(p, f, kL * kL / 2);
    p = fma(p, f, kL) * f;
    const double v = table[n & (kTable - 1)];
    const double two = __hiloint2double(__double2hiint(v) + (n >> kTableBits << 20), __double2loint(v));
    return d * s > -1020.0 * kTable ? fma(two, p, two) : 0.0;      // (NaN: 0; a row with one is not summed)
}

// x in 64 bits by integer operations (the conversion has a twelfth of their rate). Zeros and
// subnormals become 2^-127 and a little more, infinities 2^128: below and above whatever matters here.
__device__ __forceinline__ double wide(float x) {
    const uint32_t b = __float_as_uint(x);
    return __hiloint2double(static_cast<int>((b & 0x80000000u) | ((b & 0x7fffffffu) >> 3) + 0x38000000u), static_cast<int>(b << 29));
}
__device__ __forceinline__ double sum_of_batch(double (&e)[kBatch]) {
#pragma unroll
    for (int o = kBatch / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < o; ++k) e[k] += e[k + o];
    return e[0];
}

// What is left of the target for a term, max(a fa - c fc, 0). Both products are rounded, neither
// goes into the difference whole: equal terms of equal rows leave nothing.
__device__ __forceinline__ double left_of(double a, double fa, double c, double fc) {
    return fmax(__dsub_rn(__dmul_rn(a, fa), __dmul_rn(c, fc)), 0.0);
}

// Greedy: a row's greatest logit, ties to the lowest index. Own: the drafts have logits.
template <int DT, bool Greedy, bool Own>
__global__ void __launch_bounds__(kThreads, Greedy ? 4 : 3) verify_kernel(const __grid_constant__ VerifyArgs P) {
    using T = typename Elem<DT>::T;
    constexpr int kVE = RowSpan<DT>::kVE;
    constexpr int kRows = Greedy || !Own ? kMaxDrafts + 1 : 2 * kMaxDrafts + 1;
    extern __shared__ double s_keep[];          // a stretch's terms: of the target's row, then of the draft's
    __shared__ uint64_t s_unit[kRounds][kWarps];      // the greatest logit and the sum (Greedy: rank key) of a part of a row
    __shared__ uint64_t s_row[kRows];           // of whole rows
    __shared__ int s_verdict[kMaxDrafts];
    __shared__ int64_t s_draft[Greedy ? 1 : kMaxDrafts];
    __shared__ double s_part[2][kWarps];        // the warps' sums in 64 bits, for the target and the draft
    __shared__ double s_left[kWarps], s_find[2], s_table[kTable];
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
    // what a draft's test needs, on its way while the rows are summed
    float given_u = 0.0f, last_u = 0.0f, draft_p = -INFINITY, draft_q = -INFINITY;
    int64_t draft = -1;
    if constexpr (!Greedy) {
        const float *u = P.uniforms + static_cast<int64_t>(b) * (P.K + 1);
        last_u = u[P.K];
        const int j = static_cast<int>(threadIdx.x);
        if (j < n) {
            given_u = u[j];
            draft = drafts[j];
            if (draft >= 0 && draft < P.V) {
                const void *base;
                int64_t off = place(j, base);
                draft_p = logit<DT>(base, off + draft);
                if (Own) {
                    off = place(n + 1 + j, base);
                    draft_q = logit<DT>(base, off + draft);
                }
            }
        }
    }

    // ---- every row's greatest logit and sum: parts of rows, as many as give each warp about the same
    int parts = 1;
    for (int rounds = 1; rounds <= 4; ++rounds) {
        parts = max(rounds * W / rows, 1);
        if (rows * parts * 8 >= rounds * W * 7) break;
    }
    parts = min(parts, max(P.V / (64 * kVE), 1));
    const auto join = [&](uint64_t a, uint64_t c) {      // of two parts
        if constexpr (Greedy) return max(a, c);
        const float ma = __uint_as_float(static_cast<uint32_t>(a >> 32)), mc = __uint_as_float(static_cast<uint32_t>(c >> 32));
        const float m = tc::fmax3_nan(ma, ma, mc), ref = fmaxf(m, -FLT_MAX);
        const float s = __uint_as_float(static_cast<uint32_t>(a)) * tc::ex2((fmaxf(ma, -FLT_MAX) - ref) * P.c2) +
                        __uint_as_float(static_cast<uint32_t>(c)) * tc::ex2((fmaxf(mc, -FLT_MAX) - ref) * P.c2);
        return static_cast<uint64_t>(__float_as_uint(m)) << 32 | __float_as_uint(s);
    };
    const auto join_lanes = [&](uint64_t v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    };
    constexpr uint64_t kNothing = Greedy ? 0 : static_cast<uint64_t>(0xff800000u) << 32;
    for (int unit = w, round = 0; unit < rows * parts; unit += W, ++round) {
        const int r = unit / parts, part = unit - r * parts;
        const void *base;
        const int64_t off = place(r, base);
        const RowSpan<DT> row(base, off, P.V);
        const int v1 = static_cast<int>(static_cast<int64_t>(row.nvec) * (part + 1) / parts);
        int v = static_cast<int>(static_cast<int64_t>(row.nvec) * part / parts) + lane;
        const int ex = part == 0 ? row.extra(lane) : -1;
        const float x_extra = ex >= 0 ? logit<DT>(row.row, ex) : -INFINITY;
        constexpr uint32_t none = DT == MOM_BF16 ? 0xff80ff80u : 0xff800000u;      // -inf adds nothing
        const auto load = [&](uint4 (&d)[kHold], int at) {
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
                d[i] = make_uint4(none, none, none, none);
                if (at + 32 * i < v1) d[i] = __ldg(row.vec + at + 32 * i);
            }
        };
        uint64_t best = Greedy && ex >= 0 ? rank_key(order_of(x_extra), ex) : 0;
        // Greedy: the first of the greatest vectors, NaN left out; which element it is comes behind the loop
        float great = -INFINITY;
        int at = v < v1 ? v : -1;
        float m = x_extra, ref = fmaxf(m, -FLT_MAX);
        uint64_t s2 = tc::f2(ex >= 0 && x_extra > -INFINITY ? 1.0f : 0.0f, 0.0f);
        const uint64_t cc2 = tc::f2(P.c2, P.c2);
        uint4 d[kHold];
        load(d, v);
        for (; v - lane < v1; v += kHold * 32) {
            uint4 next[kHold];
            load(next, v + kHold * 32);
            if constexpr (Greedy) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    const float x = vec_max<DT>(d[i]);
                    m = tc::fmax3_nan(m, m, x);
                    if (x > great) great = x, at = v + 32 * i;
                }
            } else {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kHold; ++i) top = tc::fmax3_nan(top, top, vec_max<DT>(d[i]));
                m = tc::fmax3_nan(m, m, top);
                if (top > ref) {
                    const float f = tc::ex2((ref - top) * P.c2);
                    s2 = tc::mul2(s2, tc::f2(f, f));
                    ref = top;
                }
                const uint64_t ref2 = tc::f2(ref, ref);
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    float x[kVE];
                    unpack<DT>(d[i], x);
#pragma unroll
                    for (int e = 0; e < kVE; e += 2)
                        s2 = tc::add2(s2, tc::ex2_pair(tc::mul2(tc::sub2(tc::f2(x[e], x[e + 1]), ref2), cc2)));
                }
            }
#pragma unroll
            for (int i = 0; i < kHold; ++i) d[i] = next[i];
        }
        if constexpr (!Greedy) {
            float to = m;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) to = tc::fmax3_nan(to, to, __shfl_xor_sync(0xffffffffu, to, o));
            const float2 s = tc::f2_split(s2);
            const float all = mom::warp_sum((s.x + s.y) * tc::ex2((ref - fmaxf(to, -FLT_MAX)) * P.c2));
            best = static_cast<uint64_t>(__float_as_uint(to)) << 32 | __float_as_uint(all);
        } else {
            if (at >= 0) {
                float x[kVE];
                unpack<DT>(__ldg(row.vec + at), x);
                int e = 0;
#pragma unroll
                for (int i = kVE - 1; i >= 0; --i)
                    if (x[i] == great) e = i;
                best = max(best, rank_key(order_of(great), row.index(at, e)));
            }
            if (m != m) best = rank_key(order_of(m), 0);      // a NaN
            best = join_lanes(best);
        }
        if (lane == 0) s_unit[round][warp] = best;
    }
    cluster_arrive();
    if constexpr (!Greedy)      // while the others arrive
        if (threadIdx.x < kTable) s_table[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / kTable);
    cluster_wait();
    // a row to a warp, or with the drafts' rows two where that takes fewer turns: a turn is a read from another CTA (0.4
    // us of 1 x 4; at 8 rows without the drafts' the choice itself would cost as much)
    const int team = Own && rows > kWarps ? 16 : 32, mate = lane & (team - 1);
    for (int r0 = warp * 32 / team; r0 < rows; r0 += kWarps * 32 / team) {
        const int r = r0 + lane / team;
        uint64_t got = kNothing;
        for (int part = mate; part < parts && r < rows; part += team) {
            const int unit = r * parts + part, of = unit % W;
            got = join(got, ld_cluster(&s_unit[unit / W][of % kWarps], of / kWarps));
        }
        for (int o = team / 2; o > 0; o >>= 1) got = join(got, __shfl_xor_sync(0xffffffffu, got, o));
        // Greedy: the token, -1 for a row with a NaN
        if (Greedy) got = static_cast<uint32_t>(got >> 32) == 0xffffffffu ? ~0ull : static_cast<uint64_t>(rank_index(got));
        if (mate == 0 && r < rows) s_row[r] = got;
    }
    __syncthreads();

    int64_t *tokens = P.tokens + static_cast<int64_t>(b) * (P.K + 1);
    auto finish = [&](int stay) {      // by the one CTA that knows the token: all but that
        for (int j = threadIdx.x; j <= P.K; j += kThreads)
            if (j != stay) tokens[j] = j >= stay ? -1 : Greedy ? drafts[j] : s_draft[j];
        if (threadIdx.x == 0) P.accepted[b] = stay;
    };
    if constexpr (Greedy) {
        if (me == 0) {
            int stay = 0;
            while (stay < n && s_row[stay] != ~0ull && drafts[stay] == static_cast<int64_t>(s_row[stay])) ++stay;
            finish(stay);
            if (threadIdx.x == 0) tokens[stay] = refused ? -1 : static_cast<int64_t>(s_row[stay]);
        }
        cluster_sync();      // nobody leaves while its part is read
        return;
    } else {
        // ---- 64 bits from here on: the terms of a row, the sums over the cluster
        const auto greatest = [&](int r) { return __uint_as_float(static_cast<uint32_t>(s_row[r] >> 32)); };
        const auto sum_of = [&](int r) { return __uint_as_float(static_cast<uint32_t>(s_row[r])); };
        const int c0 = static_cast<int>(static_cast<int64_t>(P.V) * me / ctas);      // this CTA's first element
        const int e0 = static_cast<int>(static_cast<int64_t>(P.V) * w / W), e1 = static_cast<int>(static_cast<int64_t>(P.V) * (w + 1) / W);
        auto row_of = [&](int r) {
            const void *base;
            const int64_t off = place(r, base);
            return static_cast<const T *>(base) + off;
        };
        auto term = [&](float x, float top) {      // e^((x - top) / T)
            return exp_of(wide(x) - wide(top), P.scale, s_table);
        };
        auto broken = [&](int r) { return !(greatest(r) < INFINITY) || greatest(r) == -INFINITY; };
        // a draft's test: u q < p, and (32 bits) whether the two are too near one another
        auto test = [&](float u, float xp, float xq, int r, double zp, double zq, bool &near) {
            const double p = term(xp, greatest(r)), q = u * (Own ? term(xq, greatest(n + 1 + r)) : 1.0);      // times z
            const double l = q * zp, m = Own ? p * zq : p;
            near = fabs(l - m) <= P.near * fmax(fabs(l), m) && m > 0.0;
            return l < m ? kStays : kFalls;
        };
        if (static_cast<int>(threadIdx.x) < n) {
            const int j = static_cast<int>(threadIdx.x);
            int v = kBroken;
            if (!broken(j) && !(Own && broken(n + 1 + j))) {
                v = kFalls;      // outside the vocabulary
                bool near = false;
                if (draft >= 0 && draft < P.V)
                    v = test(given_u, draft_p, draft_q, j, sum_of(j), Own ? sum_of(n + 1 + j) : 1.0f, near);
                if (near) v = kUnsure;
            }
            s_verdict[j] = v;
            s_draft[j] = draft;
        }
        __syncthreads();
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
                const double goal = last_u * __shfl_sync(0xffffffffu, upto, 31);
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
        // All of the cluster's threads come to the same verdicts. The row that decides is summed in 64 bits, for
        // a verdict on its draft first where that is unsure, then for the token.
        int stay = 0, skip;
        bool both, own_alone = false;
        double fp, fq;
        const T *p, *q;
        float mp, mq;
        auto left = [&](int i) {      // what the token is drawn from, where it is not kept
            const double v = i == skip ? 0.0 : term(Elem<DT>::load(p, i), mp);
            return both ? left_of(v, fp, term(Elem<DT>::load(q, i), mq), fq) : v;
        };
        while (true) {
            while (stay < n && s_verdict[stay] == kStays) ++stay;
            const int verdict = stay < n ? s_verdict[stay] : kFalls;
            if (refused || broken(stay) || verdict == kBroken) {
                if (me == 0) {
                    finish(stay);
                    if (threadIdx.x == 0) tokens[stay] = -1;
                }
                cluster_sync();
                return;
            }
            const int64_t d = stay < n ? s_draft[stay] : -1;
            both = Own && stay < n && !own_alone;
            skip = !Own && verdict == kFalls && !own_alone && d >= 0 && d < P.V ? static_cast<int>(d) : -1;
            p = row_of(stay), q = both ? row_of(n + 1 + stay) : p;
            mp = greatest(stay), mq = both ? greatest(n + 1 + stay) : 0.0f;
            double a = 0.0, c = 0.0;
            // a batch of both rows on its way together, and its terms side by side: each is a chain of a dozen operations
            for (int i = e0 + lane; i - lane < e1; i += 32 * kBatch) {
                float x[2][kBatch];
                if constexpr (Own) {
                    // (unconditional, where there is nothing from the stretch's last place: under conditions 16 loads take turns,
                    // 1 x 4 0.4 us; 8 did not)
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) x[0][k] = Elem<DT>::load(p, min(i + 32 * k, e1 - 1));
                    if (both) {
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) x[1][k] = Elem<DT>::load(q, min(i + 32 * k, e1 - 1));
                    }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int at = i + 32 * k;
                        if (at >= e1) x[0][k] = x[1][k] = -INFINITY;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int at = i + 32 * k;
                        x[0][k] = at < e1 && at != skip ? Elem<DT>::load(p, at) : -INFINITY;
                        x[1][k] = -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (r == 1 && !both) break;
                    double e[kBatch];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) e[k] = term(x[r][k], r == 0 ? mp : mq);
                    if (P.keep) {
#pragma unroll
                        for (int k = 0; k < kBatch; ++k)
                            if (i + 32 * k < e1) s_keep[r * P.keep + i + 32 * k - c0] = e[k];
                    }
                    (r == 0 ? a : c) += sum_of_batch(e);
                }
            }
            a = warp_sum(a);
            if (both) c = warp_sum(c);
            if (lane == 0) s_part[0][warp] = a, s_part[1][warp] = c;
            if (both || verdict == kUnsure) {
                cluster_sync();
                // all warps' sums by the lanes at once, in the same order everywhere
                const auto whole = [&](const double (&part)[kWarps]) {
                    double x[kMostCtas * kWarps / 32], sum = 0.0;
#pragma unroll
                    for (int k = 0; k < kMostCtas * kWarps / 32; ++k) {
                        const int i = lane + 32 * k;
                        x[k] = i < W ? ld_cluster(&part[i % kWarps], i / kWarps) : 0.0;
                    }
#pragma unroll
                    for (int k = 0; k < kMostCtas * kWarps / 32; ++k) sum += x[k];
                    return warp_sum(sum);
                };
                const double zp = whole(s_part[0]), zq = both ? whole(s_part[1]) : 0.0;
                if (verdict == kUnsure) {
                    const float u = P.uniforms[static_cast<int64_t>(b) * (P.K + 1) + stay];
                    bool near;
                    const int now = test(u, Elem<DT>::load(p, d), Own ? Elem<DT>::load(q, d) : 0.0f, stay, zp, zq, near);
                    cluster_sync();      // the sums are read, and the verdict
                    if (threadIdx.x == 0) s_verdict[stay] = now;
                    __syncthreads();
                    continue;
                }
                fp = zq, fq = zp;      // p - q, times both sums
            }
            if (both) {
                a = 0.0;
                for (int i = e0 + lane; i - lane < e1; i += 32 * kBatch) {
                    double e[kBatch];
                    if (P.keep) {
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            const int at = i + 32 * k - c0;
                            e[k] = i + 32 * k < e1 ? left_of(s_keep[at], fp, s_keep[P.keep + at], fq) : 0.0;
                        }
#pragma unroll
                        for (int k = 0; k < kBatch; ++k)
                            if (i + 32 * k < e1) s_keep[i + 32 * k - c0] = e[k];
                    } else {
#pragma unroll 1
                        for (int k = 0; k < kBatch; ++k) a += i + 32 * k < e1 ? left(i + 32 * k) : 0.0;
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) e[k] = 0.0;
                    }
                    a += sum_of_batch(e);
                }
                a = warp_sum(a);
            }
            if (lane == 0) s_left[warp] = a;
            cluster_sync();
            find();
            // nothing is left (the draft's distribution is the target's): from the target's own
            if (s_owner >= 0 || own_alone) break;
            own_alone = true;
            cluster_sync();      // the sums are read
        }
        const int owner = s_owner;
        if (owner >= 0 && owner / kWarps == me) {
            finish(stay);
            if (owner % kWarps == warp) {
                // the owner's lanes take neighbouring elements each, an odd number of them: no bank conflicts
                const int per = (e1 - e0 + 31) / 32 | 1, i0 = min(e0 + lane * per, e1), i1 = min(i0 + per, e1);
                double mine = 0.0;
                for (int i = i0; i < i1; i += kBatch) {
                    double e[kBatch];
                    if (P.keep) {
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) e[k] = i + k < i1 ? s_keep[i + k - c0] : 0.0;
                    } else {
#pragma unroll 1
                        for (int k = 0; k < kBatch; ++k) mine += i + k < i1 ? left(i + k) : 0.0;
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) e[k] = 0.0;
                    }
                    mine += sum_of_batch(e);
                }
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
                // that lane's elements, one to each lane in turn
                const int of = __ffs(past) - 1;
                double run = __shfl_sync(0xffffffffu, upto - mine, of);
                const int f0 = __shfl_sync(0xffffffffu, i0, of), f1 = __shfl_sync(0xffffffffu, i1, of);
                int at = -1;
                for (int i = f0; i < f1; i += 32) {
                    const double x = i + lane >= f1 ? 0.0 : P.keep ? s_keep[i + lane - c0] : left(i + lane);
                    double sum = x;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double y = __shfl_up_sync(0xffffffffu, sum, o);
                        if (lane >= o) sum += y;
                    }
                    const uint32_t any = __ballot_sync(0xffffffffu, x > 0.0);
                    const uint32_t over = __ballot_sync(0xffffffffu, x > 0.0 && run + sum > goal);
                    if (any) at = i + (over ? __ffs(over) - 1 : 31 - __clz(any));
                    if (over) break;
                    run += __shfl_sync(0xffffffffu, sum, 31);
                }
                if (lane == 0) tokens[stay] = at;
            }
        }
        cluster_sync();      // nobody leaves while its sums are read
    }
}

template <int DT, bool Greedy, bool Own>
cudaError_t launch(VerifyArgs &p, int64_t B, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0}, most{0};      // devices whose kernel has its shared memory set; that place kMostCtas
    const auto kernel = verify_kernel<DT, Greedy, Own>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kMostCtas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(kMostCtas, static_cast<unsigned>(B));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kMostKeep * sizeof(double);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const uint64_t bit = uint64_t(1) << (dev & 63);
    bool fits;
    if (dev < 64 && ready.load(std::memory_order_acquire) & bit) {
        fits = most.load(std::memory_order_relaxed) & bit;
    } else {
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostKeep * 8)) != cudaSuccess ||
            (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
            return e;
        // more than 8 CTAs a cluster are not promised: a part of a GPU may have no 16 processors side by side
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0, cudaGetLastError();
        fits = n > 0;
        if (dev < 64) {
            if (fits) most.fetch_or(bit, std::memory_order_relaxed);
            ready.fetch_or(bit, std::memory_order_release);
        }
    }
    // as many CTAs a sequence as fit the GPU with those of all sequences; 16 for few of them (4 sampled drafts of 32000, 16 and
    // 8: 1 sequence 11.1 and 13.1 us, 4 12.4 and 14.8, 8 14.1 and 14.9, 20 17.0 and 16.7, 27 26.6 and 18.0)
    p.ctas = B <= 8 && fits ? kMostCtas : 8;
    while (p.ctas > 1 && B * p.ctas > (Greedy ? 4 : 3) * device_sm_count()) p.ctas /= 2;
    const int keep = (p.V + p.ctas - 1) / p.ctas + 1, kept = Own ? 2 : 1;
    if (!Greedy && static_cast<int64_t>(keep) * kept <= kMostKeep) p.keep = keep;
    attr.val.clusterDim.x = static_cast<unsigned>(p.ctas);
    cfg.gridDim.x = static_cast<unsigned>(p.ctas);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.keep) * kept * sizeof(double);
    e = cudaLaunchKernelEx(&cfg, kernel, p);
    count_launch();
    return e;
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
    const double per = greedy ? 1.0 : 1.4426950408889634 / temperature;
    p.c2 = static_cast<float>(per);
    p.scale = kTable * per;
    // a lane adds up to V / 64 terms to each of its two sums, which all may round the same way, by 2^-24 of the sum: twice that
    // for the two rows; 2^-13 for exponentials and what joins the lanes (2^-18) and vocabularies up to 65536
    p.near = std::max(0x1p-13, V * 0x1p-29);
    p.tokens = tokens;
    p.accepted = accepted;
    if (dt == MOM_BF16)
        return greedy ? launch<MOM_BF16, true, false>(p, B, st)
                      : draft ? launch<MOM_BF16, false, true>(p, B, st) : launch<MOM_BF16, false, false>(p, B, st);
    return greedy ? launch<MOM_F32, true, false>(p, B, st)
                  : draft ? launch<MOM_F32, false, true>(p, B, st) : launch<MOM_F32, false, false>(p, B, st);
}

}  // namespace mom
