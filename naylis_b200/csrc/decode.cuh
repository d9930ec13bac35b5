// What the attentions of new tokens over a paged cache share (serve.cu, in bf16, and
// serve_int4.cu, in 4 bits): the work of sequences of any lengths cut into one span for
// each CTA, and the join of the parts. A list is a sequence's key head with a group of up
// to kDecHeads rows that read it: its query heads, of one new token or several.
#pragma once

#include "launch.h"
#include "tc_common.cuh"

namespace mom {

namespace {

__device__ __forceinline__ int64_t load_index(const void *p, int i64, int64_t i) {
    return i64 ? static_cast<const int64_t *>(p)[i] : static_cast<int64_t>(static_cast<const int32_t *>(p)[i]);
}

__device__ __forceinline__ void unpack8(const uint4 &v, float (&f)[8]) {
    const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(a[i] << 16);
        f[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
}

constexpr int kDecWarps = 4;
constexpr int kDecHeads = 16;                     // rows of a list at most
constexpr int kClusterMost = 8;

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The same place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float2 ld_cluster(const float2 *p, int rank) {
    uint32_t at;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

struct DecodeArgs {
    const uint16_t *q, *kp, *vp;
    const int32_t *table, *seq_lens;
    int64_t q_ld, table_ld, n_pages, max_len, B;
    int H, Hk, page_shift, n_chunks, chunk;     // n_chunks, chunk (keys): a cluster's
    int rows, per;      // rows of a key head (new tokens x query heads of its group), and of a list at most
    int n_new;                  // new tokens of a sequence, at most
    const int32_t *new_lens;    // and of each one (null: all of them)
    float scale_log2;
    uint16_t *out;
    float *part;        // [part][head of the CTA][m, l, -, -, HD]
    int2 *cut;          // where lists are cut, by the smaller of the two: [list] its first CTA and its number of
                        // CTAs, or [CTA] the list that begins in its span and ends behind it, and its number
    bool by_list;
};

// A sequence's keys as the kernels take them, and its tiles: one without keys for a
// sequence without (its output is zero) and for one that is too long (NaN).
template <int Tile>
struct DecLen {
    int n, tiles;
    bool lost;
    __device__ __forceinline__ DecLen(int32_t len, int64_t max_len) {
        lost = len > max_len;
        n = lost || len < 0 ? 0 : len;
        tiles = max(static_cast<int>((static_cast<unsigned>(n) + Tile - 1) / Tile), 1);
    }
};

// A sequence's new tokens, its last ones: token j sees the keys before sees(j).
struct DecNew {
    int first, count;
    bool lost;      // more of them than the call has, or fewer than none
    __device__ __forceinline__ DecNew(const DecodeArgs &P, int b, int32_t len) {
        count = P.new_lens ? P.new_lens[b] : P.n_new;
        lost = count < 0 || count > P.n_new;
        first = max(len, 0) - count + 1;
        if (lost) count = P.n_new, first = 1;      // every token's result is NaN
    }
    __device__ __forceinline__ int sees(int j) const { return j < count ? first + j : 0; }
};

// The work of all lists (a sequence's key head), one after another, cut into equal spans
// for the grid's CTAs. It is counted in tiles, and a list's start and end as ListCost
// of them ahead of its own. Where span blockIdx.x begins:
struct DecSpan {
    int64_t base, span;          // units before the list that it begins in, and units of a span
    int b, y, i, n;              // sequence, list of it, tile of that, the sequence's length
    int end;                     // the span's end, in units from base
};
template <int Tile, int ListCost, int Least>      // Least: tiles of a span, at least
__device__ __forceinline__ bool decode_span(const DecodeArgs &P, int lists, DecSpan &got) {
    __shared__ int64_t s_sum[kDecWarps];
    __shared__ DecSpan s_got;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int per = static_cast<int>((P.B + kDecWarps * 32 - 1) / (kDecWarps * 32));      // sequences of a thread
    const int64_t b0 = static_cast<int64_t>(t) * per, b1 = min(b0 + per, P.B);
    int64_t mine = 0;
    for (int64_t b = b0; b < b1; ++b) mine += DecLen<Tile>(P.seq_lens[b], P.max_len).tiles + ListCost;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
        if (w < warp) upto += s_sum[w];
        total += s_sum[w];
    }
    total *= lists;
    const int64_t span = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(Least));
    const int64_t from = blockIdx.x * span;
    if (from >= total) return false;
    int64_t base = (upto - mine) * lists;
    if (from >= base && from < upto * lists) {
        for (int64_t b = b0; b < b1; ++b) {
            const int32_t len = P.seq_lens[b];
            const int units = DecLen<Tile>(len, P.max_len).tiles + ListCost;
            const int64_t next = base + static_cast<int64_t>(units) * lists;
            if (from < next) {
                const int y = static_cast<int>((from - base) / units);
                base += static_cast<int64_t>(y) * units;
                s_got = {base, span, static_cast<int>(b), y, max(static_cast<int>(from - base) - ListCost, 0), len,
                         static_cast<int>(min(from + span, total) - base)};
                break;
            }
            base = next;
        }
    }
    __syncthreads();
    got = s_got;
    return true;
}

// Joins the parts of the lists that are cut: a CTA for each of these, each head and (Wide)
// each 32 columns. Lanes threads, four columns each, take a part, the others further
// parts; their sums are joined at the end. Wide is for lists of many parts: 1 sequence of
// 32768, 32 heads on 2 (148 parts): the call takes 18 us, 34 with the narrow form; 18 parts:
// 135 and 138 us.
struct DecSum {
    float M, L;
    float4 o;
    __device__ __forceinline__ void add(float m, float l, float4 x) {
        // what has a maximum of -inf saw no key, or NaN alone (its sum says so)
        const float top = fmaxf(M, m), f = M == -INFINITY ? 0.0f : tc::ex2(M - top), g = m == -INFINITY ? 0.0f : tc::ex2(m - top);
        L = (M == -INFINITY ? L : f * L) + (m == -INFINITY ? l : g * l);
        o.x = fmaf(g, x.x, f * o.x), o.y = fmaf(g, x.y, f * o.y);
        o.z = fmaf(g, x.z, f * o.z), o.w = fmaf(g, x.w, f * o.w);
        M = top;
    }
};
// (48 registers a thread: at the 40 that were chosen without a word the narrow form at
// head_dim 64 spilled; 48 sequences of 64 to 4096 44.8 -> 43.9 us.)
// Drafts: a key head's rows are of several new tokens, some of which may see no key.
template <int HD, bool Wide, bool Drafts>
__global__ void __launch_bounds__(Wide ? 512 : 128, Wide ? 2 : 10)
decode_join_kernel(const __grid_constant__ DecodeArgs P) {
    constexpr int kThreads = Wide ? 512 : 128, kLanes = Wide ? 8 : HD / 4, kGroups = kThreads / kLanes, kRound = 4;
    __shared__ DecSum s_sum[kThreads / 32][kLanes];
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, warp = threadIdx.x / 32;
    const int d = (static_cast<int>(blockIdx.z) * kLanes + lane) * 4;
    const int G = P.H / P.Hk, per = P.per, groups = (P.rows + per - 1) / per, lists = P.Hk * groups;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");      // the parts are written
    const int2 cut = P.cut[blockIdx.x];
    const int list = P.by_list ? blockIdx.x : cut.x, cta = P.by_list ? cut.x : blockIdx.x;
    const int y = list % lists, row = y % groups * per + static_cast<int>(blockIdx.y);
    if (cut.y <= 1 || row >= P.rows) return;
    const int64_t step = static_cast<int64_t>(per) * (HD + 4);
    const float *src = P.part + (static_cast<int64_t>(cta) + list) * step + blockIdx.y * (HD + 4);
    DecSum sum = {-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    for (int c0 = group; c0 < cut.y; c0 += kRound * kGroups) {
        float2 ml[kRound];
        float4 x[kRound];
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
            const int c = c0 + u * kGroups;
            ml[u] = make_float2(-INFINITY, 0.0f);
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (c < cut.y) {
                ml[u] = *reinterpret_cast<const float2 *>(src + c * step);
                x[u] = *reinterpret_cast<const float4 *>(src + c * step + 4 + d);
            }
        }
#pragma unroll
        for (int u = 0; u < kRound; ++u) sum.add(ml[u].x, ml[u].y, x[u]);
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) {
        const auto other = [&](float v) { return __shfl_xor_sync(0xffffffffu, v, o); };
        const float m = other(sum.M), l = other(sum.L);
        sum.add(m, l, make_float4(other(sum.o.x), other(sum.o.y), other(sum.o.z), other(sum.o.w)));
    }
    if (threadIdx.x % 32 < kLanes) s_sum[warp][lane] = sum;
    __syncthreads();
    if (group > 0) return;
    for (int w = 1; w < kThreads / 32; ++w) {
        const DecSum &x = s_sum[w][lane];
        sum.add(x.M, x.L, x.o);
    }
    const float inv = 1.0f / sum.L;      // a list that is cut has keys
    uint2 got = make_uint2(pack_bf16x2(sum.o.x * inv, sum.o.y * inv), pack_bf16x2(sum.o.z * inv, sum.o.w * inv));
    int64_t at = list / lists;
    int h = y / groups * G + row;
    if constexpr (Drafts) {
        const int j = row / G;
        if (DecNew(P, static_cast<int>(at), P.seq_lens[at]).sees(j) <= 0) got = make_uint2(0, 0);
        at = at * P.n_new + j;
        h -= j * G;
    }
    *reinterpret_cast<uint2 *>(P.out + (at * P.H + h) * HD + d) = got;
}

}  // namespace

}  // namespace mom
