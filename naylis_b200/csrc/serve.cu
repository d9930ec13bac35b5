// Rotary embedding with the cache write, and attention of one new token per
// sequence over a paged key-value cache.
//
// Cache layout: K and V pages (num_pages, Hk, page_size, hd) bf16, so that the
// keys of one head in one page are one contiguous run; a token's slot is
// page * page_size + offset. The page size is a power of two (8 .. 256): a
// key's page and offset are a shift and a mask.
#include <algorithm>
#include <atomic>

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

// ------------------------------------------------------------------ rope_append
// One thread per (token, head, 8 rotation pairs). Bound by memory: the projection in; q,
// pages (and k) out. 16384 tokens of 16 + 2 x 4 heads of 128: 38 us, 5.8 TB/s; 64 tokens
// of 48 heads of 64: 2.0 us. (A warp per token that keeps the tables' values for all its
// heads: 36.7 and 3.2 us.)
template <int HD>
__global__ void __launch_bounds__(256)
rope_append_kernel(const uint16_t *__restrict__ qkv, int64_t ld, const float *__restrict__ cosv,
                   const float *__restrict__ sinv, int64_t n_pos, const void *__restrict__ positions, int pos64,
                   const void *__restrict__ slots, int slot64, int64_t T, int H, int Hk, int64_t n_slots,
                   int page_shift, uint16_t *__restrict__ kp, uint16_t *__restrict__ vp, uint16_t *__restrict__ q,
                   uint16_t *__restrict__ k) {
    constexpr int kHalf = HD / 2, kGroups = kHalf / 8;
    const int heads = H + 2 * Hk;
    const int64_t total = T * heads * kGroups;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int p = static_cast<int>(i % kGroups) * 8;
        const int h = static_cast<int>(i / kGroups % heads);
        const int64_t t = i / kGroups / heads;
        const uint16_t *src = qkv + t * ld + static_cast<int64_t>(h) * HD;
        uint4 lo = *reinterpret_cast<const uint4 *>(src + p), hi = *reinterpret_cast<const uint4 *>(src + p + kHalf);
        if (h < H + Hk) {
            const int64_t pos = load_index(positions, pos64, t);
            float x1[8], x2[8], y1[8], y2[8];
            unpack8(lo, x1);
            unpack8(hi, x2);
            if (pos >= 0 && pos < n_pos) {
                const float *cs = cosv + pos * HD + p, *sn = sinv + pos * HD + p;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // two products and a sum, each rounded: what the training trunk's rotation computes
                    y1[j] = __fadd_rn(__fmul_rn(x1[j], cs[j]), __fmul_rn(-x2[j], sn[j]));
                    y2[j] = __fadd_rn(__fmul_rn(x2[j], cs[j + kHalf]), __fmul_rn(x1[j], sn[j + kHalf]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) y1[j] = y2[j] = __int_as_float(0x7fc00000);
            }
            lo = pack8(y1);
            hi = pack8(y2);
        }
        auto put = [&](uint16_t *dst) {
            *reinterpret_cast<uint4 *>(dst + p) = lo;
            *reinterpret_cast<uint4 *>(dst + p + kHalf) = hi;
        };
        if (h < H) {
            put(q + (t * H + h) * HD);
            continue;
        }
        const int hk = (h - H) % Hk;
        const int64_t slot = load_index(slots, slot64, t);
        if (slot >= 0 && slot < n_slots) {
            const int64_t row = (((slot >> page_shift) * Hk + hk) << page_shift) + (slot & ((1 << page_shift) - 1));
            put((h < H + Hk ? kp : vp) + row * HD);
        }
        if (k && h < H + Hk) put(k + (t * Hk + hk) * HD);
    }
}

// ------------------------------------------------------------------ decode attention
// out[b, h] = sum_j softmax_j(scale q . k_j) v_j over the sequence's seq_lens[b] keys.
//
// Bound by reading the cache once. A CTA takes a chunk of one sequence's keys for the
// (up to 16) query heads that share a key head, so that a key is read once for all of
// them; its warps take tiles of 16 keys in turn, each through a ring of its own in
// shared memory (16-byte asynchronous copies, kStages tiles ahead, no barrier between
// warps), and keep a running maximum, sum and output per head. Scores and outputs are
// m16n8k16 products with the heads as rows: at one query per sequence the tensor pipe
// is idle whatever the shape, and one instruction serves 1 to 16 heads alike. The
// weights enter as two bf16 terms (p = hi + lo), which the idle pipe gives for free:
// the result is rounded once. Rows behind the sequence's end are zero-filled by the
// copy, so stale pages never reach a product. 64 sequences of 8192, 32 heads on 8 of 128:
// 325 us, 6.6 TB/s; 4 of 87000 to 131072, 16 heads on 4: 143 us, 6.2 TB/s; 48 of 64 to
// 4096, 16 heads of 64: 45 us, 4.3 TB/s (bound by the longest sequences' last chunks).
constexpr int kDecWarps = 4;
constexpr int kDecTile = 16;                      // keys of a warp's step
constexpr int kDecHeads = 16;                     // query heads of a CTA
constexpr int kDecMaxChunk = 4096;                // keys of a CTA

template <int HD>
struct Dec {
    static constexpr int kStages = 3;
    static constexpr int kRowBytes = HD * 2;
    static constexpr int kTileBytes = kDecTile * kRowBytes;
    static constexpr int kRing = kDecWarps * kStages * 2 * kTileBytes;
    // the ring, later the warps' outputs [warp][16][HD] fp32
    static constexpr int kOut = kDecWarps * kDecHeads * HD * 4;
    static constexpr int kSmem = (kRing > kOut ? kRing : kOut) + (kDecMaxChunk / 8 + 1) * 4;
};

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
    int64_t q_ld, table_ld, n_pages, max_len;
    int H, Hk, page_shift, chunk, n_chunks;
    float scale_log2;
    uint16_t *out;
    float *part;        // [b][h][chunk][m, l, HD] when n_chunks > 1
};

// Cluster: the chunks of a list are one cluster, which joins its own parts through its
// shared memory (no second launch, no workspace). For calls that fit the GPU at once:
// a CTA whose chunk the sequence does not reach stays for the join.
template <int HD, bool Cluster>
__global__ void __launch_bounds__(kDecWarps * 32)
decode_split_kernel(const __grid_constant__ DecodeArgs P) {
    using C = Dec<HD>;
    extern __shared__ __align__(128) unsigned char dsm[];
    __shared__ float s_m[kDecWarps][kDecHeads], s_l[kDecWarps][kDecHeads];
    __shared__ float2 s_part[kDecHeads];
    int32_t *s_page = reinterpret_cast<int32_t *>(dsm + C::kSmem - (kDecMaxChunk / 8 + 1) * 4);
    const int b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = P.H / P.Hk, groups = (G + kDecHeads - 1) / kDecHeads;
    const int hk = blockIdx.y / groups, g0 = blockIdx.y % groups * kDecHeads, nh = min(kDecHeads, G - g0);
    const int h0 = hk * G + g0;
    const int64_t j0 = static_cast<int64_t>(blockIdx.x) * P.chunk;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    // length, pages and queries are on their way together: the pages up to max_len are
    // read before the length is known
    const int page_mask = (1 << P.page_shift) - 1, off = static_cast<int>(j0) & page_mask;
    const int most = static_cast<int>(min(P.max_len - j0, static_cast<int64_t>(P.chunk)));
    const int pages_most = most > 0 ? ((off + most - 1) >> P.page_shift) + 1 : 0;
    const int32_t *row = P.table + b * P.table_ld + (j0 >> P.page_shift);
    const int32_t page0 = static_cast<int>(threadIdx.x) < pages_most ? row[threadIdx.x] : 0;
    // queries: row lane / 4 (+ 8), dimensions 16 kk + 2 (lane % 4) (+ 8)
    uint32_t qa[HD / 16][4];
    {
        const int r = lane >> 2, d = 2 * (lane & 3);
        const uint16_t *q0 = P.q + b * P.q_ld + static_cast<int64_t>(h0 + r) * HD + d;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                qa[kk][e] = r + 8 * (e & 1) < nh
                                ? *reinterpret_cast<const uint32_t *>(q0 + 8 * (e & 1) * HD + 16 * kk + 8 * (e >> 1))
                                : 0u;
    }
    const int64_t len = P.seq_lens[b];
    bool lost = len > P.max_len;
    if (!Cluster && P.n_chunks > 1 && j0 > 0 && (j0 >= len || lost)) return;      // the join does not look
    const int n = lost ? 0 : static_cast<int>(max(min(len - j0, static_cast<int64_t>(P.chunk)), static_cast<int64_t>(0)));
    // one page outside the cache makes the sequence's result NaN
    const int pages = n > 0 ? ((off + n - 1) >> P.page_shift) + 1 : 0;
    for (int i = threadIdx.x; i < pages; i += blockDim.x) {
        const int32_t p = i == static_cast<int>(threadIdx.x) ? page0 : row[i];
        if (p < 0 || p >= P.n_pages) lost = true;
        s_page[i] = p;
    }
    lost = __syncthreads_or(lost);

    float acc[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    const int tiles = lost ? 0 : (n + kDecTile - 1) / kDecTile;
    if (warp < tiles) {
        const uint32_t ring = smem_u32(dsm) + warp * C::kStages * 2 * C::kTileBytes;
        constexpr int kLanes = HD / 8;                // lanes of a row
        constexpr int kRowsPer = 32 / kLanes;         // rows of one copy instruction
        const int chunk_col = lane % kLanes, row0 = lane / kLanes;
        auto fetch = [&](int i, int stage) {
            if (i < tiles) {
                const uint32_t sk = ring + stage * 2 * C::kTileBytes, sv = sk + C::kTileBytes;
#pragma unroll
                for (int u = 0; u < kDecTile / kRowsPer; ++u) {
                    const int row = row0 + u * kRowsPer, j = i * kDecTile + row;
                    const bool in = j < n;
                    const int jc = off + (in ? j : 0);
                    const int64_t at = (((static_cast<int64_t>(s_page[jc >> P.page_shift]) * P.Hk + hk) << P.page_shift) +
                                        (jc & page_mask)) * HD + chunk_col * 8;
                    const uint32_t dst = swz(row, chunk_col, C::kRowBytes);
                    cp_async16(sk + dst, P.kp + at, in ? 16 : 0);
                    cp_async16(sv + dst, P.vp + at, in ? 16 : 0);
                }
            }
            cp_async_commit();
        };
        int head = 0;
#pragma unroll
        for (int s = 0; s < C::kStages - 1; ++s) fetch(warp + s * kDecWarps, s);
        for (int i = warp; i < tiles; i += kDecWarps) {
            cp_async_wait<C::kStages - 2>();
            __syncwarp();
            const uint32_t sk = ring + head * 2 * C::kTileBytes, sv = sk + C::kTileBytes;
            float s[2][4] = {};
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                uint32_t kb[4];
                ldmatrix_x4(kb, sk + swz((lane & 7) + (lane >> 4) * 8, 2 * kk + (lane >> 3 & 1), C::kRowBytes));
                mma_bf16_16816(s[0], qa[kk], kb[0], kb[1]);
                mma_bf16_16816(s[1], qa[kk], kb[2], kb[3]);
            }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = i * kDecTile + 8 * t + 2 * (lane & 3) + (e & 1) < n;
                    s[t][e] = in ? s[t][e] * P.scale_log2 : -INFINITY;
                    mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                mx[r] = fmaxf(mx[r], m[r]);
            }
            if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
                float f[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    f[r] = mx[r] > m[r] ? tc::ex2(m[r] - mx[r]) : 1.0f;
                    l[r] *= f[r];
                    m[r] = mx[r];
                }
#pragma unroll
                for (int d = 0; d < HD / 8; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][e] *= f[e >> 1];
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float ref = m[r] == -INFINITY ? 0.0f : m[r];
                    const float p0 = tc::ex2(s[t][2 * r] - ref), p1 = tc::ex2(s[t][2 * r + 1] - ref);
                    l[r] += p0 + p1;
                    const uint32_t h = pack_bf16x2(p0, p1);
                    hi[2 * t + r] = h;
                    lo[2 * t + r] = pack_bf16x2(p0 - __uint_as_float(h << 16), p1 - __uint_as_float(h & 0xffff0000u));
                }
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t vb[4];
                ldmatrix_x4_trans(vb, sv + swz((lane & 7) + (lane >> 3 & 1) * 8, 2 * d + (lane >> 4), C::kRowBytes));
                mma_bf16_16816(acc[2 * d], hi, vb[0], vb[1]);
                mma_bf16_16816(acc[2 * d + 1], hi, vb[2], vb[3]);
                mma_bf16_16816(acc[2 * d], lo, vb[0], vb[1]);
                mma_bf16_16816(acc[2 * d + 1], lo, vb[2], vb[3]);
            }
            __syncwarp();      // the stage that the next copy overwrites has been read
            const int ahead = i + (C::kStages - 1) * kDecWarps;
            fetch(ahead, head == 0 ? C::kStages - 1 : head - 1);
            head = head + 1 == C::kStages ? 0 : head + 1;
        }
        cp_async_wait<0>();
    }

    // join the warps: their maxima and sums, then the outputs through the ring's memory
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if ((lane & 3) == 0) {
            s_m[warp][(lane >> 2) + 8 * r] = m[r];
            s_l[warp][(lane >> 2) + 8 * r] = l[r];
        }
    }
    __syncthreads();
    float *s_o = reinterpret_cast<float *>(dsm);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int g = (lane >> 2) + 8 * r;
        if (g >= nh) continue;
        float M = s_m[0][g];
#pragma unroll
        for (int w = 1; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][g]);
        const float f = m[r] == -INFINITY ? 0.0f : tc::ex2(m[r] - M);
#pragma unroll
        for (int d = 0; d < HD / 8; ++d)
            *reinterpret_cast<float2 *>(s_o + (warp * kDecHeads + g) * HD + 8 * d + 2 * (lane & 3)) =
                make_float2(acc[d][2 * r] * f, acc[d][2 * r + 1] * f);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nh * (HD / 4); e += blockDim.x) {
        const int g = e / (HD / 4), d = e % (HD / 4) * 4;
        float M = s_m[0][g], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][g]);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
            // a warp whose maximum is -inf saw nothing, or NaN alone
            L += s_m[w][g] == -INFINITY ? s_l[w][g] : s_l[w][g] * tc::ex2(s_m[w][g] - M);
            const float4 x = *reinterpret_cast<const float4 *>(s_o + (w * kDecHeads + g) * HD + d);
            o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
        }
        if (lost) L = __int_as_float(0x7fc00000);
        const int64_t row = static_cast<int64_t>(b) * P.H + h0 + g;
        if constexpr (Cluster) {
            // this CTA's part stays where warp 0's outputs were
            *reinterpret_cast<float4 *>(s_o + g * HD + d) = o;
            if (d == 0) s_part[g] = make_float2(M, L);
        } else if (P.n_chunks == 1) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            *reinterpret_cast<uint2 *>(P.out + row * HD + d) =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        } else {
            float *dst = P.part + (row * P.n_chunks + blockIdx.x) * (HD + 4);
            *reinterpret_cast<float4 *>(dst + 4 + d) = o;
            if (d == 0) *reinterpret_cast<float2 *>(dst) = make_float2(M, L);
        }
    }
    if constexpr (Cluster) {
        cluster_sync();
        // pairs of columns, dealt out over the cluster's threads; parts in chunk order
        const int ctas = P.n_chunks, me = static_cast<int>(blockIdx.x);
        for (int e = me * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x); e < nh * (HD / 2);
             e += ctas * static_cast<int>(blockDim.x)) {
            const int g = e / (HD / 2), d = e % (HD / 2) * 2;
            float2 ml[kClusterMost], x[kClusterMost];
            float M = -INFINITY, L = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (int c = 0; c < kClusterMost; ++c) {
                ml[c] = make_float2(-INFINITY, 0.0f);
                x[c] = make_float2(0.0f, 0.0f);
                if (c < ctas) {
                    ml[c] = ld_cluster(&s_part[g], c);
                    x[c] = ld_cluster(reinterpret_cast<const float2 *>(s_o + g * HD + d), c);
                }
                M = fmaxf(M, ml[c].x);
            }
#pragma unroll
            for (int c = 0; c < kClusterMost; ++c) {
                // a chunk whose maximum is -inf saw no key, or NaN alone (its sum says so)
                const float f = ml[c].x == -INFINITY ? 0.0f : tc::ex2(ml[c].x - M);
                L += ml[c].x == -INFINITY ? ml[c].y : f * ml[c].y;
                o0 = fmaf(f, x[c].x, o0);
                o1 = fmaf(f, x[c].y, o1);
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            *reinterpret_cast<uint32_t *>(P.out + (static_cast<int64_t>(b) * P.H + h0 + g) * HD + d) =
                pack_bf16x2(o0 * inv, o1 * inv);
        }
        cluster_sync();      // nobody leaves while its part is read
    }
}

// Joins the parts of the chunks that a sequence has, per (sequence, head): a CTA of
// eight warps, each taking every eighth chunk, or (W = 1, few chunks) a warp.
constexpr int kJoinWarps = 8;
template <int HD, int W>
__global__ void __launch_bounds__(kJoinWarps * 32)
decode_join_kernel(const __grid_constant__ DecodeArgs P, int64_t rows) {
    constexpr int kD = HD / 32;
    __shared__ float s_m[kJoinWarps], s_l[kJoinWarps], s_o[kJoinWarps][HD];
    const int64_t r = W == 1 ? blockIdx.x * static_cast<int64_t>(kJoinWarps) + (threadIdx.x >> 5) : blockIdx.x;
    const int warp = W == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (r >= rows) return;
    const int64_t len = P.seq_lens[r / P.H];
    const int chunks = len > P.max_len ? 1 : static_cast<int>(max((len + P.chunk - 1) / P.chunk, static_cast<int64_t>(1)));
    const float *src = P.part + r * P.n_chunks * (HD + 4);
    asm volatile("griddepcontrol.wait;\n" ::: "memory");      // the parts are written
    // this warp's parts against its own maximum, all loads of a round under way at once
    float M = -INFINITY, L = 0.0f, o[kD] = {};
    constexpr int kRound = 8;
    for (int c0 = warp; c0 < chunks; c0 += kRound * W) {
        float2 ml[kRound];
        float x[kRound][kD];
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
            const int c = c0 + u * W;
            ml[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int d = 0; d < kD; ++d) x[u][d] = 0.0f;
            if (c < chunks) {
                const float *p = src + c * (HD + 4);
                ml[u] = *reinterpret_cast<const float2 *>(p);
#pragma unroll
                for (int d = 0; d < kD; d += 2)
                    *reinterpret_cast<float2 *>(&x[u][d]) = *reinterpret_cast<const float2 *>(p + 4 + lane * kD + d);
            }
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < kRound; ++u) top = fmaxf(top, ml[u].x);
        const float f = M == -INFINITY ? 0.0f : tc::ex2(M - top);
        L *= M == -INFINITY ? 1.0f : f;
        M = top;
#pragma unroll
        for (int d = 0; d < kD; ++d) o[d] *= f;
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
            // a chunk whose maximum is -inf saw no key, or NaN alone (its sum says so)
            const float g = ml[u].x == -INFINITY ? 0.0f : tc::ex2(ml[u].x - M);
            L += ml[u].x == -INFINITY ? ml[u].y : g * ml[u].y;
#pragma unroll
            for (int d = 0; d < kD; ++d) o[d] = fmaf(g, x[u][d], o[d]);
        }
    }
    if constexpr (W == 1) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int d = 0; d < kD; d += 2)
            *reinterpret_cast<uint32_t *>(P.out + r * HD + lane * kD + d) = pack_bf16x2(o[d] * inv, o[d + 1] * inv);
        return;
    }
    if (lane == 0) {
        s_m[warp] = M;
        s_l[warp] = L;
    }
#pragma unroll
    for (int d = 0; d < kD; ++d) s_o[warp][lane * kD + d] = o[d];
    __syncthreads();
    if (threadIdx.x >= HD / 2) return;
    const int d = 2 * threadIdx.x;
    float top = -INFINITY, x = 0.0f, y = 0.0f;
    L = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_m[w]);
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        const float g = s_m[w] == -INFINITY ? 0.0f : tc::ex2(s_m[w] - top);
        L += s_m[w] == -INFINITY ? s_l[w] : g * s_l[w];
        x = fmaf(g, s_o[w][d], x);
        y = fmaf(g, s_o[w][d + 1], y);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<uint32_t *>(P.out + r * HD + d) = pack_bf16x2(x * inv, y * inv);
}

}  // namespace

cudaError_t launch_rope_append(const void *qkv, int64_t ld, const float *cosv, const float *sinv, int64_t n_pos,
                               const void *positions, int pos64, const void *slots, int slot64, int64_t T, int H,
                               int Hk, int hd, int64_t n_pages, int page_shift, void *kp, void *vp, void *q, void *k,
                               cudaStream_t st) {
    const int64_t work = T * (H + 2 * Hk) * (hd / 16);
    const int grid = static_cast<int>(std::min<int64_t>((work + 255) / 256, 148 * 16));
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, st>>>(static_cast<const uint16_t *>(qkv), ld, cosv, sinv, n_pos, positions, pos64,
                                     slots, slot64, T, H, Hk, n_pages << page_shift, page_shift,
                                     static_cast<uint16_t *>(kp), static_cast<uint16_t *>(vp),
                                     static_cast<uint16_t *>(q), static_cast<uint16_t *>(k));
    };
    if (hd == 64) go(rope_append_kernel<64>);
    else go(rope_append_kernel<128>);
    count_launch();
    return cudaGetLastError();
}

// Keys of a chunk. The host knows only the longest length a sequence may have: about
// 12 CTAs an SM by that bound keep ragged batches level (48 sequences of 64 to 4096:
// 45 us, 57 with 6 an SM, 41 with 24; 4 of 131072: 142, 151, 156), but a CTA of under 512 keys pays more for its start and its
// part than it saves (8 sequences of 2048, 16 heads: 15 us with 512, 17 with 256),
// except where there would not be two CTAs an SM (1 sequence of 32768, 2 key heads:
// 13.7 us with 256, 18 with 512).
DecodeSplit decode_split(int64_t B, int64_t H, int64_t Hk, int64_t max_len) {
    DecodeSplit s;
    const int64_t G = H / std::max<int64_t>(Hk, 1), lists = B * Hk * ((G + kDecHeads - 1) / kDecHeads);
    const auto over = [&](int64_t ctas) { return (lists * max_len + ctas - 1) / ctas; };
    int64_t chunk = std::max(over(12 * 148), std::min<int64_t>(512, over(2 * 148)));
    chunk = std::min<int64_t>(std::max<int64_t>((chunk + 63) / 64 * 64, 64), kDecMaxChunk);
    // few short lists: as one cluster each, of up to 8 chunks of up to 512 keys
    if (lists * kClusterMost <= 2 * 148 && max_len <= kClusterMost * 512) {
        chunk = std::max<int64_t>((max_len + kClusterMost - 1) / kClusterMost, 64);
        chunk = (chunk + 63) / 64 * 64;
        s.cluster = true;
    }
    s.chunk = static_cast<int>(chunk);
    s.n_chunks = static_cast<int>(std::max<int64_t>(1, (max_len + s.chunk - 1) / s.chunk));
    s.cluster = s.cluster && s.n_chunks > 1;
    return s;
}

template <int HD>
static cudaError_t launch_decode(const DecodeArgs &p, const DecodeSplit &s, dim3 grid, int64_t rows, cudaStream_t st) {
    constexpr int smem = Dec<HD>::kSmem;
    static std::atomic<uint64_t> ready{0};      // devices whose kernels have their shared memory set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(decode_split_kernel<HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      smem)) != cudaSuccess ||
            (e = cudaFuncSetAttribute(decode_split_kernel<HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      smem)) != cudaSuccess)
            return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (s.cluster) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(kDecWarps * 32);
        cfg.dynamicSmemBytes = smem;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = static_cast<unsigned>(s.n_chunks);
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        e = cudaLaunchKernelEx(&cfg, decode_split_kernel<HD, true>, p);
        count_launch();
        return e;
    }
    decode_split_kernel<HD, false><<<grid, kDecWarps * 32, smem, st>>>(p);
    count_launch();
    e = cudaGetLastError();
    if (e != cudaSuccess || s.n_chunks == 1) return e;
    // the join's launch overlaps the split's end; its threads wait for the parts
    const bool few = s.n_chunks <= 2 || (s.n_chunks <= 16 && rows >= 1024);
    cfg.gridDim = dim3(static_cast<unsigned>(few ? (rows + kJoinWarps - 1) / kJoinWarps : rows));
    cfg.blockDim = dim3(kJoinWarps * 32);
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    e = few ? cudaLaunchKernelEx(&cfg, decode_join_kernel<HD, 1>, p, rows)
            : cudaLaunchKernelEx(&cfg, decode_join_kernel<HD, 8>, p, rows);
    count_launch();
    return e;
}

cudaError_t launch_decode_attn(const void *q, int64_t q_ld, const void *kp, const void *vp, int64_t n_pages,
                               int page_shift, const int32_t *table, int64_t table_ld, const int32_t *seq_lens,
                               int64_t max_len, int64_t B, int H, int Hk, int hd, float scale, void *out, float *part,
                               cudaStream_t st) {
    const DecodeSplit s = decode_split(B, H, Hk, max_len);
    const int G = H / Hk;
    const dim3 grid(s.n_chunks, Hk * ((G + kDecHeads - 1) / kDecHeads), static_cast<unsigned>(B));
    DecodeArgs p;
    p.q = static_cast<const uint16_t *>(q);
    p.kp = static_cast<const uint16_t *>(kp);
    p.vp = static_cast<const uint16_t *>(vp);
    p.table = table;
    p.seq_lens = seq_lens;
    p.q_ld = q_ld;
    p.table_ld = table_ld;
    p.n_pages = n_pages;
    p.max_len = max_len;
    p.H = H;
    p.Hk = Hk;
    p.page_shift = page_shift;
    p.chunk = s.chunk;
    p.n_chunks = s.n_chunks;
    p.scale_log2 = scale * kLog2e;
    p.out = static_cast<uint16_t *>(out);
    p.part = part;
    return hd == 64 ? launch_decode<64>(p, s, grid, B * H, st) : launch_decode<128>(p, s, grid, B * H, st);
}

}  // namespace mom
