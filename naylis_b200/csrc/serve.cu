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
// Bound by reading the cache once. A list is a sequence's key head with the (up to 16)
// query heads that share it, so that a key is read once for all of them. The lists' tiles
// of 16 keys, one list after another, are cut into one span for each CTA that fits the GPU;
// only the device knows the lengths, so each CTA finds its span from their running sum. A
// CTA's warps take its tiles in turn, each through a ring of its own in shared memory
// (16-byte asynchronous copies, kStages tiles ahead whatever list they are of, no barrier
// between warps), and keep a running maximum, sum and output per head until the list ends.
// Scores and outputs are m16n8k16 products with the heads as rows: at one query per
// sequence the tensor pipe is idle whatever the shape, and one instruction serves 1 to 16
// heads alike. The weights enter as two bf16 terms (p = hi + lo, to 2^-16 of p), which the
// idle pipe gives for free: the result is rounded once. Rows behind the sequence's end are zero-filled by
// the copy, so stale pages never reach a product. With the join: 64 sequences of 8192, 32
// heads on 8 of 128: 316 us, 6.8 TB/s (326 with a CTA for each chunk of a list); 4 of 87000 to
// 131072, 16 heads on 4: 135 us, 6.6 TB/s (143); 128 of 1024, 32 on 8: 91 us, 5.9 TB/s (99);
// 48 of 64 to 4096, 16 heads of 64: 44 us, 4.5 TB/s (46): the spans begin to read after 3.5 us
// and end after 30 to 40, an SM's first CTA before its fourth (further, shorter spans for
// the SMs that are done first: 47 to 52; spans after the CTA's place: 46).
constexpr int kDecWarps = 4;
constexpr int kDecTile = 16;                      // keys of a warp's step
constexpr int kDecHeads = 16;                     // query heads of a CTA
constexpr int kDecLeast = 8;                      // tiles of a CTA's span, at least
// tiles that a list's start and end cost (48 sequences of 64 to 4096: 43 us with 6, 47 with 3, 44 with 10)
constexpr int kDecListCost = 6;

template <int HD>
struct Dec {
    static constexpr int kStages = 3;
    static constexpr int kCtas = HD == 64 ? 4 : 2;    // resident on an SM
    static constexpr int kRowBytes = HD * 2;
    static constexpr int kTileBytes = kDecTile * kRowBytes;
    static constexpr int kRing = kDecWarps * kStages * 2 * kTileBytes;
    // the warps' outputs, four heads at a time: [warp][4][HD] fp32
    static constexpr int kSmem = kRing + kDecWarps * 4 * HD * 4;
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
    int64_t q_ld, table_ld, n_pages, max_len, B;
    int H, Hk, page_shift, n_chunks, chunk;     // n_chunks, chunk (keys): a cluster's
    float scale_log2;
    uint16_t *out;
    float *part;        // [part][head of the CTA][m, l, -, -, HD]
    int2 *cut;          // where lists are cut, by the smaller of the two: [list] its first CTA and its number of
                        // CTAs, or [CTA] the list that begins in its span and ends behind it, and its number
    bool by_list;
};

// A sequence's keys as the kernels take them, and its tiles: one without keys for a
// sequence without (its output is zero) and for one that is too long (NaN).
struct DecLen {
    int n, tiles;
    bool lost;
    __device__ __forceinline__ DecLen(int32_t len, int64_t max_len) {
        lost = len > max_len;
        n = lost || len < 0 ? 0 : len;
        tiles = max(static_cast<int>((static_cast<unsigned>(n) + kDecTile - 1) / kDecTile), 1);
    }
};

// The work of all lists (a sequence's key head), one after another, cut into equal spans
// for the grid's CTAs. It is counted in tiles, and a list's start and end as kDecListCost
// of them ahead of its own. Where span blockIdx.x begins:
struct DecSpan {
    int64_t base, span;          // units before the list that it begins in, and units of a span
    int b, y, i, n;              // sequence, list of it, tile of that, the sequence's length
    int end;                     // the span's end, in units from base
};
__device__ __forceinline__ bool decode_span(const DecodeArgs &P, int lists, DecSpan &got) {
    __shared__ int64_t s_sum[kDecWarps];
    __shared__ DecSpan s_got;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int per = static_cast<int>((P.B + kDecWarps * 32 - 1) / (kDecWarps * 32));      // sequences of a thread
    const int64_t b0 = static_cast<int64_t>(t) * per, b1 = min(b0 + per, P.B);
    int64_t mine = 0;
    for (int64_t b = b0; b < b1; ++b) mine += DecLen(P.seq_lens[b], P.max_len).tiles + kDecListCost;
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
    const int64_t span = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(kDecLeast));
    const int64_t from = blockIdx.x * span;
    if (from >= total) return false;
    int64_t base = (upto - mine) * lists;
    if (from >= base && from < upto * lists) {
        for (int64_t b = b0; b < b1; ++b) {
            const int32_t len = P.seq_lens[b];
            const int units = DecLen(len, P.max_len).tiles + kDecListCost;
            const int64_t next = base + static_cast<int64_t>(units) * lists;
            if (from < next) {
                const int y = static_cast<int>((from - base) / units);
                base += static_cast<int64_t>(y) * units;
                s_got = {base, span, static_cast<int>(b), y, max(static_cast<int>(from - base) - kDecListCost, 0), len,
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

// Cluster: the chunks of a list are one cluster, which joins its own parts through its
// shared memory (no second launch, no workspace). For calls that fit the GPU at once:
// a CTA whose chunk the sequence does not reach stays for the join.
template <int HD, bool Cluster>
__global__ void __launch_bounds__(kDecWarps * 32, Dec<HD>::kCtas)
decode_split_kernel(const __grid_constant__ DecodeArgs P) {
    using C = Dec<HD>;
    extern __shared__ __align__(128) unsigned char dsm[];
    __shared__ float s_m[kDecWarps][kDecHeads], s_l[kDecWarps][kDecHeads];
    __shared__ float2 s_part[kDecHeads];
    float *s_o = reinterpret_cast<float *>(dsm + C::kRing);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = P.H / P.Hk, groups = (G + kDecHeads - 1) / kDecHeads, lists = P.Hk * groups;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    DecSpan at;
    if constexpr (Cluster) {
        const int first = static_cast<int>(blockIdx.x) * P.chunk / kDecTile;
        at = {0, 0, static_cast<int>(blockIdx.z), static_cast<int>(blockIdx.y), first, P.seq_lens[blockIdx.z],
              first + P.chunk / kDecTile + kDecListCost};
    } else if (!decode_span(P, lists, at)) {
        if (threadIdx.x == 0 && !P.by_list) P.cut[blockIdx.x] = make_int2(0, 0);
        return;
    }
    DecLen len(at.n, P.max_len);
    // the tiles of a list that are before the span's end
    const int end = at.end;
    const auto tiles_to = [&](int base, int tiles) { return max(min(tiles, end - base - kDecListCost), 0); };

    // The copies' side of this warp: it takes every fourth tile of the span, whatever list
    // it is of. The page numbers of a tile are read while the copies of the one before it
    // are issued. A tile starts at a multiple of 16 keys: it lies in one page, or in two of
    // 8. A page outside the cache copies nothing and makes the sequence's result NaN.
    const uint32_t ring = smem_u32(dsm) + warp * C::kStages * 2 * C::kTileBytes;
    constexpr int kLanes = HD / 8;                // lanes of a row
    constexpr int kRowsPer = 32 / kLanes;         // rows of one copy instruction
    const int chunk_col = lane % kLanes, row0 = lane / kLanes;
    const int page_mask = (1 << P.page_shift) - 1;
    int fbase = 0, fb = at.b, fy = at.y, fhk = fy / groups, fi = at.i, fn = len.n, fall = len.tiles;
    int fend = tiles_to(fbase, fall);
    int32_t flen = !Cluster && fb + 1 < P.B ? P.seq_lens[fb + 1] : 0;      // the next sequence's
    struct Tile {
        int32_t page[2];
        int rows, in_page, hk;      // rows: of the sequence; < 0: no tile
    };
    bool more = true, bad[C::kStages] = {};
    auto look = [&](int step) {
        Tile tile = {{0, 0}, -1, 0, 0};
        if (!more) return tile;
        fi += step;
        while (fi >= fend) {
            fi -= fend;
            fbase += fall + kDecListCost;
            if (Cluster || fbase + kDecListCost >= end) {
                more = false;
                return tile;
            }
            if (++fy == lists) {
                fy = 0;
                ++fb;
                const DecLen next(flen, P.max_len);
                fn = next.n, fall = next.tiles;
                flen = fb + 1 < P.B ? P.seq_lens[fb + 1] : 0;
            }
            fhk = fy / groups;
            fend = tiles_to(fbase, fall);
        }
        tile.rows = min(fn - fi * kDecTile, kDecTile);
        tile.in_page = (fi * kDecTile) & page_mask;
        tile.hk = fhk;
        if (tile.rows > 0) {
            const int32_t *row = P.table + fb * P.table_ld;
            const int64_t j = static_cast<int64_t>(fi) * kDecTile;
            tile.page[0] = row[j >> P.page_shift];
            tile.page[1] = tile.rows > 8 ? row[(j + 8) >> P.page_shift] : tile.page[0];
        }
        return tile;
    };
    auto fetch = [&](int stage, const Tile &tile) {
        if (tile.rows >= 0) {
            const uint32_t sk = ring + stage * 2 * C::kTileBytes, sv = sk + C::kTileBytes;
            const bool out = tile.rows > 0 && (tile.page[0] < 0 || tile.page[0] >= P.n_pages || tile.page[1] < 0 ||
                                               tile.page[1] >= P.n_pages);
#pragma unroll
            for (int e = 0; e < C::kStages; ++e)
                if (e == stage) bad[e] = out;
#pragma unroll
            for (int u = 0; u < kDecTile / kRowsPer; ++u) {
                const int r = row0 + u * kRowsPer;
                const bool in = !out && r < tile.rows;
                const int64_t from = (((static_cast<int64_t>(tile.page[r >> 3]) * P.Hk + tile.hk) << P.page_shift) +
                                      ((tile.in_page + r) & page_mask)) * HD + chunk_col * 8;
                const uint32_t dst = swz(r, chunk_col, C::kRowBytes);
                cp_async16(sk + dst, in ? P.kp + from : P.q, in ? 16 : 0);      // zeros behind the end
                cp_async16(sv + dst, in ? P.vp + from : P.q, in ? 16 : 0);
            }
        }
        cp_async_commit();
    };
    int head = 0;
    static_assert(C::kStages == 3);
    const Tile tile0 = look(warp), tile1 = look(kDecWarps);      // both tables' reads under way together
    fetch(0, tile0);
    fetch(1, tile1);
    Tile tile = look(kDecWarps);

    // The products' side, list by list.
    int b = at.b, y = at.y, i0 = at.i, taken = 0;
    // queries: row lane / 4 (+ 8), dimensions 16 kk + 2 (lane % 4) (+ 8)
    uint32_t qa[HD / 16][4];
    auto queries = [&](int qb, int qy) {
        const int r = lane >> 2, d = 2 * (lane & 3), g0 = qy % groups * kDecHeads, nh = min(kDecHeads, G - g0);
        const uint16_t *q0 = P.q + qb * P.q_ld + static_cast<int64_t>(qy / groups * G + g0 + r) * HD + d;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                qa[kk][e] = r + 8 * (e & 1) < nh
                                ? *reinterpret_cast<const uint32_t *>(q0 + 8 * (e & 1) * HD + 16 * kk + 8 * (e >> 1))
                                : 0u;
    };
    queries(b, y);
    int2 cut = make_int2(0, 0);
    for (int base = 0; Cluster || base + kDecListCost < end;) {
        const int g0 = y % groups * kDecHeads, nh = min(kDecHeads, G - g0), h0 = y / groups * G + g0;
        const int tiles = tiles_to(base, len.tiles) - i0;
        bool lost = len.lost;
        float acc[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
        for (int i = (warp - taken) & (kDecWarps - 1); i < tiles; i += kDecWarps) {
            cp_async_wait<C::kStages - 2>();
            __syncwarp();
#pragma unroll
            for (int e = 0; e < C::kStages; ++e)
                if (e == head) lost |= bad[e];
            const int n = len.n - (i0 + i) * kDecTile;
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
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = 8 * u + 2 * (lane & 3) + (e & 1) < n;
                    s[u][e] = in ? s[u][e] * P.scale_log2 : -INFINITY;
                    mx[e >> 1] = fmaxf(mx[e >> 1], s[u][e]);
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
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float ref = m[r] == -INFINITY ? 0.0f : m[r];
                    const float p0 = tc::ex2(s[u][2 * r] - ref), p1 = tc::ex2(s[u][2 * r + 1] - ref);
                    l[r] += p0 + p1;
                    // hi is cut, not rounded, and lo above 0: an infinite value has the same sign in both
                    // products. (2^-126 is below a weight's last bit wherever the value is finite.)
                    const float c0 = __uint_as_float(__float_as_uint(p0) & 0xffff0000u);
                    const float c1 = __uint_as_float(__float_as_uint(p1) & 0xffff0000u);
                    hi[2 * u + r] = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
                    lo[2 * u + r] = pack_bf16x2(fmaxf(p0 - c0, 0x1p-126f), fmaxf(p1 - c1, 0x1p-126f));
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
            fetch(head == 0 ? C::kStages - 1 : head - 1, tile);
            tile = look(kDecWarps);
            head = head + 1 == C::kStages ? 0 : head + 1;
        }

        // the next list, and its queries on their way
        const int next = base + len.tiles + kDecListCost;
        int32_t blen = 0;
        int ny = y + 1, nb = b;
        if (ny == lists) ny = 0, ++nb;
        if (!Cluster && next + kDecListCost < end) {
            queries(nb, ny);
            if (nb != b) blen = P.seq_lens[nb];
        }

        // join the warps: their maxima and sums, then the outputs of four heads at a time
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if ((lane & 3) == 0) {
                s_m[warp][(lane >> 2) + 8 * r] = m[r];
                s_l[warp][(lane >> 2) + 8 * r] = l[r];
            }
        }
        lost = __syncthreads_or(lost);
        const int64_t list = static_cast<int64_t>(b) * lists + y;
        const bool whole = i0 == 0 && tiles == len.tiles;
#pragma unroll
        for (int p = 0; p < kDecHeads / 4; ++p) {
            if (4 * p >= nh) break;
            const int r = p >> 1, g = (lane >> 2) + 8 * r;
            if (g >> 2 == p && g < nh) {
                float M = s_m[0][g];
#pragma unroll
                for (int w = 1; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][g]);
                const float f = m[r] == -INFINITY ? 0.0f : tc::ex2(m[r] - M);
#pragma unroll
                for (int d = 0; d < HD / 8; ++d)
                    *reinterpret_cast<float2 *>(s_o + (warp * 4 + (g & 3)) * HD + 8 * d + 2 * (lane & 3)) =
                        make_float2(acc[d][2 * r] * f, acc[d][2 * r + 1] * f);
            }
            __syncthreads();
            const int left = min(nh - 4 * p, 4) * (HD / 4);
            for (int e = threadIdx.x; e < left; e += blockDim.x) {
                const int g = 4 * p + e / (HD / 4), d = e % (HD / 4) * 4;
                float M = s_m[0][g], L = 0.0f;
#pragma unroll
                for (int w = 1; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][g]);
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w) {
                    // a warp whose maximum is -inf saw nothing, or NaN alone
                    L += s_m[w][g] == -INFINITY ? s_l[w][g] : s_l[w][g] * tc::ex2(s_m[w][g] - M);
                    const float4 x = *reinterpret_cast<const float4 *>(s_o + (w * 4 + (g & 3)) * HD + d);
                    o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
                }
                if (lost) L = __int_as_float(0x7fc00000);
                if constexpr (Cluster) {
                    // this CTA's part stays where the ring was
                    *reinterpret_cast<float4 *>(reinterpret_cast<float *>(dsm) + g * HD + d) = o;
                    if (d == 0) s_part[g] = make_float2(M, L);
                } else if (whole) {
                    const float inv = len.n == 0 && !lost ? 0.0f : 1.0f / L;
                    *reinterpret_cast<uint2 *>(P.out + (static_cast<int64_t>(b) * P.H + h0 + g) * HD + d) =
                        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                } else {
                    // a CTA and a list that follow one another in the order of tiles: no two
                    // parts have the same sum
                    float *dst = P.part + ((blockIdx.x + list) * min(G, kDecHeads) + g) * (HD + 4);
                    *reinterpret_cast<float4 *>(dst + 4 + d) = o;
                    if (d == 0) *reinterpret_cast<float2 *>(dst) = make_float2(M, L);
                }
            }
            __syncthreads();
        }
        if constexpr (Cluster) break;
        if (i0 == 0 && threadIdx.x == 0) {
            const int n = static_cast<int>((at.base + next - 1) / at.span) - static_cast<int>(blockIdx.x) + 1;
            if (P.by_list) P.cut[list] = make_int2(blockIdx.x, n);
            else if (n > 1) cut = make_int2(static_cast<int>(list), n);
        }
        taken += tiles;
        base = next;
        i0 = 0;
        y = ny;
        if (nb != b) {
            b = nb;
            len = DecLen(blen, P.max_len);
        }
    }
    if (!Cluster && threadIdx.x == 0 && !P.by_list) P.cut[blockIdx.x] = cut;
    if constexpr (Cluster) {
        cluster_sync();
        // pairs of columns, dealt out over the cluster's threads; parts in chunk order
        const int ctas = P.n_chunks, me = static_cast<int>(blockIdx.x);
        const int g0 = y % groups * kDecHeads, nh = min(kDecHeads, G - g0), h0 = y / groups * G + g0;
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
                    x[c] = ld_cluster(reinterpret_cast<const float2 *>(reinterpret_cast<float *>(dsm) + g * HD + d), c);
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
            const float inv = len.n == 0 && !len.lost ? 0.0f : 1.0f / L;
            *reinterpret_cast<uint32_t *>(P.out + (static_cast<int64_t>(b) * P.H + h0 + g) * HD + d) =
                pack_bf16x2(o0 * inv, o1 * inv);
        }
        cluster_sync();      // nobody leaves while its part is read
    }
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
template <int HD, bool Wide>
__global__ void __launch_bounds__(Wide ? 512 : 128, Wide ? 2 : 10)
decode_join_kernel(const __grid_constant__ DecodeArgs P) {
    constexpr int kThreads = Wide ? 512 : 128, kLanes = Wide ? 8 : HD / 4, kGroups = kThreads / kLanes, kRound = 4;
    __shared__ DecSum s_sum[kThreads / 32][kLanes];
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, warp = threadIdx.x / 32;
    const int d = (static_cast<int>(blockIdx.z) * kLanes + lane) * 4;
    const int G = P.H / P.Hk, per = min(G, kDecHeads), groups = (G + kDecHeads - 1) / kDecHeads, lists = P.Hk * groups;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");      // the parts are written
    const int2 cut = P.cut[blockIdx.x];
    const int list = P.by_list ? blockIdx.x : cut.x, cta = P.by_list ? cut.x : blockIdx.x;
    const int y = list % lists, h = y / groups * G + y % groups * kDecHeads + static_cast<int>(blockIdx.y);
    if (cut.y <= 1 || h >= (y / groups + 1) * G) return;
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
    *reinterpret_cast<uint2 *>(P.out + (static_cast<int64_t>(list / lists) * P.H + h) * HD + d) =
        make_uint2(pack_bf16x2(sum.o.x * inv, sum.o.y * inv), pack_bf16x2(sum.o.z * inv, sum.o.w * inv));
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

DecodeSplit decode_split(int64_t B, int64_t H, int64_t Hk, int64_t hd, int64_t max_len) {
    DecodeSplit s;
    const int64_t G = H / std::max<int64_t>(Hk, 1), lists = B * Hk * ((G + kDecHeads - 1) / kDecHeads);
    const int64_t resident = static_cast<int64_t>(device_sm_count()) * (hd == 64 ? Dec<64>::kCtas : Dec<128>::kCtas);
    // few short lists: as one cluster each, of up to 8 chunks of up to 512 keys (8 sequences of
    // 2048, 16 heads of 64: 16 us, 21 in spans with a join)
    const int64_t most = std::min<int64_t>(kClusterMost, resident / std::max<int64_t>(lists, 1));
    if (most > 0 && max_len <= most * 512) {
        const int64_t chunk = std::max<int64_t>((max_len + most - 1) / most, 64);
        s.chunk = static_cast<int>((chunk + 63) / 64 * 64);
        s.n_chunks = static_cast<int>(std::max<int64_t>(1, (max_len + s.chunk - 1) / s.chunk));
        s.cluster = true;
        return s;
    }
    s.ctas = resident;
    s.ctas = std::min(s.ctas, lists * std::max<int64_t>((max_len + kDecTile * kDecLeast - 1) / (kDecTile * kDecLeast), 1));
    s.lists = lists;
    return s;
}

template <int HD>
static cudaError_t launch_decode(const DecodeArgs &p, const DecodeSplit &s, dim3 grid, cudaStream_t st) {
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
    if (e != cudaSuccess) return e;
    // the join's launch overlaps the split's end; its threads wait for the parts
    const bool wide = s.ctas > 8 * s.lists;
    cfg.blockDim = dim3(wide ? 512 : 128);
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(s.ctas, s.lists)), std::min(p.H / p.Hk, kDecHeads), wide ? HD / 32 : 1);
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    e = wide ? cudaLaunchKernelEx(&cfg, decode_join_kernel<HD, true>, p)
             : cudaLaunchKernelEx(&cfg, decode_join_kernel<HD, false>, p);
    count_launch();
    return e;
}

cudaError_t launch_decode_attn(const void *q, int64_t q_ld, const void *kp, const void *vp, int64_t n_pages,
                               int page_shift, const int32_t *table, int64_t table_ld, const int32_t *seq_lens,
                               int64_t max_len, int64_t B, int H, int Hk, int hd, float scale, void *out, float *part,
                               cudaStream_t st) {
    const DecodeSplit s = decode_split(B, H, Hk, hd, max_len);
    const int G = H / Hk;
    const unsigned lists = Hk * ((G + kDecHeads - 1) / kDecHeads);
    const dim3 grid = s.cluster ? dim3(s.n_chunks, lists, static_cast<unsigned>(B)) : dim3(static_cast<unsigned>(s.ctas));
    DecodeArgs p = {};
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
    p.B = B;
    p.chunk = s.chunk;
    p.n_chunks = s.n_chunks;
    p.scale_log2 = scale * kLog2e;
    p.out = static_cast<uint16_t *>(out);
    p.part = part;
    // the parts, then the CTAs' cut lists
    p.by_list = s.lists <= s.ctas;
    p.cut = s.cluster ? nullptr : reinterpret_cast<int2 *>(part + s.part_floats(H, Hk, hd));
    return hd == 64 ? launch_decode<64>(p, s, grid, st) : launch_decode<128>(p, s, grid, st);
}

}  // namespace mom
