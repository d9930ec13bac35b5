// A paged key-value cache in 4 bits: the rotary embedding that files into it, and the
// attention of one or several new tokens of each sequence over it.
//
// A row (a token's key or value of one head) is cut into groups of 64 values. A group
// keeps zero = its least value and scale = bf16((greatest - least) fp32(1 / 15)), and of each
// value x the number n = round((x - zero) / scale), 0 .. 15; it stands for zero + n scale.
// Pages (num_pages, Hk, page_size, hd / 2) bytes, the even dimension in a byte's low half;
// scales (num_pages, Hk, page_size, hd / 64, 4) bf16: the key's scale and zero, the
// value's. A row of hd 64 is 36 bytes, of hd 128 72: 9/32 of bf16.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "decode.cuh"

namespace mom {

namespace {

// ------------------------------------------------------------------ rope_append
// A thread takes 8 rotation pairs of a token, in Heads heads that follow one another: it reads
// its part of the tables once, and all of its heads' values before it computes. The threads
// of a group find its range by shuffles among themselves, on the packed bf16 values. The
// quotient is the reciprocal's product, corrected once (Markstein, 1990): rounded as a
// division is, in 3 operations. Bound by memory: 8 x 2048 tokens of 16 + 2 x 4 heads of 128, with
// k and v handed back: 40 us, 5.3 TB/s; 48 tokens of 48 heads of 64: 2.2 us.
constexpr int kAppendThreads = 128;

__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void load8(float (&f)[8], const float *p) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// A group as its values are divided: scaled by a power of two so that neither the divisor nor
// its reciprocal leaves fp32's normal numbers.
struct Int4Group {
    float least, step;
    float scale, from, by, inv, most;      // (x scale - from) / by, at most `most`
    __device__ __forceinline__ Int4Group() {}
    __device__ __forceinline__ Int4Group(float least_, float range) {
        least = least_;
        step = round_bf16(__fmul_rn(range, 1.0f / 15.0f));
        // a value that is not finite (the least or the greatest then is not), or a range beyond fp32: the group stands for NaN
        if (!(range < INFINITY)) step = least = __int_as_float(0x7fc00000);
        const bool some = step > 0.0f;
        scale = step < 1e-30f ? 0x1p100f : step > 1e30f ? 0x1p-100f : 1.0f;
        from = least * scale;
        by = step * scale;
        inv = some ? __frcp_rn(by) : 0.0f;
        most = some ? 15.0f : 0.0f;
    }
};

// Eight values of a group to their numbers, packed, and to what they stand for.
__device__ __forceinline__ uint32_t to_int4(const uint4 &v, const Int4Group &g, uint4 &stands) {
    constexpr float kMagic = 12582912.0f;      // 1.5 2^23: the sum's low bits are the rounded number
    float x[8];
    unpack8(v, x);
    uint32_t word = 0;
#pragma unroll
    for (int j = 7; j >= 0; --j) {
        const float a = __fmaf_rn(x[j], g.scale, -g.from);      // the difference, rounded once
        float q = __fmul_rn(a, g.inv);
        q = __fmaf_rn(__fmaf_rn(-q, g.by, a), g.inv, q);
        const float n = __fadd_rn(fminf(q, g.most), kMagic);      // (NaN: 0)
        word = word * 16 + __float_as_uint(n);
        x[j] = __fmaf_rn(__fsub_rn(n, kMagic), g.step, g.least);      // the product is exact
    }
    stands = pack8(x);
    return word - 0x3f400000u;      // of the sums' bits, 0x4b400000 + n, the constant part
}

template <int HD, int Heads>
__global__ void __launch_bounds__(kAppendThreads, Heads == 1 ? 8 : 6)
rope_append_int4_kernel(const uint16_t *__restrict__ qkv, int64_t ld, const float *__restrict__ cosv,
                        const float *__restrict__ sinv, int64_t n_pos, const void *__restrict__ positions, int pos64,
                        const void *__restrict__ slots, int slot64, int64_t T, int H, int Hk, int64_t n_slots,
                        int page_shift, uint8_t *__restrict__ kp, uint8_t *__restrict__ vp,
                        uint16_t *__restrict__ scales, uint16_t *__restrict__ q, uint16_t *__restrict__ k,
                        uint16_t *__restrict__ v) {
    constexpr int kHalf = HD / 2, kMates = kHalf / 8, kGroups = HD / 64;      // kMates: threads of a head
    const int heads = H + 2 * Hk, spans = (heads + Heads - 1) / Heads;
    const int64_t t = static_cast<int64_t>(blockIdx.x / spans) * (kAppendThreads / kMates) + threadIdx.x / kMates;
    const int h0 = static_cast<int>(blockIdx.x % spans) * Heads, p = static_cast<int>(threadIdx.x) % kMates * 8;
    if (t >= T) return;      // all of a head's threads
    const uint32_t mates = ((1u << kMates) - 1) << (threadIdx.x & 31 & ~(kMates - 1));
    const uint16_t *src = qkv + t * ld + static_cast<int64_t>(h0) * HD + p;
    uint4 lo[Heads], hi[Heads];
#pragma unroll
    for (int i = 0; i < Heads; ++i)
        if (h0 + i < heads) {
            lo[i] = *reinterpret_cast<const uint4 *>(src + i * HD);
            hi[i] = *reinterpret_cast<const uint4 *>(src + i * HD + kHalf);
        }
    float c1[8], c2[8], s1[8], s2[8];
    if (h0 < H + Hk) {
        const int64_t pos = load_index(positions, pos64, t);
        if (pos >= 0 && pos < n_pos) {
            load8(c1, cosv + pos * HD + p);
            load8(c2, cosv + pos * HD + p + kHalf);
            load8(s1, sinv + pos * HD + p);
            load8(s2, sinv + pos * HD + p + kHalf);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) c1[j] = c2[j] = s1[j] = s2[j] = __int_as_float(0x7fc00000);
        }
    }
    int64_t slot = -1;
    if (h0 + Heads > H) slot = load_index(slots, slot64, t);
#pragma unroll
    for (int i = 0; i < Heads; ++i) {
        const int h = h0 + i;
        if (h >= heads) break;
        if (h < H + Hk) {
            float x1[8], x2[8], y1[8], y2[8];
            unpack8(lo[i], x1);
            unpack8(hi[i], x2);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // two products and a sum, each rounded: what the training trunk's rotation computes
                y1[j] = __fadd_rn(__fmul_rn(x1[j], c1[j]), __fmul_rn(-x2[j], s1[j]));
                y2[j] = __fadd_rn(__fmul_rn(x2[j], c2[j]), __fmul_rn(x1[j], s2[j]));
            }
            lo[i] = pack8(y1);
            hi[i] = pack8(y2);
            if (h < H) {
                uint16_t *dst = q + (t * H + h) * HD + p;
                *reinterpret_cast<uint4 *>(dst) = lo[i];
                *reinterpret_cast<uint4 *>(dst + kHalf) = hi[i];
                continue;
            }
        }
        // the range of each group: at hd 64 one of all, at hd 128 one of each half of the row
        const uint4 x[2] = {lo[i], hi[i]};
        Int4Group group[2];
        uint32_t mn[2], mx[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            mn[s] = min2(min2(x[s].x, x[s].y), min2(x[s].z, x[s].w));
            mx[s] = max2(max2(x[s].x, x[s].y), max2(x[s].z, x[s].w));
        }
        if (kGroups == 1) mn[0] = min2(mn[0], mn[1]), mx[0] = max2(mx[0], mx[1]);
#pragma unroll
        for (int s = 0; s < kGroups; ++s) {
#pragma unroll
            for (int o = 1; o < kMates; o <<= 1) {
                mn[s] = min2(mn[s], __shfl_xor_sync(mates, mn[s], o));
                mx[s] = max2(mx[s], __shfl_xor_sync(mates, mx[s], o));
            }
            const float least = __uint_as_float(min2(mn[s], mn[s] >> 16) << 16);
            group[s] = Int4Group(least, __fsub_rn(__uint_as_float(max2(mx[s], mx[s] >> 16) << 16), least));
        }
        if (kGroups == 1) group[1] = group[0];
        uint4 stands[2];
        uint32_t word[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) word[s] = to_int4(x[s], group[s], stands[s]);
        const bool value = h >= H + Hk;
        const int hk = h - H - (value ? Hk : 0);
        if (slot >= 0 && slot < n_slots) {
            const int64_t row = (((slot >> page_shift) * Hk + hk) << page_shift) + (slot & ((1 << page_shift) - 1));
            uint8_t *dst = (value ? vp : kp) + row * (HD / 2) + p / 2;
            *reinterpret_cast<uint32_t *>(dst) = word[0];
            *reinterpret_cast<uint32_t *>(dst + kHalf / 2) = word[1];
            if (p < 8 * kGroups)      // the head's first thread, or its first two: a group each
                *reinterpret_cast<uint32_t *>(scales + (row * kGroups + p / 8) * 4 + (value ? 2 : 0)) =
                    pack_bf16x2(p == 0 ? group[0].step : group[1].step, p == 0 ? group[0].least : group[1].least);
        }
        if (uint16_t *to = value ? v : k) {
            uint16_t *dst = to + (t * Hk + hk) * HD + p;
            *reinterpret_cast<uint4 *>(dst) = stands[0];
            *reinterpret_cast<uint4 *>(dst + kHalf) = stands[1];
        }
    }
}

// ------------------------------------------------------------------ decode attention
// out[b, j, h] = sum_t softmax_t(scale q . k_t) v_t over the keys t that new token j sees.
//
// With n_t the numbers, s_t, z_t a group's scale and zero and Q the sum of q over it:
//   q . k_t = sum over groups of s_t (q . n_t) + z_t Q
//   out     = sum_t (p_t s_t) n_t + sum_t p_t z_t
// so that neither product needs the values themselves. The numbers enter the m16n8k16
// products as fp16 straight from memory's bits: a number in bits 0 .. 3 of a half is the
// subnormal n 2^-24, in bits 4 .. 7 n 2^-20, both exact, for one AND each (and a shift for
// every second pair). Up to 4 rows' scores take a byte n + 16 n' at once and the upper
// number's part off again: fp32 sums over one row of the cache, 16 times what is left. An
// output's sum is long and what is left of it small, so there each number enters by itself,
// and the products' accumulators (which round towards zero) are added up in fp32 after
// each tile (8 rows: after four, in shared memory): 4 sequences of 131072, error against 64
// bits 1.7e-3, a bf16 result's own 1.6e-3; with bytes and one accumulator it was 3.3e-3.
//
// Both products have the numbers as their first operand: scores are keys by rows (heads, new
// tokens), outputs dimensions by rows, so that 8 rows cost half of what 16 do; the weights turn
// from the one layout to the other by movmatrix. Up to 4 rows have two columns each, which take
// the parts of a byte and of a word apart: neither masks nor pairs of keys to make. One row alone
// (a head of keys for each of queries, one new token) has its softmax shared out over all lanes.
// More than 8 rows are lists of their own, which read the keys again (from L2: 24 sequences of
// 1024 to 8191, 20 rows on each of 4 heads of 128: 55 us; up to 16 or 24 rows a list, whose sums
// leave room for 2 CTAs an SM, 8 and 15 % more). The queries of a row are scaled by a power of two
// to 2^9 .. 2^10 at most, so that fp16 holds their bits: those 2^-31 of the greatest and smaller
// may lose some, 2^-39 of it. A score before the scale is in units of that: of keys that stand for
// less than about 2^-100 it may lose bits. The weights p_t s_t are fp16, against a unit for each
// row and group, a power of two: 11 bits, a quarter of the output's own rounding; those below
// 2^-21 of the row's greatest so far lose bits, below 2^-32 they vanish. p is taken against a
// reference within 2^3 of the greatest so far, which moves when that is passed: no search for the
// maximum in a tile that does not. The unit likewise is lowered when a weight passes 2^15, and
// rises with the reference: keys that a row does not see, or that have no weight, do not count for
// it, whatever their scales. Everything else is fp32.
//
// A warp takes tiles of 64 keys (hd 128: 32) through a ring of its own, as the bf16 kernel
// does, by bulk copies: a lane for each page's keys, values or scales (16-byte copies of
// each row took 105 instructions a tile). What a page holds behind the sequence's end
// comes along and is hidden like all that a row does not see.
//
// Bound by memory where there is much of it (16 sequences of 32768, 16 heads of 64: 103.5 us, 5.8
// TB/s; the copies alone 96), by instruction issue and by memory alike for grouped heads (4 of
// 87,000 to 131,072, 16 heads on 4 of 128: 58 us; the copies alone 45, the rest alone 47), by
// issue with many rows, by starts and ends of lists when these are short (48 of 64 to 4096, 16
// heads of 64: 25 us; 1 of 577: 5 us).
constexpr float kSlack = 3.0f;      // log2
constexpr int kMostUnit = 120;      // log2 of the weights' greatest unit: 2^4 times it, the most that kSlack rounds to, is in fp32
constexpr float kMostWeight = 32768.0f;      // what weights stay below, fp16 having 65504
constexpr int kLeast = 4;           // tiles of a CTA's span, at least
constexpr int kListCost = 6;        // tiles that a list's start and end cost
constexpr int kMostRows = 8;        // of a list

template <int HD, int ROWS>
struct Dec4 {
    static constexpr int kStages = 2;
    static constexpr int kCtas = ROWS == 1 ? 4 : 3;   // resident on an SM
    static constexpr int kTile = 4096 / HD;           // keys of a warp's step
    static constexpr int kGroups = HD / 64, kRowBytes = HD / 2, kScaleBytes = 8 * kGroups;
    static constexpr int kSide = kTile * kRowBytes;
    static constexpr int kStage = 2 * kSide + kTile * kScaleBytes;
    static constexpr int kRing = kDecWarps * kStages * kStage;
    // a warp's words between its lanes: the weights of a tile, in the low and in the high half
    // (1 row), or its scales and zeros in fp32, twice each (8)
    static constexpr int kStride = kTile / 4 + 4;
    static constexpr int kWords = ROWS == 1 ? 8 * kStride * kGroups : ROWS == 8 ? kTile * 8 * kGroups : 0;
    static constexpr int kSums = kRing + (ROWS == 8 ? kDecWarps * kWords * 4 : 0);
    // that, and the warps' outputs: at a list's end, with 8 rows also on the way
    static constexpr int kSmem = std::max(kRing + kDecWarps * kWords * 4, kSums + kDecWarps * ROWS * HD * 4);
    // a grid of kCtas an SM is resident at once: an SM's shared memory, 1 KB and the static part a CTA
    static_assert(kCtas * (kSmem + 1024 + kDecWarps * (kStages * 8 + (2 + kGroups) * 8 * 4) + 512) <= 228 * 1024);
};

struct Decode4Args : DecodeArgs {
    const uint8_t *k4, *v4;
    const uint16_t *scales;
};

// D(16x8 fp32) += A(16x16 fp16, row) * B(16x8 fp16, col)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same without anything to add to.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t v;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 .. 127
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// The transpose of an 8 x 8 matrix of halves, a row's two neighbours in a thread.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// One lane of the warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
}
// Waits for a barrier's phase, for about a second at most.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!tc::mbar_try_wait_suspend(bar, parity, tc::kWaitSuspendNs))
        if (clock64() - t0 > tc::kWaitLimitCycles) return false;
    return true;
}
constexpr uint32_t kEven = 0x000F000Fu, kOdd = 0x00F000F0u;      // numbers 0 and 4, 1 and 5 of a word's eight
// Byte 0 (1) of both halves of a word, as halves.
__device__ __forceinline__ uint32_t bytes_of(uint32_t w, int which) { return __byte_perm(w, 0, which ? 0x4341 : 0x4240); }
// The key of eight in row p of a score block. Rows p of four threads, and after the transpose
// rows 2 c (or 2 c + 1) of four, are then rows of the ring that differ mod 4: no bank conflicts.
__device__ __forceinline__ int key_of(int p) { return (p >> 1 & 1) | ((p ^ p >> 2) & 1) << 1 | (p & 4); }

template <int HD, int ROWS, bool Cluster>
__global__ void __launch_bounds__(kDecWarps * 32, Dec4<HD, ROWS>::kCtas)
decode_int4_kernel(const __grid_constant__ Decode4Args P) {
    using C = Dec4<HD, ROWS>;
    constexpr int NG = C::kGroups, kTile = C::kTile, kKeys = kTile / 32, NB = kTile / 8;      // NB: score blocks, of 8 keys
    constexpr int NA = ROWS == 8 ? 4 : 2;       // output tiles of a group: pairs of numbers of a word, or its bytes 0, 2 and 1, 3
    extern __shared__ __align__(128) unsigned char dsm[];
    __shared__ uint64_t s_full[kDecWarps][C::kStages];
    __shared__ __align__(16) float s_m[kDecWarps][8], s_l[kDecWarps][8], s_z[kDecWarps][NG][8];
    __shared__ float2 s_part[8];
    float *s_o = reinterpret_cast<float *>(dsm + C::kSums);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0);
    const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
    uint32_t *s_w = reinterpret_cast<uint32_t *>(dsm + C::kRing) + warp * C::kWords;
    const int G = P.H / P.Hk, groups = (P.rows + P.per - 1) / P.per, lists = P.Hk * groups;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (lane == 0) {
#pragma unroll
        for (int e = 0; e < C::kStages; ++e) tc::mbar_init(&s_full[warp][e], 1);
        tc::fence_proxy_async_smem();
    }
    __syncwarp();
    DecSpan at;
    if constexpr (Cluster) {
        const int first = static_cast<int>(blockIdx.x) * P.chunk / kTile;
        at = {0, 0, static_cast<int>(blockIdx.z), static_cast<int>(blockIdx.y), first, P.seq_lens[blockIdx.z],
              first + P.chunk / kTile + kListCost};
    } else if (!decode_span<kTile, kListCost, kLeast>(P, lists, at)) {
        if (threadIdx.x == 0 && !P.by_list) P.cut[blockIdx.x] = make_int2(0, 0);
        return;
    }
    using Len = DecLen<kTile>;
    Len len(at.n, P.max_len);
    // the tiles of a list that are before the span's end
    const int end = at.end;
    const auto tiles_to = [&](int base, int tiles) { return max(min(tiles, end - base - kListCost), 0); };

    // The copies' side of this warp: it takes every fourth tile of the span, whatever list
    // it is of. Lane i looks the tile's page i up while the tile before is copied; one lane then
    // copies each page's keys, values and scales. A page outside the cache is not copied and
    // makes the sequence's result NaN.
    const int page_mask = (1 << P.page_shift) - 1, page_rows = min(1 << P.page_shift, kTile);
    const uint32_t ring = smem_u32(dsm) + warp * C::kStages * C::kStage;
    const int piece_first = lane * page_rows;      // the first key of the page that this lane looks up
    int fbase = 0, fb = at.b, fy = at.y, fhk = fy / groups, fi = at.i, fn = len.n, fall = len.tiles;
    int fend = tiles_to(fbase, fall);
    int32_t flen = !Cluster && fb + 1 < P.B ? P.seq_lens[fb + 1] : 0;      // the next sequence's
    const int32_t *frow = P.table + fb * P.table_ld;
    struct Tile {
        int32_t page;
        int rows, first, hk;      // rows: of the sequence; < 0: no tile
    };
    bool more = true;
    uint32_t bad = 0;      // a bit for each stage
    auto look = [&](int step) {
        Tile tile = {0, -1, 0, 0};
        if (!more) return tile;
        fi += step;
        while (fi >= fend) {
            fi -= fend;
            fbase += fall + kListCost;
            if (Cluster || fbase + kListCost >= end) {
                more = false;
                return tile;
            }
            if (++fy == lists) {
                fy = 0;
                ++fb;
                const Len next(flen, P.max_len);
                fn = next.n, fall = next.tiles;
                flen = fb + 1 < P.B ? P.seq_lens[fb + 1] : 0;
                frow = P.table + fb * P.table_ld;
            }
            fhk = fy / groups;
            fend = tiles_to(fbase, fall);
        }
        tile.first = fi * kTile;
        tile.rows = fn - tile.first;
        tile.hk = fhk;
        if (piece_first < min(tile.rows, kTile)) tile.page = frow[(tile.first >> P.page_shift) + lane];
        return tile;
    };
    auto fetch = [&](int stage, const Tile &tile) {
        if (tile.rows >= 0) {
            const bool mine = piece_first < min(tile.rows, kTile);
            const bool in = mine && static_cast<uint32_t>(tile.page) < static_cast<uint32_t>(P.n_pages);
            bad = (bad & ~(1u << stage)) | static_cast<uint32_t>(mine && !in) << stage;
            uint32_t have = __ballot_sync(0xffffffffu, in);
            uint64_t *bar = &s_full[warp][stage];
            const bool one = elect_one();
            if (one) tc::mbar_arrive_expect_tx(bar, __popc(have) * page_rows * (2 * C::kRowBytes + C::kScaleBytes));
            // rows of the cache are counted in 32 bits (the caller's check), bytes in 64
            const uint32_t row = ((static_cast<uint32_t>(tile.page) * P.Hk + tile.hk) << P.page_shift) + (tile.first & page_mask);
            for (; have; have &= have - 1) {
                const int piece = __ffs(have) - 1;
                const uint64_t from = __shfl_sync(0xffffffffu, row, piece);
                const uint32_t to = ring + stage * C::kStage + piece * page_rows * C::kRowBytes;
                if (one) {
                    bulk_load(to, P.k4 + from * C::kRowBytes, page_rows * C::kRowBytes, bar);
                    bulk_load(to + C::kSide, P.v4 + from * C::kRowBytes, page_rows * C::kRowBytes, bar);
                    bulk_load(ring + stage * C::kStage + 2 * C::kSide + piece * page_rows * C::kScaleBytes,
                              reinterpret_cast<const uint8_t *>(P.scales) + from * C::kScaleBytes, page_rows * C::kScaleBytes, bar);
                }
            }
        }
    };
    int head = 0;
    uint32_t parity = 0;
    bool waits = true;      // none has run out
    Tile ahead[C::kStages];      // the tables' reads under way together
#pragma unroll
    for (int e = 0; e < C::kStages; ++e) ahead[e] = look(e == 0 ? warp : kDecWarps);
#pragma unroll
    for (int e = 0; e < C::kStages; ++e) fetch(e, ahead[e]);
    Tile tile = look(kDecWarps);

    // The products' side, list by list. Queries: of row r8 and each group the 16 dimensions
    // from 16 c4 on, as the numbers of a thread's two words pair up; up to 4 rows, columns 2 r
    // and 2 r + 1 are row r's. A thread's scores are of rows 2 c4 and 2 c4 + 1, of row c4 (4 rows), of
    // the row: for these, from products to scores, and the queries' sums in the products' units.
    uint32_t qb[NG][4][2];
    uint64_t crow, qsum[NG];
    const auto of_rows = [&](float v) {      // of the rows that threads r8 hold, this thread's
        if constexpr (ROWS == 1) return tc::f2(v, 0.0f);
        const float v0 = __shfl_sync(0xffffffffu, v, 8 * c4);
        return tc::f2(v0, ROWS == 4 ? 0.0f : __shfl_sync(0xffffffffu, v, 8 * c4 + 4));
    };
    auto queries = [&](int seq, int qy) {
        const int row0 = qy % groups * P.per, nr = min(P.per, P.rows - row0), hk = qy / groups;
        const int mine = ROWS == 1 ? 0 : ROWS == 4 ? r8 >> 1 : r8, row = row0 + mine;
        const bool odd = ROWS < 8 && (r8 & 1);
        uint4 raw[NG][2];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                raw[g][w] = make_uint4(0, 0, 0, 0);
                if (mine < nr)
                    raw[g][w] = *reinterpret_cast<const uint4 *>(
                        P.q + (static_cast<int64_t>(seq) * P.n_new + row / G) * P.q_ld +
                        static_cast<int64_t>(hk * G + row % G) * HD + 64 * g + 16 * c4 + 8 * w);
            }
        uint32_t top = 0;      // the greatest magnitude's bits
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t x[4] = {raw[g][w].x, raw[g][w].y, raw[g][w].z, raw[g][w].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max(x[e] & 0x7fffu, x[e] >> 16 & 0x7fffu));
            }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^up takes the greatest to 2^9 .. 2^10 (from 2^-117 down not as far: multiples of 2^-133, which fp16 holds then)
        const int up = min(136 - static_cast<int>(top >> 7), 126);
        const float f = pow2(up);
        // 2^(20 - up), up to 2^138, in two steps of one direction. Positive and finite: beyond these bounds one key has
        // all the weight, or all have the same
        const int back = 20 - up, half = back / 2;
        float c = fminf(fmaxf(P.scale_log2 * pow2(half) * pow2(back - half), __int_as_float(1)), 3e38f);
        if (top >= 0x7f80u) c = __int_as_float(0x7fc00000);            // a query that is not finite
        crow = of_rows(c);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float x[8];
                unpack8(raw[g][w], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] *= f;
                    sum += x[e];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // against numbers in the low places (or bytes), 16 times, and in the high ones. Up to 4 rows, an even
                    // column has the bytes' and the upper numbers' products, an odd one what the bytes' have of the upper
                    const uint32_t low = pack_f16x2(16.0f * x[2 * e], 16.0f * x[2 * e + 4]);
                    const uint32_t high = pack_f16x2(x[2 * e + 1], x[2 * e + 5]);
                    qb[g][2 * w + e][0] = odd ? 0u : low;
                    qb[g][2 * w + e][1] = odd ? low : high;
                }
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qsum[g] = of_rows(sum * 0x1p-20f);
        }
    };
    int b = at.b, y = at.y, i0 = at.i, taken = 0;
    queries(b, y);
    DecNew fresh(P, b, at.n);
    int2 cut = make_int2(0, 0);
    for (int base = 0; Cluster || base + kListCost < end;) {
        const int row0 = y % groups * P.per, nr = min(P.per, P.rows - row0);
        const int tiles = tiles_to(base, len.tiles) - i0;
        bool lost = len.lost || fresh.lost;
        // keys that this thread's rows see (of rows that are no new token's: whatever there is), and that all see
        int sees[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = (row0 + (ROWS == 1 ? 0 : ROWS == 4 ? c4 : 2 * c4 + e)) / G;
            sees[e] = j < fresh.count ? fresh.first + j : INT32_MAX;
        }
        const int all_see = row0 / G < fresh.count ? fresh.first + row0 / G : INT32_MAX;
        // sums of this thread's keys, references and limits: of its row, or of its two
        const uint64_t none2 = tc::f2(0.0f, 0.0f);
        float acc[NG][NA][4], m[2] = {-INFINITY, -INFINITY};
        float far[2] = {-INFINITY, -INFINITY};      // a score above moves the references
        uint64_t l2 = none2, z2[NG], ref = none2;   // ref: what is added to a score for its weight, -m or 0
        uint64_t unit[NG];      // of each row's weights, a power of two
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            unit[g] = tc::f2(pow2(kMostUnit), pow2(kMostUnit));
            z2[g] = none2;
#pragma unroll
            for (int i = 0; i < NA; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[g][i][e] = 0.0f;
        }
        // 8 rows: the sums of tiles that are through, as this thread has them in acc
        float4 *const kept = reinterpret_cast<float4 *>(s_o + warp * ROWS * HD) + lane;
        bool some_kept = false;
        // every output so far times f (of the row that a column is of)
        auto rescale = [&](int g, float f0, float f1) {
#pragma unroll
            for (int i = 0; i < NA; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[g][i][e] *= e & 1 ? f1 : f0;
            if (ROWS == 8 && some_kept) {
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    float4 &x = kept[(g * NA + i) * 32];
                    x = make_float4(x.x * f0, x.y * f1, x.z * f0, x.w * f1);
                }
            }
        };
        // over the lanes that share a row
        const auto most_of_row = [&](float x) {
#pragma unroll
            for (int o = ROWS == 1 ? 1 : 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            return x;
        };
        const auto exponent = [](float x) { return (__float_as_int(x) >> 23) - 127; };      // of a positive one
        // x0, x1: the greatest weights times scales of this lane's keys, times 2^-8 (finite where the scales are). Rows
        // whose weights pass kMostWeight get the unit that brings the greatest to 2^7 .. 2^8: room for what the next
        // tiles bring (24 x 5 tokens 55.3 us; to 2^11 58.1, to 2^3 55.2).
        auto lower = [&](int g, float x0, float x1) {
            const float2 u = tc::f2_split(unit[g]);
            float x[2] = {x0, x1}, from[2] = {u.x, u.y}, f[2];
#pragma unroll
            for (int e = 0; e < (ROWS == 8 ? 2 : 1); ++e) {
                x[e] = most_of_row(x[e]);
                const int was = exponent(from[e]);
                const int to = x[e] * 256.0f * from[e] >= kMostWeight ? max(-1 - exponent(x[e]), -126) : was;
                f[e] = to - was < -126 ? 0.0f : pow2(to - was);
                from[e] = pow2(to);
            }
            if (ROWS < 8) f[1] = f[0], from[1] = from[0];
            unit[g] = tc::f2(from[0], from[1]);
            rescale(g, f[0], f[1]);
        };
        // the references to the greatest scores, over the lanes that share a row
        auto move = [&](float x0, float x1) {
            float f[2], rise[2], x[2] = {fmaxf(x0, m[0]), fmaxf(x1, m[1])};      // not NaN
#pragma unroll
            for (int e = 0; e < (ROWS == 8 ? 2 : 1); ++e) {
                x[e] = most_of_row(x[e]);
                rise[e] = x[e] > m[e] ? x[e] - m[e] : 0.0f;      // (from -inf: inf)
                f[e] = tc::ex2(-rise[e]);
                m[e] = x[e];
                far[e] = x[e] + kSlack;
            }
            if (ROWS < 8) f[1] = f[0], rise[1] = rise[0];
            ref = tc::f2(m[0] == -INFINITY ? 0.0f : -m[0], m[1] == -INFINITY ? 0.0f : -m[1]);
            const uint64_t f2 = tc::f2(f[0], f[1]);
            l2 = tc::mul2(l2, f2);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                z2[g] = tc::mul2(z2[g], f2);
                // weights that have become small get a larger unit, their sums so far keep theirs
                const float2 u = tc::f2_split(unit[g]);
                float from[2] = {u.x, u.y}, back[2];
#pragma unroll
                for (int e = 0; e < (ROWS == 8 ? 2 : 1); ++e) {
                    const int was = exponent(from[e]), by = min(__float2int_rn(rise[e]), kMostUnit - was);
                    back[e] = tc::ex2(static_cast<float>(by) - rise[e]);
                    from[e] = pow2(was + by);
                }
                if (ROWS < 8) back[1] = back[0], from[1] = from[0];
                unit[g] = tc::f2(from[0], from[1]);
                rescale(g, back[0], back[1]);
            }
        };
        const auto low = [](uint64_t v) { return tc::f2_split(v).x; };
        // a weight's exponent. The product is rounded by itself, as the reference was: the difference of a huge score to
        // its own rounding is no exponent. (In packed pairs the product and the sum became one operation again.)
        const auto weight_of = [&](float t, int row) {
            const float2 c = tc::f2_split(crow), r = tc::f2_split(ref);
            return __fadd_rn(__fmul_rn(t, row ? c.y : c.x), row ? r.y : r.x);
        };
        for (int i = (warp - taken) & (kDecWarps - 1); i < tiles; i += kDecWarps) {
            if (waits && !wait_phase(&s_full[warp][head], parity)) waits = false;
            lost |= (bad >> head & 1) || !waits;
            const int key0 = (i0 + i) * kTile;
            const unsigned char *sk = dsm + (warp * C::kStages + head) * C::kStage, *sv = sk + C::kSide, *ss = sv + C::kSide;
            const bool masked = all_see - key0 < kTile;
            // the two words that a thread multiplies of a key's group
            const auto key_words = [&](int key, int g) {
                return *reinterpret_cast<const uint2 *>(sk + key * C::kRowBytes + 32 * g + 8 * c4);
            };
            // up to 4 rows: the products with keys in rows r8 of blocks 2 mt and 2 mt + 1, in even columns with the bytes and
            // the upper numbers, in odd ones what the bytes have of the upper numbers
            const auto byte_products = [&](float (&d)[4], uint2 k0, uint2 k1, int g) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const uint32_t x = bytes_of(s & 2 ? k0.y : k0.x, s & 1), x2 = bytes_of(s & 2 ? k1.y : k1.x, s & 1);
                    if (s == 0) mma_f16_first(d, x, x2, x & kOdd, x2 & kOdd, qb[g][s][0], qb[g][s][1]);
                    else mma_f16(d, x, x2, x & kOdd, x2 & kOdd, qb[g][s][0], qb[g][s][1]);
                }
            };
            // and with values: words x and x2 of two keys, whose weights are b0 and b1; numbers 0, 4 and 1, 5, then 2, 6 and 3, 7
            const auto value_products = [&](float (&d)[2][4], uint32_t x, uint32_t x2, uint32_t b0, uint32_t b1, bool first) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t y = x >> 8 * s, y2 = x2 >> 8 * s;
                    if (first) mma_f16_first(d[s], y & kEven, y & kOdd, y2 & kEven, y2 & kOdd, b0, b1);
                    else mma_f16(d[s], y & kEven, y & kOdd, y2 & kEven, y2 & kOdd, b0, b1);
                }
            };
            const auto add = [&](int g, const float (&d)[2][4]) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[g][s][e] += d[s][e];
            };
            if constexpr (ROWS == 1) {
                // scores: this lane's are of keys 8 c4 + r8 (+ 32), one of each four blocks
                float t[kKeys];
                uint2 raw[NG][kKeys];
#pragma unroll
                for (int k = 0; k < kKeys; ++k) t[k] = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll
                    for (int k = 0; k < kKeys; ++k)
                        raw[g][k] = *reinterpret_cast<const uint2 *>(ss + (32 * k + 8 * c4 + r8) * C::kScaleBytes + 8 * g);
                    float d[NB / 2][4];
#pragma unroll
                    for (int mt = 0; mt < NB / 2; ++mt)
                        byte_products(d[mt], key_words(16 * mt + r8, g), key_words(16 * mt + 8 + r8, g), g);
#pragma unroll
                    for (int k = 0; k < kKeys; ++k) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = d[2 * k + (e >> 1)][2 * (e & 1)] - d[2 * k + (e >> 1)][2 * (e & 1) + 1];
                        const float dot = c4 & 2 ? (c4 & 1 ? x[3] : x[2]) : (c4 & 1 ? x[1] : x[0]);
                        t[k] = fmaf(bf_lo(raw[g][k].x), dot, fmaf(bf_hi(raw[g][k].x), low(qsum[g]), t[k]));
                    }
                }
                float mx = -INFINITY;
                if (masked) {
                    // what the row does not see does not reach it: a value that stands for NaN neither
#pragma unroll
                    for (int k = 0; k < kKeys; ++k)
                        if (key0 + 32 * k + 8 * c4 + r8 >= sees[0]) {
                            t[k] = -INFINITY;
#pragma unroll
                            for (int g = 0; g < NG; ++g) raw[g][k].y = 0u;
                        }
                }
#pragma unroll
                for (int k = 0; k < kKeys; ++k) mx = fmaxf(mx, t[k]);
                if (__any_sync(0xffffffffu, mx * low(crow) > far[0])) move(mx * low(crow), -INFINITY);
                // weights to the lanes that multiply them: key t at (t mod 4, t / 4), once in the low half and once in the high one
                const auto weigh = [&] {
                    float most = 0.0f;
#pragma unroll
                    for (int k = 0; k < kKeys; ++k) {
                        const int key = 32 * k + 8 * c4 + r8;
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            const float w = t[k] * low(unit[g]) * bf_lo(raw[g][k].y);
                            most = fmaxf(most, w);
                            const uint32_t half = pack_f16x2(w, 0.0f);
                            uint32_t *to = s_w + 8 * C::kStride * g + (key & 3) * C::kStride + (key >> 2);
                            to[0] = half;
                            to[4 * C::kStride] = half << 16;
                        }
                    }
                    return most;
                };
#pragma unroll
                for (int k = 0; k < kKeys; ++k) {
                    t[k] = tc::ex2(weight_of(t[k], 0));
                    l2 = tc::f2(low(l2) + t[k], 0.0f);
#pragma unroll
                    for (int g = 0; g < NG; ++g) z2[g] = tc::f2(fmaf(t[k], bf_hi(raw[g][k].y), low(z2[g])), 0.0f);
                }
                if (__any_sync(0xffffffffu, weigh() >= kMostWeight)) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float most = 0.0f;
#pragma unroll
                        for (int k = 0; k < kKeys; ++k) most = fmaxf(most, t[k] * (bf_lo(raw[g][k].y) * 0x1p-8f));
                        lower(g, most, 0.0f);
                    }
                    weigh();
                }
                __syncwarp();
                // outputs: words r8 of keys 4 j + c4; an even column has their low halves' products, an odd one the high ones'
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float d[2][4];
#pragma unroll
                    for (int j = 0; j < kTile / 4; j += 4) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(s_w + 8 * C::kStride * g + (4 * (r8 & 1) + c4) * C::kStride + j);
                        const uint32_t pw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            const unsigned char *at = sv + (4 * (j + u) + c4) * C::kRowBytes + 32 * g + 4 * r8;
                            value_products(d, *reinterpret_cast<const uint32_t *>(at),
                                           *reinterpret_cast<const uint32_t *>(at + 4 * C::kRowBytes), pw[u], pw[u + 1], j + u == 0);
                        }
                    }
                    add(g, d);
                }
            } else if constexpr (ROWS == 4) {
                // scores of row c4: keys key_of(r8) of each block
                const int mine = key_of(r8);
                float t[NB];
                uint2 raw[NG][NB];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) raw[g][n] = *reinterpret_cast<const uint2 *>(ss + (8 * n + mine) * C::kScaleBytes + 8 * g);
#pragma unroll
                    for (int mt = 0; mt < NB / 2; ++mt) {
                        float d[4];
                        byte_products(d, key_words(16 * mt + mine, g), key_words(16 * mt + 8 + mine, g), g);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int n = 2 * mt + h;
                            const float zero = bf_hi(raw[g][n].x) * low(qsum[g]);
                            t[n] = fmaf(bf_lo(raw[g][n].x), d[2 * h] - d[2 * h + 1], g == 0 ? zero : t[n] + zero);
                        }
                    }
                }
                float mx = -INFINITY;
                if (masked) {
                    // what a row does not see does not reach it: a value that stands for NaN neither
#pragma unroll
                    for (int n = 0; n < NB; ++n)
                        if (key0 + 8 * n + mine >= sees[0]) {
                            t[n] = -INFINITY;
#pragma unroll
                            for (int g = 0; g < NG; ++g) raw[g][n].y = 0u;
                        }
                }
#pragma unroll
                for (int n = 0; n < NB; n += 2) mx = tc::fmax3(mx, t[n], t[n + 1]);
                if (__any_sync(0xffffffffu, mx * low(crow) > far[0])) move(mx * low(crow), -INFINITY);
                uint32_t pw[NG][NB];
                const auto weigh = [&] {
                    float most = 0.0f;
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int n = 0; n < NB; n += 2) {
                            const float w = t[n] * low(unit[g]) * bf_lo(raw[g][n].y);
                            const float w2 = t[n + 1] * low(unit[g]) * bf_lo(raw[g][n + 1].y);
                            pw[g][n] = pack_f16x2(w, w);
                            pw[g][n + 1] = pack_f16x2(w2, w2);
                            most = tc::fmax3(most, w, w2);
                        }
                    return most;
                };
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    t[n] = tc::ex2(weight_of(t[n], 0));
                    l2 = tc::f2(low(l2) + t[n], 0.0f);
#pragma unroll
                    for (int g = 0; g < NG; ++g) z2[g] = tc::f2(fmaf(t[n], bf_hi(raw[g][n].y), low(z2[g])), 0.0f);
                }
                if (__any_sync(0xffffffffu, weigh() >= kMostWeight)) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float most = 0.0f;
#pragma unroll
                        for (int n = 0; n < NB; ++n) most = fmaxf(most, t[n] * (bf_lo(raw[g][n].y) * 0x1p-8f));
                        lower(g, most, 0.0f);
                    }
                    weigh();
                }
                // weights: transposed, a thread has those of keys in rows 2 c4 and 2 c4 + 1 of row r8 / 2: in an even column
                // for the words' low halves, in an odd one for the high ones
                const uint32_t first = r8 & 1 ? 0x1044u : 0x4410u, second = r8 & 1 ? 0x3244u : 0x4432u;
                const unsigned char *v0 = sv + key_of(2 * c4) * C::kRowBytes + 4 * r8, *v1 = sv + key_of(2 * c4 + 1) * C::kRowBytes + 4 * r8;
                float d[NG][2][4];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const uint32_t both = transpose8(pw[g][n]);
                        const int at = 8 * n * C::kRowBytes + 32 * g;
                        value_products(d[g], *reinterpret_cast<const uint32_t *>(v0 + at), *reinterpret_cast<const uint32_t *>(v1 + at),
                                       __byte_perm(both, 0, first), __byte_perm(both, 0, second), n == 0);
                    }
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) add(g, d[g]);
            } else {
                // [group][key's, value's][key]: scale, scale, zero, zero in fp32, once for the warp, each lane its keys'
                ulonglong2 *s_x = reinterpret_cast<ulonglong2 *>(s_w);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll
                    for (int k = 0; k < kKeys; ++k) {
                        const uint2 raw = *reinterpret_cast<const uint2 *>(ss + (lane + 32 * k) * C::kScaleBytes + 8 * g);
                        const float ks = bf_lo(raw.x), kz = bf_hi(raw.x), vs = bf_lo(raw.y), vz = bf_hi(raw.y);
                        s_x[(2 * g) * kTile + lane + 32 * k] = make_ulonglong2(tc::f2(ks, ks), tc::f2(kz, kz));
                        s_x[(2 * g + 1) * kTile + lane + 32 * k] = make_ulonglong2(tc::f2(vs, vs), tc::f2(vz, vz));
                    }
                }
                __syncwarp();
                // scores of keys key_of(r8) of each block, both rows of a pair in one register pair
                const int mine = key_of(r8);
                uint64_t t[NB];
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int mt = 0; mt < NB / 2; ++mt) {
                        const uint2 k0 = key_words(16 * mt + mine, g), k1 = key_words(16 * mt + 8 + mine, g);
                        float d[4];
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            const uint32_t x = (s & 2 ? k0.y : k0.x) >> 8 * (s & 1), x2 = (s & 2 ? k1.y : k1.x) >> 8 * (s & 1);
                            if (s == 0) mma_f16_first(d, x & kEven, x2 & kEven, x & kOdd, x2 & kOdd, qb[g][s][0], qb[g][s][1]);
                            else mma_f16(d, x & kEven, x2 & kEven, x & kOdd, x2 & kOdd, qb[g][s][0], qb[g][s][1]);
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int n = 2 * mt + h;
                            const ulonglong2 sz = s_x[(2 * g) * kTile + 8 * n + mine];
                            const uint64_t zero = g == 0 ? tc::mul2(sz.y, qsum[g]) : tc::fma2(sz.y, qsum[g], t[n]);
                            t[n] = tc::fma2(sz.x, tc::f2(d[2 * h], d[2 * h + 1]), zero);
                        }
                    }
                if (masked) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const float2 x = tc::f2_split(t[n]);
                        const int key = key0 + 8 * n + mine;
                        t[n] = tc::f2(key < sees[0] ? x.x : -INFINITY, key < sees[1] ? x.y : -INFINITY);
                    }
                }
                // the greatest score that this thread has of each row (NaN left out); the references move if one is far above
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < NB; n += 2) {
                    const float2 x = tc::f2_split(t[n]), x2 = tc::f2_split(t[n + 1]);
                    mx[0] = tc::fmax3(mx[0], x.x, x2.x);
                    mx[1] = tc::fmax3(mx[1], x.y, x2.y);
                }
                const float2 c = tc::f2_split(crow);
                mx[0] *= c.x, mx[1] *= c.y;
                if (__any_sync(0xffffffffu, mx[0] > far[0] || mx[1] > far[1])) move(mx[0], mx[1]);
                uint32_t pw[NG][NB];
                // a value's scale or zero for both rows; what a row does not see does not reach it: NaN scales neither
                const auto seen = [&](uint64_t v, int n) {
                    const int key = key0 + 8 * n + mine;
                    return tc::f2(key < sees[0] ? low(v) : 0.0f, key < sees[1] ? low(v) : 0.0f);
                };
                float most = 0.0f;
                auto weigh = [&](auto some_hidden) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        t[n] = tc::ex2_pair(tc::f2(weight_of(tc::f2_split(t[n]).x, 0), weight_of(tc::f2_split(t[n]).y, 1)));
                        l2 = tc::add2(l2, t[n]);
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            ulonglong2 sz = s_x[(2 * g + 1) * kTile + 8 * n + mine];
                            if constexpr (some_hidden.value) sz.x = seen(sz.x, n), sz.y = seen(sz.y, n);
                            z2[g] = tc::fma2(t[n], sz.y, z2[g]);
                            const float2 w = tc::f2_split(tc::mul2(tc::mul2(t[n], unit[g]), sz.x));
                            pw[g][n] = transpose8(pack_f16x2(w.x, w.y));
                            most = tc::fmax3(most, w.x, w.y);
                        }
                    }
                };
                if (masked) weigh(std::true_type{});
                else weigh(std::false_type{});
                if (__any_sync(0xffffffffu, most >= kMostWeight)) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const auto scale = [&](int n) { return seen(s_x[(2 * g + 1) * kTile + 8 * n + mine].x, n); };
                        const uint64_t small = tc::f2(0x1p-8f, 0x1p-8f);
                        float x[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            const float2 v = tc::f2_split(tc::mul2(t[n], tc::mul2(scale(n), small)));
                            x[0] = fmaxf(x[0], v.x), x[1] = fmaxf(x[1], v.y);
                        }
                        lower(g, x[0], x[1]);
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            const float2 w = tc::f2_split(tc::mul2(tc::mul2(t[n], unit[g]), scale(n)));
                            pw[g][n] = transpose8(pack_f16x2(w.x, w.y));
                        }
                    }
                }
                const unsigned char *v0 = sv + key_of(2 * c4) * C::kRowBytes + 4 * r8, *v1 = sv + key_of(2 * c4 + 1) * C::kRowBytes + 4 * r8;
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int mt = 0; mt < NB / 2; ++mt) {
                        uint32_t w[2][2];      // numbers 0 .. 3 and 4 .. 7 of the keys in rows 2 c4 and 2 c4 + 1 of both blocks
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int at = (16 * mt + 8 * h) * C::kRowBytes + 32 * g;
                            const uint32_t x0 = *reinterpret_cast<const uint32_t *>(v0 + at);
                            const uint32_t x1 = *reinterpret_cast<const uint32_t *>(v1 + at);
                            w[h][0] = __byte_perm(x0, x1, 0x5410);
                            w[h][1] = __byte_perm(x0, x1, 0x7632);
                        }
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) {
                            const uint32_t x = w[0][i2 >> 1] >> 8 * (i2 & 1), x2 = w[1][i2 >> 1] >> 8 * (i2 & 1);
                            mma_f16(acc[g][i2], x & kEven, x & kOdd, x2 & kEven, x2 & kOdd, pw[g][2 * mt], pw[g][2 * mt + 1]);
                        }
                    }
                if ((i & (4 * kDecWarps - 1)) < kDecWarps) {      // every fourth of this warp's tiles
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int i2 = 0; i2 < NA; ++i2) {
                            float4 &x = kept[(g * NA + i2) * 32];
                            const float4 old = some_kept ? x : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            x = make_float4(old.x + acc[g][i2][0], old.y + acc[g][i2][1], old.z + acc[g][i2][2], old.w + acc[g][i2][3]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[g][i2][e] = 0.0f;
                        }
                    some_kept = true;
                }
            }
            __syncwarp();      // the stage, and the words between the lanes, have been read
            fetch(head, tile);
            tile = look(kDecWarps);
            if (++head == C::kStages) head = 0, parity ^= 1;
        }

        // the next list, and its queries on their way
        const int next = base + len.tiles + kListCost;
        int32_t blen = 0;
        int ny = y + 1, nb = b;
        if (ny == lists) ny = 0, ++nb;
        const DecNew now = fresh;
        if (!Cluster && next + kListCost < end) {
            queries(nb, ny);
            if (nb != b) blen = P.seq_lens[nb];
        }

        // join the warps: their references and sums, then the outputs
        const auto whole_rows = [](uint64_t v2) {
            float2 v = tc::f2_split(v2);
#pragma unroll
            for (int o = ROWS == 1 ? 1 : 4; o < 32; o <<= 1) {
                v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
                if (ROWS == 8) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
            }
            return v;
        };
        const auto put = [&](float *to, float2 v) {
            if constexpr (ROWS == 8) *reinterpret_cast<float2 *>(to + 2 * c4) = v;
            else to[c4] = v.x;
        };
        const float2 l = whole_rows(l2);
        if (r8 == 0) {
            put(s_m[warp], make_float2(m[0], m[1]));
            put(s_l[warp], l);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float2 z = whole_rows(z2[g]);
            if (r8 == 0) put(s_z[warp][g], z);
        }
        lost = __syncthreads_or(lost);
        const int64_t list = static_cast<int64_t>(b) * lists + y;
        const bool whole = i0 == 0 && tiles == len.tiles;
        const auto reference = [&](int row) {
            float M = s_m[0][row];
#pragma unroll
            for (int w = 1; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][row]);
            return M;
        };
        if (ROWS == 8 && some_kept) {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int i2 = 0; i2 < NA; ++i2) {
                    const float4 x = kept[(g * NA + i2) * 32];
                    acc[g][i2][0] += x.x, acc[g][i2][1] += x.y, acc[g][i2][2] += x.z, acc[g][i2][3] += x.w;
                }
            __syncwarp();      // the warp's sums are read; their place takes its outputs
        }
        // the numbers' 2^-24 and 2^-20 and the weights' unit taken out: that is 2^-124 (where scales are finite) to 2^120
        const auto part_of = [&](int row, int g, int e) {
            const float f = s_m[warp][row] == -INFINITY ? 0.0f : tc::ex2(s_m[warp][row] - reference(row));
            const float2 u = tc::f2_split(unit[g]);
            return pow2(min(3 - exponent(e ? u.y : u.x), 127)) * f;
        };
        const auto pair_of = [](const float (&x)[4], int e, float u) {
            return make_float2(x[e] * 0x1p21f * u, x[2 + e] * 0x1p17f * u);
        };
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if constexpr (ROWS < 8) {
                const int row = ROWS == 1 ? 0 : c4;
                if (ROWS == 4 || c4 == 0) {
                    const float u = part_of(row, g, 0);
                    float4 *to = reinterpret_cast<float4 *>(s_o + (warp * ROWS + row) * HD + 64 * g + 8 * r8);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 x = pair_of(acc[g][0], e, u), x2 = pair_of(acc[g][1], e, u);
                        to[e] = make_float4(x.x, x.y, x2.x, x2.y);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float u = part_of(2 * c4 + e, g, e);
                    float4 *to = reinterpret_cast<float4 *>(s_o + (warp * ROWS + 2 * c4 + e) * HD + 64 * g + 8 * r8);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 x = pair_of(acc[g][2 * h], e, u), x2 = pair_of(acc[g][2 * h + 1], e, u);
                        to[h] = make_float4(x.x, x.y, x2.x, x2.y);
                    }
                }
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < nr * (HD / 4); e += blockDim.x) {
            const int row = e / (HD / 4), d = e % (HD / 4) * 4;
            const float M = reference(row);
            float L = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) {
                // a warp without a reference saw nothing, or NaN alone
                const float f = s_m[w][row] == -INFINITY ? 1.0f : tc::ex2(s_m[w][row] - M);
                L += s_l[w][row] * f;
                const float4 x = *reinterpret_cast<const float4 *>(s_o + (w * ROWS + row) * HD + d);
                const float zero = s_z[w][d / 64][row] * f;
                o.x += x.x + zero, o.y += x.y + zero, o.z += x.z + zero, o.w += x.w + zero;
            }
            if (lost) L = __int_as_float(0x7fc00000);
            if constexpr (Cluster) {
                // this CTA's part stays where the ring was
                *reinterpret_cast<float4 *>(reinterpret_cast<float *>(dsm) + row * HD + d) = o;
                if (d == 0) s_part[row] = make_float2(M, L);
            } else if (whole) {
                const int j = (row0 + row) / G, h = y / groups * G + (row0 + row) % G;
                const float inv = 1.0f / L;
                uint2 got = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                if (now.sees(j) <= 0) got = make_uint2(0, 0);
                *reinterpret_cast<uint2 *>(P.out + ((static_cast<int64_t>(b) * P.n_new + j) * P.H + h) * HD + d) = got;
            } else {
                // a CTA and a list that follow one another in the order of tiles: no two
                // parts have the same sum
                float *dst = P.part + ((blockIdx.x + list) * P.per + row) * (HD + 4);
                *reinterpret_cast<float4 *>(dst + 4 + d) = o;
                if (d == 0) *reinterpret_cast<float2 *>(dst) = make_float2(M, L);
            }
        }
        __syncthreads();
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
            len = Len(blen, P.max_len);
            if (base + kListCost < end) fresh = DecNew(P, b, blen);
        }
    }
    if (!Cluster && threadIdx.x == 0 && !P.by_list) P.cut[blockIdx.x] = cut;
    if constexpr (Cluster) {
        cluster_sync();
        // pairs of columns, dealt out over the cluster's threads; parts in chunk order
        const int ctas = P.n_chunks, me = static_cast<int>(blockIdx.x);
        const int row0 = y % groups * P.per, nr = min(P.per, P.rows - row0);
        for (int e = me * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x); e < nr * (HD / 2);
             e += ctas * static_cast<int>(blockDim.x)) {
            const int row = e / (HD / 2), d = e % (HD / 2) * 2;
            float2 ml[kClusterMost], x[kClusterMost];
            float M = -INFINITY, L = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (int c = 0; c < kClusterMost; ++c) {
                ml[c] = make_float2(-INFINITY, 0.0f);
                x[c] = make_float2(0.0f, 0.0f);
                if (c < ctas) {
                    ml[c] = ld_cluster(&s_part[row], c);
                    x[c] = ld_cluster(reinterpret_cast<const float2 *>(reinterpret_cast<float *>(dsm) + row * HD + d), c);
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
            const int j = (row0 + row) / G, h = y / groups * G + (row0 + row) % G;
            const float inv = 1.0f / L;
            *reinterpret_cast<uint32_t *>(P.out + ((static_cast<int64_t>(b) * P.n_new + j) * P.H + h) * HD + d) =
                fresh.sees(j) <= 0 ? 0u : pack_bf16x2(o0 * inv, o1 * inv);
        }
        cluster_sync();      // nobody leaves while its part is read
    }
}

}  // namespace

cudaError_t launch_rope_append_int4(const void *qkv, int64_t ld, const float *cosv, const float *sinv, int64_t n_pos,
                                    const void *positions, int pos64, const void *slots, int slot64, int64_t T, int H,
                                    int Hk, int hd, int64_t n_pages, int page_shift, void *kp, void *vp, void *scales,
                                    void *q, void *k, void *v, cudaStream_t st) {
    // three heads a thread read the tables once (16384 tokens of 24 heads of 128: 40 us, 46 one by one, 42 two, 41 four),
    // where there are enough threads all the same (231 tokens of 24: 3.2 us one by one, 6.7 four)
    const int heads = H + 2 * Hk, per = kAppendThreads / (hd / 16);
    const bool many = T * heads >= 65536;
    const int64_t grid = (T + per - 1) / per * ((heads + (many ? 3 : 1) - 1) / (many ? 3 : 1));
    auto go = [&](auto kernel) {
        kernel<<<static_cast<unsigned>(grid), kAppendThreads, 0, st>>>(
            static_cast<const uint16_t *>(qkv), ld, cosv, sinv, n_pos, positions, pos64, slots, slot64, T, H, Hk,
            n_pages << page_shift, page_shift, static_cast<uint8_t *>(kp), static_cast<uint8_t *>(vp),
            static_cast<uint16_t *>(scales), static_cast<uint16_t *>(q), static_cast<uint16_t *>(k),
            static_cast<uint16_t *>(v));
    };
    if (hd == 64) many ? go(rope_append_int4_kernel<64, 3>) : go(rope_append_int4_kernel<64, 1>);
    else many ? go(rope_append_int4_kernel<128, 3>) : go(rope_append_int4_kernel<128, 1>);
    count_launch();
    return cudaGetLastError();
}

// Rows of a key head that one list takes: all up to kMostRows (one pass over the keys), else shared out evenly.
static int list_rows(int64_t rows) {
    const int64_t groups = (rows + kMostRows - 1) / kMostRows;
    return static_cast<int>((rows + groups - 1) / groups);
}

// f with the kernel's head_dim and rows: those that a list of `per` rows takes.
template <typename F>
static auto with_form(int64_t hd, int per, F f) {
    if (hd == 64) return per == 1 ? f(Dec4<64, 1>{}) : per <= 4 ? f(Dec4<64, 4>{}) : f(Dec4<64, 8>{});
    return per == 1 ? f(Dec4<128, 1>{}) : per <= 4 ? f(Dec4<128, 4>{}) : f(Dec4<128, 8>{});
}

static DecodeSplit decode_int4_split(int64_t B, int64_t rows, int64_t Hk, int64_t hd, int64_t max_len) {
    DecodeSplit s;
    const int per = list_rows(rows);
    const int64_t lists = B * Hk * ((rows + per - 1) / per), tile = 4096 / hd;
    const int ctas = with_form(hd, per, [](auto form) { return decltype(form)::kCtas; });
    const int64_t resident = static_cast<int64_t>(device_sm_count()) * ctas;
    // few short lists: as one cluster each, of up to 8 chunks of up to 1024 keys
    const int64_t most = std::min<int64_t>(kClusterMost, resident / std::max<int64_t>(lists, 1));
    if (most > 0 && max_len <= most * 1024) {
        const int64_t chunk = std::max<int64_t>((max_len + most - 1) / most, 4 * tile);
        s.chunk = static_cast<int>((chunk + 63) / 64 * 64);
        s.n_chunks = static_cast<int>(std::max<int64_t>(1, (max_len + s.chunk - 1) / s.chunk));
        s.cluster = true;
        return s;
    }
    s.ctas = std::min(resident, lists * std::max<int64_t>((max_len + tile * kLeast - 1) / (tile * kLeast), 1));
    s.lists = lists;
    return s;
}

// A call's parts; where the lists are cut comes behind them.
static size_t part_floats(const DecodeSplit &s, int per, int64_t hd) {
    return static_cast<size_t>(s.ctas + s.lists) * per * (hd + 4);
}

size_t decode_int4_bytes(int64_t B, int64_t rows, int64_t Hk, int64_t hd, int64_t max_len) {
    const DecodeSplit s = decode_int4_split(B, rows, Hk, hd, max_len);
    return s.cluster ? 0 : part_floats(s, list_rows(rows), hd) * sizeof(float) + static_cast<size_t>(std::min(s.ctas, s.lists)) * 8;
}

template <int HD, int ROWS>
static cudaError_t launch_decode(Dec4<HD, ROWS>, const Decode4Args &p, const DecodeSplit &s, dim3 grid, cudaStream_t st) {
    constexpr int smem = Dec4<HD, ROWS>::kSmem;
    static std::atomic<uint64_t> ready{0};      // devices whose kernels have their shared memory set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(decode_int4_kernel<HD, ROWS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      smem)) != cudaSuccess ||
            (e = cudaFuncSetAttribute(decode_int4_kernel<HD, ROWS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
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
        e = cudaLaunchKernelEx(&cfg, decode_int4_kernel<HD, ROWS, true>, p);
        count_launch();
        return e;
    }
    decode_int4_kernel<HD, ROWS, false><<<grid, kDecWarps * 32, smem, st>>>(p);
    count_launch();
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // the join's launch overlaps the split's end; its threads wait for the parts
    const bool wide = s.ctas > 8 * s.lists;
    cfg.blockDim = dim3(wide ? 512 : 128);
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(s.ctas, s.lists)), p.per, wide ? HD / 32 : 1);
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    const DecodeArgs &join = p;
    e = wide ? cudaLaunchKernelEx(&cfg, decode_join_kernel<HD, true, true>, join)
             : cudaLaunchKernelEx(&cfg, decode_join_kernel<HD, false, true>, join);
    count_launch();
    return e;
}

cudaError_t launch_decode_attn_int4(const void *q, int64_t q_ld, const void *kp, const void *vp, const void *scales,
                                    int64_t n_pages, int page_shift, const int32_t *table, int64_t table_ld,
                                    const int32_t *seq_lens, const int32_t *new_lens, int64_t max_len, int64_t B,
                                    int n_new, int H, int Hk, int hd, float scale, void *out, float *part,
                                    cudaStream_t st) {
    const int G = H / Hk, rows = G * n_new, per = list_rows(rows);
    const DecodeSplit s = decode_int4_split(B, rows, Hk, hd, max_len);
    const unsigned lists = Hk * ((rows + per - 1) / per);
    const dim3 grid = s.cluster ? dim3(s.n_chunks, lists, static_cast<unsigned>(B)) : dim3(static_cast<unsigned>(s.ctas));
    Decode4Args p = {};
    p.q = static_cast<const uint16_t *>(q);
    // a cache without pages: addresses that nothing is copied from
    p.k4 = static_cast<const uint8_t *>(kp ? kp : q);
    p.v4 = static_cast<const uint8_t *>(vp ? vp : q);
    p.scales = static_cast<const uint16_t *>(scales ? scales : q);
    p.table = table;
    p.seq_lens = seq_lens;
    p.new_lens = new_lens;
    p.q_ld = q_ld;
    p.table_ld = table_ld;
    p.n_pages = n_pages;
    p.max_len = max_len;
    p.H = H;
    p.Hk = Hk;
    p.n_new = n_new;
    p.rows = rows;
    p.per = per;
    p.page_shift = page_shift;
    p.B = B;
    p.chunk = s.chunk;
    p.n_chunks = s.n_chunks;
    p.scale_log2 = scale * kLog2e;
    p.out = static_cast<uint16_t *>(out);
    p.part = part;
    // the parts, then the CTAs' cut lists
    p.by_list = s.lists <= s.ctas;
    p.cut = s.cluster ? nullptr : reinterpret_cast<int2 *>(part + part_floats(s, per, hd));
    return with_form(hd, per, [&](auto form) { return launch_decode(form, p, s, grid, st); });
}

}  // namespace mom
