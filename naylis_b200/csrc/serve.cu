// Rotary embedding with the cache write, and attention of one new token per
// sequence over a paged key-value cache.
//
// Cache layout: K and V pages (num_pages, Hk, page_size, hd) bf16, so that the
// keys of one head in one page are one contiguous run; a token's slot is
// page * page_size + offset. The page size is a power of two (8 .. 256): a
// key's page and offset are a shift and a mask.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

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
// One thread per (token, head, 8 rotation pairs).
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
// out[b, h] = sum_j softmax_j(scale q . k_j) v_j over the sequence's seq_lens[b]
// keys. One CTA per (chunk of keys, key head, sequence); one warp per query head
// of the group, its lanes hold hd/32 dimensions each.
template <int HD>
__global__ void __launch_bounds__(128)
decode_split_kernel(const uint16_t *__restrict__ q, int64_t q_ld, const uint16_t *__restrict__ kp,
                    const uint16_t *__restrict__ vp, int64_t n_pages, int page_shift,
                    const int32_t *__restrict__ table, int64_t table_ld, const int32_t *__restrict__ seq_lens,
                    int64_t max_len, int H, int Hk, int chunk, int n_chunks, float scale_log2,
                    uint16_t *__restrict__ out, float *__restrict__ part) {
    constexpr int kD = HD / 32;
    const int b = blockIdx.z, hk = blockIdx.y, c = blockIdx.x, G = H / Hk;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t len = seq_lens[b];
    const bool bad = len > max_len;
    const int64_t j0 = static_cast<int64_t>(c) * chunk, j1 = min(len, j0 + chunk);
    for (int g = warp; g < G; g += 4) {
        const int h = hk * G + g;
        float qv[kD], acc[kD], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < kD; ++d) {
            qv[d] = bf16_bits_to_f32(q[b * q_ld + static_cast<int64_t>(h) * HD + lane * kD + d]);
            acc[d] = 0.0f;
        }
        bool lost = bad;
        if (!bad)
            for (int64_t j = j0; j < j1; ++j) {
                const int64_t page = table[b * table_ld + (j >> page_shift)];
                if (page < 0 || page >= n_pages) {
                    lost = true;
                    break;
                }
                const int64_t row = ((page * Hk + hk) << page_shift) + (j & ((1 << page_shift) - 1));
                float s = 0.0f;
#pragma unroll
                for (int d = 0; d < kD; ++d) s += qv[d] * bf16_bits_to_f32(kp[row * HD + lane * kD + d]);
                s = warp_sum(s) * scale_log2;
                const float mn = fmaxf(m, s);
                const float f = m == mn ? 1.0f : exp2f(m - mn), p = exp2f(s - mn);
                l = l * f + p;
#pragma unroll
                for (int d = 0; d < kD; ++d)
                    acc[d] = acc[d] * f + p * bf16_bits_to_f32(vp[row * HD + lane * kD + d]);
                m = mn;
            }
        if (lost) l = __int_as_float(0x7fc00000);
        if (n_chunks == 1) {
#pragma unroll
            for (int d = 0; d < kD; ++d)
                out[(static_cast<int64_t>(b) * H + h) * HD + lane * kD + d] =
                    f32_to_bf16_bits(l == 0.0f ? 0.0f : acc[d] / l);
        } else {
            float *dst = part + ((static_cast<int64_t>(b) * H + h) * n_chunks + c) * (HD + 2);
#pragma unroll
            for (int d = 0; d < kD; ++d) dst[2 + lane * kD + d] = acc[d];
            if (lane == 0) {
                dst[0] = m;
                dst[1] = l;
            }
        }
    }
}

// One warp per (sequence, head): joins the chunks' partial sums.
template <int HD>
__global__ void __launch_bounds__(128)
decode_join_kernel(const float *__restrict__ part, int64_t rows, int n_chunks, uint16_t *__restrict__ out) {
    constexpr int kD = HD / 32;
    const int64_t r = blockIdx.x * 4LL + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (r >= rows) return;
    const float *src = part + r * n_chunks * (HD + 2);
    float m = -INFINITY, l = 0.0f, acc[kD] = {};
    for (int c = 0; c < n_chunks; ++c) m = fmaxf(m, src[c * (HD + 2)]);
    for (int c = 0; c < n_chunks; ++c) {
        const float mc = src[c * (HD + 2)], lc = src[c * (HD + 2) + 1];
        const float f = mc == -INFINITY ? (lc == lc ? 0.0f : lc) : exp2f(mc - m);
        l += f * lc;
#pragma unroll
        for (int d = 0; d < kD; ++d) acc[d] += f * src[c * (HD + 2) + 2 + lane * kD + d];
    }
#pragma unroll
    for (int d = 0; d < kD; ++d) out[r * HD + lane * kD + d] = f32_to_bf16_bits(l == 0.0f ? 0.0f : acc[d] / l);
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

DecodeSplit decode_split(int64_t B, int64_t H, int64_t Hk, int64_t max_len) {
    DecodeSplit s;
    (void)B, (void)H, (void)Hk;
    s.chunk = 512;
    s.n_chunks = static_cast<int>(std::max<int64_t>(1, (max_len + s.chunk - 1) / s.chunk));
    return s;
}

cudaError_t launch_decode_attn(const void *q, int64_t q_ld, const void *kp, const void *vp, int64_t n_pages,
                               int page_shift, const int32_t *table, int64_t table_ld, const int32_t *seq_lens,
                               int64_t max_len, int64_t B, int H, int Hk, int hd, float scale, void *out, float *part,
                               cudaStream_t st) {
    const DecodeSplit s = decode_split(B, H, Hk, max_len);
    const dim3 grid(s.n_chunks, Hk, static_cast<unsigned>(B));
    const float sl2 = scale * kLog2e;
    auto go = [&](auto kernel) {
        kernel<<<grid, 128, 0, st>>>(static_cast<const uint16_t *>(q), q_ld, static_cast<const uint16_t *>(kp),
                                     static_cast<const uint16_t *>(vp), n_pages, page_shift, table, table_ld,
                                     seq_lens, max_len, H, Hk, s.chunk, s.n_chunks, sl2,
                                     static_cast<uint16_t *>(out), part);
    };
    if (hd == 64) go(decode_split_kernel<64>);
    else go(decode_split_kernel<128>);
    count_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || s.n_chunks == 1) return e;
    const int64_t rows = B * H;
    const unsigned jg = static_cast<unsigned>((rows + 3) / 4);
    if (hd == 64) decode_join_kernel<64><<<jg, 128, 0, st>>>(part, rows, s.n_chunks, static_cast<uint16_t *>(out));
    else decode_join_kernel<128><<<jg, 128, 0, st>>>(part, rows, s.n_chunks, static_cast<uint16_t *>(out));
    count_launch();
    return cudaGetLastError();
}

}  // namespace mom
