// Causal attention over packed prompts: sequences of different lengths one after
// another in q (Tq, H, hd) and k, v (Tk, Hk, hd), query head h on key head
// h / (H / Hk), the mask aligned at each sequence's end (row r of a sequence of
// Lq queries and Lk keys sees keys 0 .. Lk - Lq + r).
//
// The plan lists tiles of up to kPromptRows query rows, the costliest first.
#include <algorithm>
#include <vector>

#include "common.cuh"
#include "launch.h"

namespace mom {

int64_t prompt_tiles(const int64_t *q_lens, int64_t n) {
    int64_t t = 0;
    for (int64_t i = 0; i < n; ++i) t += (q_lens[i] + kPromptRows - 1) / kPromptRows;
    return t;
}

void prompt_plan(const int64_t *q_lens, const int64_t *k_lens, int64_t n, PromptTile *tiles) {
    int64_t q0 = 0, k0 = 0, t = 0;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t lq = q_lens[i], lk = k_lens ? k_lens[i] : lq;
        for (int64_t r = 0; r < lq; r += kPromptRows, ++t) {
            tiles[t].q0 = static_cast<int32_t>(q0 + r);
            tiles[t].rows = static_cast<int32_t>(std::min<int64_t>(kPromptRows, lq - r));
            tiles[t].k0 = static_cast<int32_t>(k0);
            tiles[t].vis = static_cast<int32_t>(lk - lq + r + 1);
        }
        q0 += lq;
        k0 += lk;
    }
    std::stable_sort(tiles, tiles + t, [](const PromptTile &a, const PromptTile &b) {
        return a.vis + a.rows > b.vis + b.rows;
    });
}

namespace {

// One warp per (row, head): 32 keys at a time, lane = key for the scores and
// lane = hd/32 dimensions for the sum over values.
template <int HD>
__global__ void __launch_bounds__(128)
prompt_kernel(const uint16_t *__restrict__ q, int64_t q_ld, const uint16_t *__restrict__ k, int64_t k_ld,
              const uint16_t *__restrict__ v, int64_t v_ld, const PromptTile *__restrict__ tiles, int64_t n_tiles,
              int H, int Hk, float scale_log2, uint16_t *__restrict__ out) {
    constexpr int kD = HD / 32;
    __shared__ float sq[4][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = blockIdx.x;
    const PromptTile t = tiles[item / H];
    const int h = static_cast<int>(item % H), hk = h / (H / Hk);
    for (int r = warp; r < t.rows; r += 4) {
        const int64_t row = t.q0 + r;
        const int n = t.vis + r;
        __syncwarp();
        for (int d = lane; d < HD; d += 32) sq[warp][d] = bf16_bits_to_f32(q[row * q_ld + h * HD + d]);
        __syncwarp();
        float m = -INFINITY, l = 0.0f, acc[kD] = {};
        for (int j0 = 0; j0 < n; j0 += 32) {
            const int j = j0 + lane;
            float s = -INFINITY;
            if (j < n) {
                const uint4 *kr = reinterpret_cast<const uint4 *>(k + (static_cast<int64_t>(t.k0) + j) * k_ld + hk * HD);
                s = 0.0f;
                for (int d = 0; d < HD / 8; ++d) {
                    const uint4 w = kr[d];
                    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s += sq[warp][8 * d + 2 * e] * __uint_as_float(a[e] << 16) +
                             sq[warp][8 * d + 2 * e + 1] * __uint_as_float(a[e] & 0xFFFF0000u);
                }
                s *= scale_log2;
            }
            float mx = s;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m, mx), mr = mn == -INFINITY ? 0.0f : mn;
            const float f = exp2f(m - mr), p = j < n ? exp2f(s - mr) : 0.0f;
            l = l * f + warp_sum(p);
#pragma unroll
            for (int d = 0; d < kD; ++d) acc[d] *= f;
            const int cnt = min(32, n - j0);
            for (int e = 0; e < cnt; ++e) {
                const float pe = __shfl_sync(0xffffffffu, p, e);
                const uint16_t *vr = v + (static_cast<int64_t>(t.k0) + j0 + e) * v_ld + hk * HD + lane * kD;
#pragma unroll
                for (int d = 0; d < kD; ++d) acc[d] += pe * bf16_bits_to_f32(vr[d]);
            }
            m = mn;
        }
        uint16_t *dst = out + (row * H + h) * HD + lane * kD;
#pragma unroll
        for (int d = 0; d < kD; ++d) dst[d] = f32_to_bf16_bits(n > 0 ? acc[d] / l : 0.0f);
    }
}

}  // namespace

cudaError_t launch_prompt_attn(const void *q, int64_t q_ld, const void *k, int64_t k_ld, const void *v, int64_t v_ld,
                               int64_t Tq, int64_t Tk, const PromptTile *tiles, int64_t n_tiles, int *err, int H,
                               int Hk, int hd, float scale, void *out, cudaStream_t st) {
    (void)Tq, (void)Tk, (void)err;
    const unsigned grid = static_cast<unsigned>(n_tiles * H);
    auto go = [&](auto kernel) {
        kernel<<<grid, 128, 0, st>>>(static_cast<const uint16_t *>(q), q_ld, static_cast<const uint16_t *>(k), k_ld,
                                     static_cast<const uint16_t *>(v), v_ld, tiles, n_tiles, H, Hk, scale * kLog2e,
                                     static_cast<uint16_t *>(out));
    };
    if (hd == 64) go(prompt_kernel<64>);
    else go(prompt_kernel<128>);
    count_launch();
    return cudaGetLastError();
}

}  // namespace mom
