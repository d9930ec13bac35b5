// Causal attention over packed prompts on the 5th-generation tensor cores: sequences
// of different lengths one after another in q (Tq, H, hd) and k, v (Tk, Hk, hd), query
// head h on key head h / (H / Hk), the mask aligned at each sequence's end (row r of a
// sequence of Lq queries and Lk keys sees keys 0 .. Lk - Lq + r).
//
//   O[r] = sum_j 2^(x_rj - m_r) v_j / sum_j 2^(x_rj - m_r),  x = (scale log2 e) q . k
//
// in one pass over the keys: m is the row's running maximum, and O and the sum are
// rescaled only when it has grown by more than 2^8 (the weights then stay below 2^8,
// exact enough in bf16, whose relative step does not depend on their size; the sum is
// fp32). The weights are rounded to bf16 for the second product, as its operand type
// asks; the output is rounded once.
//
// A CTA works on two halves of 128 rows that share their keys: two heads of a group
// where the group is even (the halves then see the same keys and a tile of 128 rows
// wastes less on short sequences), else 256 rows of a head. Per half a softmax
// warpgroup (one row a thread: no exchange between threads) and an issuing thread; one
// loader (K and V tiles of 128 keys through a ring, TMA), one epilogue warpgroup an
// item behind. Tensor memory is full at head_dim 128 (two S, two O of 128 columns).
//
// What bounds it, 148 SMs, B200: head_dim 128 the chain softmax - product with V -
// scores of the next tile of a half, under which the other half's is laid (a step of
// both halves takes about 2900 cycles; their products alone 2048): 8 sequences of 2048,
// 16 heads on 4, 130 us, 1.06 PFLOP/s of the causal half's flops, tensor pipe 56 % busy;
// one of 16384 862 us, 1.28 PFLOP/s (under a lasting load 990 us: the power limit takes
// the clock from 1.9 to 1.6 GHz). head_dim 64 has half the products for the same
// exponentials: bound by the special-function unit (63 %) and what the softmax waits
// for: 8 of 2048, 16 heads, 108 us, 635 TFLOP/s. Also tried: exponentials partly on the
// FMA pipe (no gain while the halves take turns; -2 % at head_dim 64), two softmax
// warps a row (more exchange than it hides: 717 against 711 us at 16384, head_dim 64),
// items handed out at run time (the waits for them cost more than their balance gave).
//
// The plan lists tiles of up to kPromptRows query rows and the work of each CTA.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <functional>
#include <queue>
#include <utility>
#include <vector>

#include "launch.h"
#include "tc_common.cuh"

namespace mom {

int64_t prompt_tiles(const int64_t *q_lens, int64_t n) {
    int64_t t = 0;
    for (int64_t i = 0; i < n; ++i) t += (q_lens[i] + kPromptRows - 1) / kPromptRows;
    return t;
}

// The tiles, and who does what: an item is a tile (or, where the halves of a CTA are two
// heads of a group, 128 rows of it) and a head (or two); the costliest goes first, each
// to the CTA that has the least to do. Cost: key tiles, and kItemCost for an item's
// start and end. (Dealt out in turn, back and forth, 24 sequences of 1 to 4099 left the
// busiest CTA 12 % over the mean.)
constexpr double kItemCost = 1.5;

void prompt_plan(const int64_t *q_lens, const int64_t *k_lens, int64_t n, int64_t H, int64_t Hk, void *plan) {
    const PromptLayout L = prompt_layout(prompt_tiles(q_lens, n), H);
    std::memset(plan, 0, L.bytes);
    char *base = static_cast<char *>(plan);
    PromptTile *tiles = reinterpret_cast<PromptTile *>(base + L.tiles);
    int32_t *first = reinterpret_cast<int32_t *>(base + L.first);
    int2 *items = reinterpret_cast<int2 *>(base + L.items);
    struct Job {
        float cost;
        int32_t tile, rem;
    };
    std::vector<Job> jobs;
    const bool pair = prompt_pairs(H, Hk);
    int64_t q0 = 0, k0 = 0, t = 0;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t lq = q_lens[i], lk = k_lens ? k_lens[i] : lq;
        for (int64_t r = 0; r < lq; r += kPromptRows, ++t) {
            PromptTile &x = tiles[t];
            x.q0 = static_cast<int32_t>(q0 + r);
            x.rows = static_cast<int32_t>(std::min<int64_t>(kPromptRows, lq - r));
            x.k0 = static_cast<int32_t>(k0);
            x.vis = static_cast<int32_t>(lk - lq + r + 1);
            for (int64_t rem = 0; rem < H; ++rem) {
                const int at = pair && rem < H / 2 ? kPromptRows / 2 : 0;
                const int rows = std::min(x.rows - at, pair ? kPromptRows / 2 : kPromptRows);
                if (rows <= 0) continue;
                const int keys = std::max(x.vis + at + rows - 1, 0);
                jobs.push_back(Job{static_cast<float>((keys + 127) / 128 + kItemCost), static_cast<int32_t>(t),
                                   static_cast<int32_t>(rem)});
            }
        }
        q0 += lq;
        k0 += lk;
    }
    std::stable_sort(jobs.begin(), jobs.end(), [](const Job &a, const Job &b) { return a.cost > b.cost; });
    using Load = std::pair<double, int>;      // work so far, CTA
    std::priority_queue<Load, std::vector<Load>, std::greater<Load>> least;
    for (int c = 0; c < kPromptCtas; ++c) least.push({0.0, c});
    std::vector<int> of(jobs.size());
    for (size_t j = 0; j < jobs.size(); ++j) {
        Load l = least.top();
        least.pop();
        of[j] = l.second;
        ++first[l.second + 1];
        l.first += jobs[j].cost;
        least.push(l);
    }
    for (int c = 0; c < kPromptCtas; ++c) first[c + 1] += first[c];
    std::vector<int32_t> at(first, first + kPromptCtas);
    for (size_t j = 0; j < jobs.size(); ++j) items[at[of[j]]++] = int2{jobs[j].tile, jobs[j].rem};
}

namespace {

constexpr int kM = 128;                        // query rows of a half (TMEM lanes)
constexpr int kN = 128;                        // keys of a tile
constexpr int kThreads = 512;
constexpr uint32_t kBox = 128 * 128;           // one TMA box: 128 rows x 64 bf16 columns
// Tensor memory: S of half A, S of half B, O of A, O of B and, at head_dim 64, P of A, P of
// B (bf16 pairs, 64 columns each). At head_dim 128 the columns are full: P takes the first
// 64 of its S.
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSCol = 0, kOCol = 256, kPCol = 384;
constexpr float kRescale = 8.0f;               // log2 growth of a row maximum that O is rescaled for

template <int HD>
struct Cfg {
    static constexpr int kBoxes = HD / 64;
    static constexpr int kQBufs = HD == 64 ? 2 : 1;           // items whose Q is held
    static constexpr uint32_t kQ = 2 * kQBufs * kN * HD * 2;
    static constexpr bool kOwnP = HD == 64;                   // P has columns of its own
    static constexpr uint32_t kTile = kN * HD * 2;            // a K, V or Q tile
    // registers of a thread of the softmax (8 warps), the epilogue (4) and the others (4)
    static constexpr int kSoftRegs = 184, kEpiRegs = 80, kRestRegs = 64;
    static_assert(32 * (8 * kSoftRegs + 4 * kEpiRegs + 4 * kRestRegs) <= 512 * 128, "registers at launch");
    static constexpr int kStages = HD == 64 ? 8 : 4;          // K and V tiles in turn
    static constexpr uint32_t kRing = kStages * kTile;
    static constexpr uint32_t kSum = 2 * 2 * kM * 4;          // row sums [item parity][half][row]
    static constexpr uint32_t kStage = kM * 128;              // 64 output columns of a half
    static constexpr uint32_t kSmem = kQ + kRing + kStage + kSum + 1024 /*barriers*/ + 1024 /*align*/;
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static_assert(16 * 4 * HD * 4 <= kQ, "redo_rows' columns");
};

struct Bars {
    uint64_t q_full[2][2], q_empty[2][2], kv_full[8], kv_empty[8], s_full[2], s_read[2], p_half[2], p_full[2], turn[2],
        pv_done[2], o_full[2], o_free[2], l_full[2][2], drain[2];
    uint32_t tmem_base;
    int abort;
    float zero;
};
static_assert(sizeof(Bars) <= 1024, "barrier block");

struct Params {
    const PromptTile *tiles;
    const int32_t *first;
    const int2 *items;
    int H, Hk, pair;      // pair: the halves are two heads of a group, else two runs of rows
    float scale_log2;
    const uint16_t *q, *k, *v;
    int64_t q_ld, k_ld, v_ld, Tk;
    uint16_t *out;
    int *err;
};

struct Half {
    int q0, rows, vis, head, n;    // n: key tiles the half has to see
};
struct Item {
    Half h[2];
    int k0, n;
};

// The items of a CTA one after another, the next one's tile and the one after's entry
// fetched ahead.
struct Items {
    const Params &p;
    int i, end;
    int2 now, after;      // the next item's entry, the one after's
    PromptTile tile;      // the next item's

    __device__ __forceinline__ explicit Items(const Params &params) : p(params) {
        i = p.first[blockIdx.x];
        end = p.first[blockIdx.x + 1];
        if (i < end) now = p.items[i];
        if (i + 1 < end) after = p.items[i + 1];
        if (i < end) tile = p.tiles[now.x];
    }
    __device__ __forceinline__ bool get(Item &it) {      // false: no more
        if (i >= end) return false;
        const PromptTile t = tile;
        const int rem = now.y;
        now = after;
        if (++i < end) tile = p.tiles[now.x];
        if (i + 1 < end) after = p.items[i + 1];
        const int sub = p.pair && rem < p.H / 2 ? 1 : 0;          // pairs: the later rows first
        const int hp = p.pair && !sub ? rem - p.H / 2 : rem;
        const int rows = t.rows - sub * kM;
        it.k0 = t.k0;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int at = p.pair ? sub * kM : a * kM, left = p.pair ? rows : rows - a * kM;
            it.h[a] = Half{t.q0 + at, min(max(left, 0), kM), t.vis + at, p.pair ? 2 * hp + a : rem, 0};
            it.h[a].n = left > 0 ? max(0, (it.h[a].vis + it.h[a].rows + kN - 2) >> 7) : 0;
        }
        it.n = max(it.h[0].n, it.h[1].n);
        return true;
    }
};
static_assert(kN == 128, "key tiles are counted by a shift");

// Whether a NaN or an infinity is in a pair of bf16.
__device__ __forceinline__ bool not_finite(uint32_t pair) {
    return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}

// What hidden values that are not finite did to the CTA's rows, undone: a warp takes 16
// rows of a half. A column is spoilt for a row if the tiles that the mask cuts hold such
// a value there behind the row's last key. Values that the row does see decide the column
// where they are not finite; else the rows' sums are taken again without the others
// (m16n8k16 products, operands read as they lie). A row without a softmax (a score of NaN
// or +inf, or none above -inf) is NaN in every column and stays so. A call of 4096 tokens, 16
// heads on 4 of 128, takes 63 us; with values that are NaN throughout 121 (they decide
// everything: 1.1 ms for 860 us at 16384), with the last token's NaN 3.8 ms (16 at
// 16384), with +inf throughout 3.7 ms. (A thread a row, whatever it saw: 475 ms for NaN.)
template <int HD>
__device__ __forceinline__ void redo_rows(const Params &P) {
    constexpr int kC = HD / 32;      // columns of a lane
    constexpr unsigned kAll = 0xffffffffu;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = warp % 8 * 16;
    // of each column: the last value that is not finite in the cut tiles, the first NaN, +inf and -inf
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    int *last = reinterpret_cast<int *>(smem_raw) + warp * 4 * HD, *first = last + HD;
    Items items(P);
    for (Item it; items.get(it);) {
        const Half h = it.h[warp / 8];
        const int rows = min(h.rows - r0, 16);
        if (h.n == 0 || rows <= 0) continue;
        uint16_t *out = P.out + (static_cast<int64_t>(h.q0 + r0) * P.H + h.head) * HD;
        const int64_t out_ld = static_cast<int64_t>(P.H) * HD;
        bool spoilt = false;
#pragma unroll 4
        for (int i = lane; i < rows * (HD / 8); i += 32) {
            const uint4 x = *reinterpret_cast<const uint4 *>(out + i / (HD / 8) * out_ld + i % (HD / 8) * 8);
            spoilt |= not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
        }
        if (!__any_sync(kAll, spoilt)) continue;
        const int vis = h.vis + r0, hk = h.head / (P.H / P.Hk);      // row i sees vis + i keys
        const uint16_t *v = P.v + static_cast<int64_t>(it.k0) * P.v_ld + hk * HD;
        const uint16_t *k = P.k + static_cast<int64_t>(it.k0) * P.k_ld + hk * HD;
        const int cut = max(h.vis, 0) / kN * kN, end = min(h.n * kN, static_cast<int>(P.Tk) - it.k0);
        auto bad = [](uint32_t x) { return (x & 0x7f80u) == 0x7f80u; };
        auto values = [&](int j, uint32_t (&x)[kC / 2]) {      // this lane's columns
            const uint16_t *row = v + j * P.v_ld + lane * kC;
            if constexpr (kC == 4) {
                const uint2 y = *reinterpret_cast<const uint2 *>(row);
                x[0] = y.x, x[1] = y.y;
            } else {
                x[0] = *reinterpret_cast<const uint32_t *>(row);
            }
        };
        int at[kC], most = -1;
#pragma unroll
        for (int c = 0; c < kC; ++c) at[c] = -1;
#pragma unroll 4
        for (int j = cut; j < end; ++j) {
            uint32_t x[kC / 2];
            values(j, x);
#pragma unroll
            for (int c = 0; c < kC; ++c)
                if (bad(x[c / 2] >> (16 * (c & 1)))) at[c] = j;
        }
#pragma unroll
        for (int c = 0; c < kC; ++c) most = max(most, at[c]);
        if (!__any_sync(kAll, most >= vis)) continue;      // the first row sees the fewest
        __syncwarp();
        int begin[3][kC];
#pragma unroll
        for (int c = 0; c < kC; ++c) begin[0][c] = begin[1][c] = begin[2][c] = INT32_MAX;
        for (int j0 = 0; j0 < end; j0 += 8) {
            bool open = false;      // a column that is spoilt for some row, without a NaN so far
#pragma unroll
            for (int c = 0; c < kC; ++c) open |= at[c] >= vis && begin[0][c] == INT32_MAX;
            if (!__any_sync(kAll, open)) break;
            uint32_t x[8][kC / 2];
#pragma unroll
            for (int e = 0; e < 8; ++e) values(min(j0 + e, end - 1), x[e]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const uint32_t y = x[e][c / 2] >> (16 * (c & 1)) & 0xffffu;
                    const int j = min(j0 + e, end - 1);
                    if ((y & 0x7fffu) > 0x7f80u) begin[0][c] = min(begin[0][c], j);
                    if (y == 0x7f80u) begin[1][c] = min(begin[1][c], j);
                    if (y == 0xff80u) begin[2][c] = min(begin[2][c], j);
                }
        }
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            last[lane * kC + c] = at[c];
#pragma unroll
            for (int i = 0; i < 3; ++i) first[lane * kC + c + i * HD] = begin[i][c];
        }
        __syncwarp();
        // what the values seen make of a column: 0 finite, else the result
        auto decided = [&](int seen, int c) -> uint16_t {
            const bool nan = first[c] < seen, up = first[c + HD] < seen, down = first[c + 2 * HD] < seen;
            return nan || (up && down) ? 0x7fff : up ? 0x7f80 : down ? 0xff80 : 0;
        };
        uint32_t sums = 0;      // rows whose sums are needed
        for (int i = 0; i < rows; ++i) {
            const int seen = vis + i;
            bool lost = true, need = false, set = false;
            for (int c = lane; c < HD; c += 32) {
                const uint16_t to = decided(seen, c);
                const bool fix = seen > 0 && last[c] >= seen && to != 0x7fff;
                need |= fix && to == 0;
                set |= fix;
                lost &= (out[i * out_ld + c] & 0x7fff) > 0x7f80;
            }
            if (!__any_sync(kAll, set)) continue;
            if (__any_sync(kAll, need) || __all_sync(kAll, lost)) {
                sums |= 1u << i;
                continue;
            }
            for (int c = lane; c < HD; c += 32) {
                const uint16_t to = decided(seen, c);
                if (last[c] >= seen && to != 0x7fff) out[i * out_ld + c] = to;
            }
        }
        if (sums == 0) continue;
        const int r = lane >> 2, d = 2 * (lane & 3), far = vis + rows;      // far: keys that some row sees, and one
        const uint16_t *q0 = P.q + static_cast<int64_t>(h.q0 + r0 + min(r, rows - 1)) * P.q_ld + h.head * HD + d;
        const uint16_t *q1 = P.q + static_cast<int64_t>(h.q0 + r0 + min(r + 8, rows - 1)) * P.q_ld + h.head * HD + d;
        auto pair = [](const uint16_t *p) { return *reinterpret_cast<const uint32_t *>(p); };
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 64) {
            float acc[8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll 1
            for (int j0 = 0; j0 < far - 1; j0 += 16) {
                float s[2][4] = {};
#pragma unroll 2
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t a[4] = {pair(q0 + 16 * kk), pair(q1 + 16 * kk), pair(q0 + 16 * kk + 8),
                                           pair(q1 + 16 * kk + 8)};
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint16_t *kr = k + min(j0 + 8 * u + r, far - 2) * P.k_ld + 16 * kk + d;
                        mma_bf16_16816(s[u], a, pair(kr), pair(kr + 8));
                    }
                }
                float top[2] = {m[0], m[1]};
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool in = j0 + 8 * u + d + (e & 1) < vis + r + 8 * (e >> 1);
                        s[u][e] = in ? s[u][e] * P.scale_log2 : -INFINITY;
                        top[e >> 1] = fmaxf(top[e >> 1], s[u][e]);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[i] = fmaxf(top[i], __shfl_xor_sync(kAll, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(kAll, top[i], 2));
                    const float f = top[i] > m[i] ? tc::ex2(m[i] - top[i]) : 1.0f;
                    m[i] = top[i];
                    l[i] *= f;
#pragma unroll
                    for (int t = 0; t < 8; ++t) acc[t][2 * i] *= f, acc[t][2 * i + 1] *= f;
                }
                uint32_t p[4];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float ref = m[i] == -INFINITY ? 0.0f : m[i];
                        const float x = tc::ex2(s[u][2 * i] - ref), y = tc::ex2(s[u][2 * i + 1] - ref);
                        l[i] += x + y;
                        p[2 * u + i] = pack_bf16x2(x, y);
                    }
                auto value = [&](int j, int c) {
                    const uint32_t x = v[min(j, far - 2) * P.v_ld + c];
                    return bad(x) ? 0u : x;
                };
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    const int c = c0 + 8 * t + r;
                    mma_bf16_16816(acc[t], p, value(j0 + d, c) | value(j0 + d + 1, c) << 16,
                                   value(j0 + d + 8, c) | value(j0 + d + 9, c) << 16);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l[i] += __shfl_xor_sync(kAll, l[i], 1);
                l[i] += __shfl_xor_sync(kAll, l[i], 2);
                const int row = r + 8 * i, seen = vis + row;
                if (row >= rows || !(sums >> row & 1u) || !(l[i] > 0.0f && l[i] < INFINITY)) continue;
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int c = c0 + 8 * t + d + e;
                        const uint16_t to = decided(seen, c);
                        if (last[c] >= seen && to != 0x7fff)
                            out[row * out_ld + c] = to ? to : f32_to_bf16_bits(acc[t][2 * i + e] / l[i]);
                    }
            }
            __syncwarp();
        }
    }
}

// The same as a call. Inlined, though never run, it costs the other code 0.5 us at
// head_dim 128 and up to 4 at 64 (64 sequences of 256: 36 -> 40 us), called 2 and 1.
template <int HD>
__device__ __noinline__ void call_redo_rows(const Params P) {
    redo_rows<HD>(P);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
prompt_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Params P) {
    using C = Cfg<HD>;
    constexpr int kStages = C::kStages;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ int s_again;      // set: a row that a hidden value may have spoilt
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char *sbase = smem_raw + (base - raw);
    const uint32_t ring = base + C::kQ;
    float *sSum = reinterpret_cast<float *>(sbase + C::kQ + C::kRing + C::kStage);
    Bars *bars = reinterpret_cast<Bars *>(sbase + C::kQ + C::kRing + C::kStage + C::kSum);
    volatile int *abort_flag = &bars->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int a = 0; a < 2; ++a) {
            tc::mbar_init(&bars->drain[a], 1);
            for (int q = 0; q < 2; ++q) {
                tc::mbar_init(&bars->q_full[a][q], 1);
                tc::mbar_init(&bars->q_empty[a][q], 1);
            }
            tc::mbar_init(&bars->s_full[a], 1);
            tc::mbar_init(&bars->s_read[a], kM);
            tc::mbar_init(&bars->pv_done[a], 1);
            tc::mbar_init(&bars->p_half[a], kM);
            tc::mbar_init(&bars->p_full[a], kM);
            tc::mbar_init(&bars->turn[a], kM);
            tc::mbar_init(&bars->o_full[a], 1);
            tc::mbar_init(&bars->o_free[a], kM);
            tc::mbar_init(&bars->l_full[a][0], kM);
            tc::mbar_init(&bars->l_full[a][1], kM);
        }
        for (int s = 0; s < kStages; ++s) {
            tc::mbar_init(&bars->kv_full[s], 1);
            tc::mbar_init(&bars->kv_empty[s], 2);
        }
        bars->abort = s_again = 0;
        bars->zero = 0.0f;
    }
    if (warp == 12) {
        tc::tmem_alloc(&bars->tmem_base, kTmemCols);
        tc::tmem_relinquish();
    }
    if (warp == 14 && lane == 0) {
        tc::prefetch_tensormap(&tmap_q);
        tc::prefetch_tensormap(&tmap_k);
        tc::prefetch_tensormap(&tmap_v);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        return tc::mbar_wait_warp(bar, parity, P.err, 2, abort_flag);
    };

    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        // Warps 0-3: half A, 4-7: half B; a thread holds one row of scores.
        tc::regs_inc<C::kSoftRegs>();
        const int a = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t tS = tmem + kSCol + a * kN + lanes, tO = tmem + kOCol + a * HD + lanes;
        const uint64_t sc2 = tc::f2(P.scale_log2, P.scale_log2);
        const uint32_t tP = C::kOwnP ? tmem + kPCol + a * 64 + lanes : tS;
        int phase = 0, par = 0, pv = 0;     // tiles begun, item parity, tiles whose product was waited for
        int turns = 0;                      // turns of the other half waited for
        bool ok = true, owed = false;       // owed: the other half's turn has to come before this one's next
        Items items(P);
        for (Item it; ok && items.get(it);) {
            const Half h = it.h[a];
            float m = -INFINITY, l = 0.0f;
            // wait for PV of the tile before the present one, once a tile
            auto pv_done = [&] {
                if (pv < phase - 1) {
                    ok = wait(&bars->pv_done[a], (phase - 2) & 1);
                    pv = phase - 1;
                    if (ok) tc::tc_fence_after();
                }
                return ok;
            };
            for (int j = 0; j < h.n; ++j) {
                if (!(ok = wait(&bars->s_full[a], phase & 1))) break;
                ++phase;
                tc::tc_fence_after();
                // cut tiles (warp-uniform: the warp's first row sees less than all): the hidden scores
                // become -inf where they lie, in a rolled loop, since this code is run once an item
                // and an unrolled select over the registers below costs more to fetch than to do
                const int seen = h.vis + r - j * kN;
                if (h.vis + quarter * 32 - j * kN < kN) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        const int first = h.vis + quarter * 32 - j * kN - 32 * c;      // what the warp's first row sees
                        if (first >= 32) continue;
                        uint32_t x[32];
                        if (first > -31) {
                            tc::tmem_ld32(tS + 32 * c, x);
                            tc::tmem_ld_wait();
                            const int left = min(max(seen - 32 * c, 0), 32);
                            const uint32_t keep = left == 32 ? 0xffffffffu : (1u << left) - 1u;
#pragma unroll
                            for (int e = 0; e < 32; ++e) x[e] = keep >> e & 1u ? x[e] : __float_as_uint(-INFINITY);
                        } else {      // hidden from all of them
#pragma unroll
                            for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(-INFINITY);
                        }
                        tc::tmem_st32(tS + 32 * c, x);
                    }
                    tc::tmem_st_wait();
                }
                uint32_t v[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tc::tmem_ld32(tS + 32 * c, v[c]);
                tc::tmem_ld_wait();
                if constexpr (C::kOwnP) {
                    tc::tc_fence_before();
                    tc::mbar_arrive(&bars->s_read[a]);
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    mx[c] = __uint_as_float(v[c][0]);
#pragma unroll
                    for (int e = 1; e < 31; e += 2)
                        mx[c] = tc::fmax3(mx[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
                    mx[c] = fmaxf(mx[c], __uint_as_float(v[c][31]));
                }
                // (a score of NaN or +inf makes its own weight NaN, and with it the row's sum)
                const float top = fmaxf(tc::fmax3(mx[0], mx[1], mx[2]), mx[3]);
                const float mn = fmaxf(m, top * P.scale_log2);
                if (j == 0) {
                    m = mn;
                } else if (__any_sync(0xffffffffu, mn > m + kRescale)) {
                    // O holds tiles 0 .. j-1 once PV(j-1) is done; with P in S's columns S(j) was
                    // issued behind it
                    if (C::kOwnP && !pv_done()) break;
                    const float mo = m == -INFINITY ? mn : m;
                    const float f = mn > m + kRescale ? tc::ex2(mo - mn) : 1.0f;
                    if (mn > m + kRescale) m = mn;
                    l *= f;
#pragma unroll
                    for (int c = 0; c < HD / 16; ++c) {
                        uint32_t o[16];
                        tc::tmem_ld16(tO + 16 * c, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tc::tmem_st16(tO + 16 * c, o);
                    }
                }
                // Turns (P in S's columns): the halves' exponentials one after the other, B's tile j
                // behind A's, A's next behind B's. In step they share the special-function unit and
                // then the tensor pipe, each idle while the other is fought over: 16384 rows, 16
                // heads 1060 us, in turns 900. Each turn is waited for exactly once.
                const bool shared = !C::kOwnP && j < min(it.h[0].n, it.h[1].n);
                if (!C::kOwnP && (a == 0 ? owed : shared)) {
                    if (!(ok = wait(&bars->turn[a ^ 1], turns++ & 1))) break;
                    owed = false;
                }
                const float mref = m == -INFINITY ? 0.0f : m;
                uint64_t l2[2] = {tc::f2(0.0f, 0.0f), tc::f2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t pk[32];
                    // a value read behind the hand-over of the first half keeps the second half's
                    // work there
                    const float ref = C::kOwnP || c == 0 ? mref : mref + *reinterpret_cast<volatile float *>(&bars->zero);
                    const uint64_t nm2 = tc::f2(-ref, -ref);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const uint32_t *s = &v[2 * c + (e >> 4)][2 * (e & 15)];
                        const uint64_t x2 = tc::fma2(tc::f2_bits(s[0], s[1]), sc2, nm2);
                        const uint64_t p2 = tc::ex2_pair(x2);
                        l2[e & 1] = tc::add2(l2[e & 1], p2);
                        const float2 p = tc::f2_split(p2);
                        pk[e] = pack_bf16x2(p.x, p.y);
                    }
                    if (C::kOwnP && c == 0 && phase > 1 && !pv_done()) break;   // the last P is read
                    tc::tmem_st32(tP + 32 * c, pk);
                    if (!C::kOwnP && c == 0) {
                        tc::tmem_st_wait();
                        tc::tc_fence_before();
                        tc::mbar_arrive(&bars->p_half[a]);
                    }
                }
                if (!ok) break;
                tc::tmem_st_wait();
                tc::tc_fence_before();
                tc::mbar_arrive(&bars->p_full[a]);
                if (shared) {
                    tc::mbar_arrive(&bars->turn[a]);
                    owed = true;
                }
                const float2 ls = tc::f2_split(tc::add2(l2[0], l2[1]));
                l += ls.x + ls.y;
            }
            if (!ok) break;
            if (h.n > 0) {
                sSum[(par * 2 + a) * kM + r] = l;
                // one barrier per item parity: a half may finish its next item before the epilogue
                // comes to this one, but not the one after
                tc::mbar_arrive(&bars->l_full[a][par]);
                par ^= 1;
            }
        }
    } else if (warp < 12) {
        // ------------------------------------------------------------ epilogue
        // One item behind the softmax: O / l to global, each thread one row.
        tc::regs_dec<C::kEpiRegs>();
        const int quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        uint4 *stage = reinterpret_cast<uint4 *>(sbase + C::kQ + C::kRing) + quarter * 32 * 8;
        int phase[2] = {0, 0};
        bool ok = true, again = false;
        Items items(P);
        for (Item it; ok && items.get(it);) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const Half h = it.h[a];
                if (h.n == 0) {
                    uint4 *dst = reinterpret_cast<uint4 *>(P.out + (static_cast<int64_t>(h.q0 + r) * P.H + h.head) * HD);
                    if (r < h.rows)
#pragma unroll
                        for (int c = 0; c < HD / 8; ++c) dst[c] = make_uint4(0, 0, 0, 0);
                    continue;
                }
                const int ph = phase[a]++;
                if (!(ok = wait(&bars->l_full[a][ph & 1], (ph >> 1) & 1) && wait(&bars->o_full[a], ph & 1))) break;
                tc::tc_fence_after();
                const float l = sSum[((ph & 1) * 2 + a) * kM + r];
                float big = 0.0f;      // the greatest magnitude of the row's sums, NaN if one is
                const float inv = h.vis + r > 0 ? 1.0f / l : 0.0f;
                const uint32_t tO = tmem + kOCol + a * HD + lanes;
                const bool none = h.vis + r <= 0;
                // 64 columns at a time to the warp's rows in shared memory (16-byte chunks swizzled
                // by row), from there to global in whole 128-byte runs; O is free once it is read
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t o[16];
                        tc::tmem_ld16(tO + 64 * c + 16 * e, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int z = 0; z < 16; z += 2)
                            big = tc::fmax3_nan(big, fabsf(__uint_as_float(o[z])), fabsf(__uint_as_float(o[z + 1])));
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            uint32_t pk[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                pk[y] = none ? 0u
                                             : pack_bf16x2(__uint_as_float(o[8 * z + 2 * y]) * inv,
                                                           __uint_as_float(o[8 * z + 2 * y + 1]) * inv);
                            stage[lane * 8 + ((2 * e + z) ^ (lane & 7))] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                        }
                    }
                    if (c + 1 == HD / 64) {
                        tc::tc_fence_before();
                        tc::mbar_arrive(&bars->o_free[a]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int z = 0; z < 8; ++z) {
                        const int row = 4 * z + (lane >> 3), chunk = lane & 7;
                        if (quarter * 32 + row < h.rows)
                            reinterpret_cast<uint4 *>(P.out + (static_cast<int64_t>(h.q0 + quarter * 32 + row) * P.H +
                                                               h.head) * HD + 64 * c)[chunk] =
                                stage[row * 8 + (chunk ^ (row & 7))];
                    }
                    __syncwarp();
                }
                again |= !(big < INFINITY) && l < INFINITY && r < h.rows && !none;
            }
        }
        if (ok && again) s_again = 1;
    } else {
        tc::regs_dec<C::kRestRegs>();
        if (warp < 14) {
            // -------------------------------------------------------- MMA issuers
            // Warp 12: half A, 13: half B, each one thread. Where P lives in S's columns: per key
            // tile PV, then S of the next tile (the tensor pipe keeps a thread's order); one half's
            // softmax runs under the other half's products. Where P has its own: S of the next
            // tile as soon as the softmax has read S, so that it never waits for products.
            const int a = warp - 12;
            const uint32_t idesc_s = tc::idesc_bf16_f32(kM, kN, false, false);
            const uint32_t idesc_o = tc::idesc_bf16_f32(kM, HD, false, true);
            const uint32_t tS = tc::uniform(tmem) + kSCol + a * kN, tO = tc::uniform(tmem) + kOCol + a * HD;
            const uint32_t tP = C::kOwnP ? tc::uniform(tmem) + kPCol + a * 64 : tS;
            const uint32_t sQ = tc::uniform(base) + a * C::kQBufs * C::kTile, sR = tc::uniform(ring);
            if (tc::elect_one()) {
                int qn = 0, pn = 0, on = 0;      // items begun, tiles, items with a product
                bool ok = true;
                auto wait1 = [&](uint64_t *bar, uint32_t parity) {
                    return tc::mbar_wait(bar, parity, P.err, 2, abort_flag);
                };
                auto full = [&](int u) { return wait1(&bars->kv_full[u % kStages], (u / kStages) & 1); };
                auto release = [&](int u) { tc::mma_commit(&bars->kv_empty[u % kStages]); };
                // a tile that this half has no use for: released once it is there, so that no two
                // of a half's releases fall into one phase of the barrier
                auto skip = [&](int u) {
                    const bool there = full(u);
                    if (there) tc::mbar_arrive(&bars->kv_empty[u % kStages]);
                    return there;
                };
                auto issue_s = [&](int u, bool last) {
                    const uint64_t ad = tc::smem_desc_sw128(sQ + (qn - 1) % C::kQBufs * C::kTile, 16, 1024);
                    const uint64_t bd = tc::smem_desc_sw128(sR + (u % kStages) * C::kTile, 16, 1024);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint64_t step = 1024u * (kk >> 2) + 2u * (kk & 3);
                        tc::mma_bf16_ss(tS, ad + step, bd + step, idesc_s, kk > 0);
                    }
                    tc::mma_commit(&bars->s_full[a]);
                    release(u);
                    if (last) tc::mma_commit(&bars->q_empty[a][(qn - 1) % C::kQBufs]);
                };
                // the half's key tiles one after another, items and all: tile j of the item's n, whose
                // K is the loader's tile t
                Items items(P);
                struct Cursor {
                    int j = 0, n = 0, rest = 0, t = -2;      // rest: tiles of the item behind the half's
                    bool live = true;
                    __device__ __forceinline__ bool last() const { return j + 1 == n; }
                };
                Cursor cs, cp;      // scores, products with V
                auto next = [&](Cursor &c) {
                    c.t += 2;      // loader tiles passed
                    if (++c.j < c.n) return;
                    c.t += 2 * c.rest;
                    Item it;
                    while ((c.live = items.get(it))) {
                        if (it.h[a].n > 0) break;
                        c.t += 2 * it.n;
                    }
                    c.j = 0;
                    c.n = it.h[a].n;
                    c.rest = it.n - c.n;
                };
                auto q_ready = [&] {
                    const int q = qn++;
                    return wait1(&bars->q_full[a][q % C::kQBufs], (q / C::kQBufs) & 1);
                };
                auto scores = [&](bool behind) {
                    ok = full(cs.t) && (cs.j > 0 || q_ready()) &&
                         (!behind || !C::kOwnP || wait1(&bars->s_read[a], (pn - 1) & 1));
                    if (ok) {
                        tc::tc_fence_after();
                        issue_s(cs.t, cs.last());
                    }
                };
                int passed = 0;      // loader tiles up to here are used or released
                auto pass_to = [&](int u) {
                    while (ok && passed < u) ok = skip(passed++);
                };
                next(cs);
                cp = cs;
                pass_to(cs.t);
                if (ok && cs.live) scores(false);
                while (ok && cp.live) {
                    next(cs);
                    ++pn;
                    // S of the next tile ahead of the product where the softmax's columns allow it
                    // and the ring reaches: its tile may be at most one that the half skips away
                    const bool lead = C::kOwnP && cs.live && cs.t - cp.t <= 4;
                    if (lead) scores(true);
                    const int uv = cp.t + 1;
                    ok = ok && full(uv) &&
                         (lead || !cs.live || cs.t != cp.t + 2 || full(cs.t)) &&
                         (cp.j > 0 || on == 0 || wait1(&bars->o_free[a], (on - 1) & 1)) &&
                         wait1(C::kOwnP ? &bars->p_full[a] : &bars->p_half[a], (pn - 1) & 1);
                    if (!ok) break;
                    if (cp.j == 0) ++on;
                    const uint64_t bv = tc::smem_desc_sw128(sR + (uv % kStages) * C::kTile, kBox, 1024);
                    tc::tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < kN / 16; ++kk) {
                        if (!C::kOwnP && kk == kN / 32) {      // the second half of P
                            if (!(ok = wait1(&bars->p_full[a], (pn - 1) & 1))) break;
                            tc::tc_fence_after();
                        }
                        tc::mma_bf16_ts(tO, tP + 8 * kk, bv + 128 * kk, idesc_o, cp.j > 0 || kk > 0);
                    }
                    if (!ok) break;
                    if (C::kOwnP) tc::mma_commit(&bars->pv_done[a]);
                    release(uv);
                    if (cp.last()) tc::mma_commit(&bars->o_full[a]);
                    passed = cp.t + 2;
                    pass_to(cs.t);
                    if (ok && !lead && cs.live) scores(true);
                    cp = cs;
                }
                tc::mma_commit(&bars->drain[a]);
                wait1(&bars->drain[a], 0);
            }
            __syncwarp();
        } else if (warp == 14) {
            // -------------------------------------------------------- loader
            int t = 0, qn[2] = {0, 0};
            bool ok = true;
            auto slot = [&](int u) { return u < kStages || wait(&bars->kv_empty[u % kStages], (u / kStages - 1) & 1); };
            auto load_kv = [&](const CUtensorMap *map, int u, int x, int y) {
                if (lane == 0) {
                    uint64_t *bar = &bars->kv_full[u % kStages];
                    tc::mbar_arrive_expect_tx(bar, C::kTile);
#pragma unroll
                    for (int c = 0; c < C::kBoxes; ++c)
                        tc::tma_load_2d(ring + (u % kStages) * C::kTile + c * kBox, map, x + 64 * c, y, bar);
                }
                __syncwarp();
            };
            Items items(P);
            for (Item it; ok && items.get(it);) {
                if (it.n == 0) continue;
                auto load_q = [&](int a) {
                    if (it.h[a].n == 0) return;
                    const int q = qn[a]++, buf = q % C::kQBufs;
                    if (q >= C::kQBufs && !(ok = wait(&bars->q_empty[a][buf], (q / C::kQBufs - 1) & 1))) return;
                    if (lane == 0) {
                        tc::mbar_arrive_expect_tx(&bars->q_full[a][buf], C::kTile);
#pragma unroll
                        for (int c = 0; c < C::kBoxes; ++c)
                            tc::tma_load_2d(base + (a * C::kQBufs + buf) * C::kTile + c * kBox, &tmap_q,
                                            it.h[a].head * HD + 64 * c, it.h[a].q0, &bars->q_full[a][buf]);
                    }
                    __syncwarp();
                };
                const int x = it.h[0].head / (P.H / P.Hk) * HD;
                for (int j = 0; ok && j < it.n; ++j) {
                    if (!(ok = slot(t))) break;
                    load_kv(&tmap_k, t, x, it.k0 + j * kN);
                    ++t;
                    if (j == 0) load_q(0);
                    if (!ok || !(ok = slot(t))) break;
                    load_kv(&tmap_v, t, x, it.k0 + j * kN);
                    ++t;
                    if (j == 0) load_q(1);      // half A need not wait for B to leave its last item
                }
            }
            // no copy may be in flight when the CTA retires
            for (int u = max(0, t - kStages); u < t; ++u) wait(&bars->kv_full[u % kStages], (u / kStages) & 1);
#pragma unroll
            for (int a = 0; a < 2; ++a)
                for (int q = max(0, qn[a] - C::kQBufs); q < qn[a]; ++q)
                    wait(&bars->q_full[a][q % C::kQBufs], (q / C::kQBufs) & 1);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 12) tc::tmem_dealloc(tmem, kTmemCols);
    // A weight of 0 does not hide a NaN or an infinity from a product: rows that a value
    // behind the mask may have spoilt are looked at again, by all warps with the registers of
    // the launch, in the tiles' memory. (In the epilogue's loop the call would take registers from
    // it: 8 sequences of 2048, 16 heads on 4 of 128: 128 us, 136 with it.)
    if (s_again) {
        if (warp < 8) tc::regs_dec<128>();
        else tc::regs_inc<128>();
        if constexpr (HD == 128) redo_rows<HD>(P);
        else call_redo_rows<HD>(P);
    }
}

}  // namespace

cudaError_t launch_prompt_attn(const void *q, int64_t q_ld, const void *k, int64_t k_ld, const void *v, int64_t v_ld,
                               int64_t Tq, int64_t Tk, void *plan, int64_t n_tiles, int H, int Hk, int hd, float scale,
                               void *out, cudaStream_t st) {
    if (Tk == 0) return cudaMemsetAsync(out, 0, static_cast<size_t>(Tq) * H * hd * 2, st);
    CUtensorMap mq, mk, mv;
    if (!make_bf16_map_pitched(&mq, q, Tq, static_cast<uint64_t>(H) * hd, q_ld, kM) ||
        !make_bf16_map_pitched(&mk, k, Tk, static_cast<uint64_t>(Hk) * hd, k_ld, kN) ||
        !make_bf16_map_pitched(&mv, v, Tk, static_cast<uint64_t>(Hk) * hd, v_ld, kN))
        return cudaErrorInvalidValue;
    const PromptLayout L = prompt_layout(n_tiles, H);
    char *base = static_cast<char *>(plan);
    Params p;
    p.tiles = reinterpret_cast<const PromptTile *>(base + L.tiles);
    p.first = reinterpret_cast<const int32_t *>(base + L.first);
    p.items = reinterpret_cast<const int2 *>(base + L.items);
    p.H = H;
    p.Hk = Hk;
    p.pair = prompt_pairs(H, Hk);
    p.scale_log2 = scale * kLog2e;
    p.q = static_cast<const uint16_t *>(q);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    p.q_ld = q_ld;
    p.k_ld = k_ld;
    p.v_ld = v_ld;
    p.Tk = Tk;
    p.out = static_cast<uint16_t *>(out);
    p.err = static_cast<int *>(plan);
    const int grid = static_cast<int>(std::min<int64_t>(n_tiles * H, kPromptCtas));
    static std::atomic<uint64_t> ready{0};      // devices whose kernels have their shared memory set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        if ((e = cudaFuncSetAttribute(prompt_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      Cfg<64>::kSmem)) != cudaSuccess ||
            (e = cudaFuncSetAttribute(prompt_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      Cfg<128>::kSmem)) != cudaSuccess)
            return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    }
    auto go = [&](auto kernel, uint32_t smem) -> cudaError_t {
        kernel<<<grid, kThreads, smem, st>>>(mq, mk, mv, p);
        count_launch();
        return cudaGetLastError();
    };
    return hd == 64 ? go(prompt_tc_kernel<64>, Cfg<64>::kSmem) : go(prompt_tc_kernel<128>, Cfg<128>::kSmem);
}

}  // namespace mom
