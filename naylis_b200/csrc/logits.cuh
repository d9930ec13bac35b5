// Rows of logits as the scoring kernels read them (scoring.cu, verify.cu).
#pragma once

#include "launch.h"
#include "tc_common.cuh"

namespace mom {

namespace {

constexpr float kNaN = __builtin_nanf("");

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

}  // namespace

}  // namespace mom
