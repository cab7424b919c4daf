// 4-bit matrices with group scales: the layout that mul_mat_q4 reads.
//
// A matrix of n rows of k numbers is held in tiles of 16 rows x 128 columns
// (rows and columns padded: padded rows and groups stand for 0, the columns
// that fill up a short group meet zeros of x), the tiles of 16 rows one
// after another and each in order of k, so that any run of a row tile's
// k-blocks is one run of memory.  A tile is
//   codes   [half 2][lane 32][4 words]: lane g * 4 + t of half h holds row
//           8 h + g; its word j the eight columns 32 j + 8 t + 0..7, columns i
//           and i + 4 (i < 4) in byte i, low and high, each as code - 8 in four
//           bits, so that a nibble at the top of a byte is 16 (code - 8).  A
//           word's low and high nibbles are operands of mma.m16n8k32 (rows g
//           and g + 8 of lane (g, t)) when the columns of x are taken in the
//           same order: a sum over k may take its terms in any order.
//   scales  [g 8][half 2][128 / group] FP16: what lane (g, t) needs of a tile
//           is one run of 16, 8 or 4 bytes.
//   minima  as the scales, present with `minimum`.
// value = scale (code - 8), or scale code + minimum.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/sdb.h"

namespace sdb {

struct Q4View {
    uint8_t* data;
    long long n, k;
    int tiles;        // of 16 rows
    int kblocks;      // of 128 columns
    int group;
    int ng;           // groups of a k-block: 128 / group
    int minimum;
    int block;        // bytes of a tile
};

constexpr long long kQ4MaxK = 1LL << 24;
constexpr long long kQ4MaxN = 1LL << 30;

inline bool q4_valid_form(int64_t k, int64_t n, int32_t group, int32_t minimum) {
    return k >= 1 && n >= 1 && k <= kQ4MaxK && n <= kQ4MaxN && (group == 32 || group == 64 || group == 128) &&
           (minimum == 0 || minimum == 1);
}

// Whether q describes a matrix with memory behind it.
inline bool q4_valid(const sdb_q4* q) {
    return q != nullptr && q->data != nullptr && (reinterpret_cast<uintptr_t>(q->data) & 15) == 0 &&
           q4_valid_form(q->k, q->n, q->group, q->minimum);
}

inline Q4View q4_view(const sdb_q4* q) {
    Q4View v{};
    v.n = q->n;
    v.k = q->k;
    v.group = q->group;
    v.ng = 128 / q->group;
    v.tiles = static_cast<int>((q->n + 15) / 16);
    v.kblocks = static_cast<int>((q->k + 127) / 128);
    v.minimum = q->minimum;
    v.block = 1024 + 32 * v.ng * (q->minimum ? 2 : 1);
    v.data = static_cast<uint8_t*>(q->data);
    return v;
}

// A row of the matrix.
struct Q4RowAt {
    uint8_t* base;  // of its row tile
    int word0, scale0, block, ng, group_log;
    __device__ __forceinline__ Q4RowAt(const Q4View& v, long long r) {
        const int h = static_cast<int>(r >> 3) & 1, g = static_cast<int>(r) & 7;
        base = v.data + (r >> 4) * v.kblocks * v.block;
        word0 = (h * 32 + g * 4) * 16;
        scale0 = 1024 + (g * 2 + h) * v.ng * 2;
        block = v.block;
        ng = v.ng;
        group_log = v.ng == 4 ? 5 : v.ng == 2 ? 6 : 7;
    }
    // The word of columns k0..k0 + 7 (k0 a multiple of 8).
    __device__ __forceinline__ uint32_t* word(int k0) const {
        return reinterpret_cast<uint32_t*>(base + static_cast<long long>(k0 >> 7) * block + word0 + (k0 >> 3 & 3) * 16 +
                                           (k0 >> 5 & 3) * 4);
    }
    // The scale of column k; its minimum, if any, lies 16 ng numbers on.
    __device__ __forceinline__ __half* scale(int k) const {
        return reinterpret_cast<__half*>(base + static_cast<long long>(k >> 7) * block + scale0 + ((k & 127) >> group_log) * 2);
    }
};

// The bit of column i (0..7) of a word.
__host__ __device__ constexpr int q4_bit(int i) { return (i & 3) * 8 + (i >> 2) * 4; }

}  // namespace sdb
