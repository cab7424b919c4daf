// The kernel of the linear layers of a few rows with 4-bit weights (q4.cuh).
//
//   y[m][n] = sum_g d[n][g] S + o[n][g] sum_{k in g} x[m][k],
//   S = sum_{k in g} (q[n][k] - z[n][g]) x[m][k],
// z = 8 and o = 0, or with a minimum z the code nearest to 0, o = min + d z.
//
// The weights' bytes are the work: each is read once for up to 32 rows of x.
// The 16 weight rows of a tile are the M of an mma and the rows of x its N; S
// is summed over one group by the tensor core, from zero, and joins FP32 sums
// with the group's scale.  x enters whole, to its last bit, whatever lies beside
// a number in its row, in one of three forms:
//
// Digits (one row).  The row's 128 numbers of a k-block are scaled by a power of
//   two and split into two integers of 22 bits, three signed base-256 digits
//   each: six columns of an integer product (m16n8k32, s8 x s8).  A nibble at
//   the top of its byte is the operand 16 (q - 8): three instructions unpack
//   eight weights (8 - z times a column's sum makes them q - z).  The sum is
//   exact; it starts from 0x4b400000, so that its bits, read as FP32, are
//   1.5 * 2^23 + 16 S, and one subtraction makes it a number (|16 S| < 2^22).
//   Six digits hold the numbers down to 2^-19 of the k-block's greatest; a
//   k-block with smaller ones (0 apart), or at the ends of FP32's range, or with
//   an infinity or a NaN, is three BF16 columns as below (a row of nothing else:
//   8192 -> 28672 45.6 us, of digits 27.3).
// Pairs (two to four FP32 rows).  A row is the sum of three BF16 columns, each
//   of which takes the next eight of a number's 24 bits, and none has a range to
//   fall out of; two rows' columns are six of a product's eight (m16n8k16).  q - z
//   is exact: a nibble is 128 + q in BF16, less 128 + z.
// Floats (more rows, and all FP16 rows but one).  FP16 rows are one column each
//   as they are; FP32 rows three BF16 columns, in products of eight rows' first,
//   second and third parts.  The first parts' sums are apart from the others',
//   which are 2^-8 of them.
//
// (Digits unpack a weight in a third of the instructions and take one row of
// 8192 -> 28672 in 27.6 us where a pair takes 38; two rows' twelve columns would
// be two products, 43 us for a pair's 42.  Four rows take 56 us in pairs, 70 in
// a product of eight rows' parts.)
//
// A CTA has 8 or 16 working warps: WR tiles of rows side by side, WK warps to a
// tile that share its k-blocks, and up to eight CTAs of a cluster that share
// them again.  x is split once into shared memory, laid out so that neither a
// column's stores nor a slice's loads over eight columns meet a bank twice, and
// stays there for all the row tiles the CTA walks.  A product's unused columns
// are not stored: their lanes read what lies there and their sums go nowhere.
// A further warp brings the weights: a round, kRun k-blocks for every working
// warp, is one bulk copy for each of the WR tiles into one of kRing places,
// announced by an mbarrier and refilled when the working warps have said by
// another that they have read it.  The working warps' sums meet in shared memory
// and are added in one order, so a result does not turn on timing; the sums of a
// cluster's other CTAs are read where they lie.  Where there are few sums, one
// more warp finishes them (chain, gate, store) while the others go on.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "chain.cuh"
#include "ptx.cuh"
#include "q4.cuh"

namespace sdb {

constexpr int kQ4MaxShared = 227 * 1024;

// The parameters, in the order of their first use: a launch's parameters come from memory a line at a time, and
// what a CTA needs before its first copies is within two lines.
struct Q4Args {
    const uint8_t* w;          // tiles (q4.cuh)
    const uint8_t* gate;       // the gated form's second matrix
    int tiles, kblocks;        // of 16 rows; of 128 columns
    int groups;                // of WR row tiles
    int range;                 // k-blocks of a CTA (the last of a cluster may have fewer)
    int chunk;                 // k-blocks of x held at a time, a multiple of WK unless all of them
    uint8_t wk_log, wr_log;    // WK = 1 << wk_log warps to a tile, WR = 1 << wr_log tiles
    uint8_t cluster_log;       // CTAs that share a tile's k-blocks
    const void* x;
    long long xnb[3];          // strides of rows in elements (dims 1..3)
    int k;
    int rows;                  // of x
    uint8_t flat;              // rows along dimension 1 alone
    uint8_t x_half, x_vec;     // FP16 rows; their runs of four numbers are aligned
    uint8_t y_half;            // FP16 output
    int ne1, ne2;
    unsigned* err;             // the device error word
    void* y;
    long long ynb[3];
    int n;
    int act;                   // SDB_GATE_*
    Chain chain;
};

// Row m's coordinates along dimensions 1..3.
struct Q4Row {
    int i1, i2, i3;
    __device__ __forceinline__ Q4Row(const Q4Args& a, int m) : i1(m), i2(0), i3(0) {
        if (!a.flat) {
            const int q = m / a.ne1;
            i1 = m - q * a.ne1;
            i3 = q / a.ne2;
            i2 = q - i3 * a.ne2;
        }
    }
    __device__ __forceinline__ long long at(const long long (&nb)[3]) const {
        return i1 * nb[0] + i2 * nb[1] + i3 * nb[2];
    }
};

// A tile of weights (q4.cuh) as a lane holds it: the words of rows g and g + 8, the scales, the minima.
template <int G>
struct Q4Stage {
    static constexpr int kNg = 128 / G;
    static constexpr int kRun = 4 * kNg;  // bytes of a lane's scales: rows g and g + 8
    uint4 lo, hi;
    uint32_t d[kNg], m[kNg];

    static __device__ __forceinline__ void run(uint32_t (&r)[kNg], const uint8_t* p) {
        if constexpr (kNg == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
        } else if constexpr (kNg == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            r[0] = v.x; r[1] = v.y;
        } else {
            r[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ void read(const uint8_t* tile, int lane, bool minima) {
        lo = *reinterpret_cast<const uint4*>(tile + lane * 16);
        hi = *reinterpret_cast<const uint4*>(tile + 512 + lane * 16);
        run(d, tile + 1024 + lane / 4 * kRun);
        if (minima) run(m, tile + 1024 + 8 * kRun + lane / 4 * kRun);
    }
    // Group i's numbers of rows g and g + 8.
    static __device__ __forceinline__ float2 pick(const uint32_t (&r)[kNg], int i) {
        if constexpr (kNg == 1) return __half22float2(*reinterpret_cast<const __half2*>(&r[0]));
        const __half2 a = *reinterpret_cast<const __half2*>(&r[i / 2]);
        const __half2 b = *reinterpret_cast<const __half2*>(&r[kNg / 2 + i / 2]);
        return i & 1 ? make_float2(__high2float(a), __high2float(b)) : make_float2(__low2float(a), __low2float(b));
    }
};

// Splitting x: a warp takes a row's k-blocks, a lane columns 4 lane .. 4 lane + 3 of each.  With fewer rows than
// warps, warps / rows of them share a row.  The numbers come first, all of them in the background, into the very
// columns that take their fragments -- a lane's four into slot(k-block, row), 16 bytes (8, FP16, with HALF_SLOT) --
// in short loops of running addresses: what a CTA does once costs it the latency of its instructions.
struct Q4Items {
    int row, row_step, block, block_step;
    __device__ __forceinline__ Q4Items(int warps, int tokens) : row(threadIdx.x / 32), row_step(warps), block(0), block_step(1) {
        if (tokens < warps) {
            block_step = tokens == 1 ? warps : warps / tokens;
            block = tokens == 1 ? row : row / tokens;
            row -= block * tokens;
            if (block >= block_step) row = tokens;  // a warp too many
        }
    }
};

template <bool HALF_SLOT, class Slot>
__device__ __forceinline__ void q4_fetch(const Q4Args& a, const Q4Items& it, int m0, int tokens, int kb0, int blocks,
                                         Slot slot) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int m = it.row; m < tokens; m += it.row_step) {
        int k = (kb0 + it.block) * 128 + lane * 4;
        const long long at = Q4Row(a, m0 + m).at(a.xnb) + k;
        uint8_t* to = slot(it.block, m);
        const int to_step = static_cast<int>(slot(it.block_step, 0) - slot(0, 0));
        if (a.x_half) {
            const __half* from = static_cast<const __half*>(a.x) + at;
#pragma unroll 2
            for (int b = it.block; b < blocks; b += it.block_step) {
                if (a.x_vec && k + 4 <= a.k)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(to)), "l"(from) : "memory");
                else
                    for (int c = 0; c < 4; ++c)
                        reinterpret_cast<__half*>(to)[c] = k + c < a.k ? from[c] : __ushort_as_half(0);
                from += it.block_step * 128;
                k += it.block_step * 128;
                to += to_step;
            }
        } else if constexpr (!HALF_SLOT) {
            const float* from = static_cast<const float*>(a.x) + at;
#pragma unroll 2
            for (int b = it.block; b < blocks; b += it.block_step) {
                if (a.x_vec && k + 4 <= a.k)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
                else
                    for (int c = 0; c < 4; ++c) reinterpret_cast<float*>(to)[c] = k + c < a.k ? from[c] : 0.0f;
                from += it.block_step * 128;
                k += it.block_step * 128;
                to += to_step;
            }
        }
    }
}

// A lane's four numbers out of its slot.
template <bool HALF_SLOT>
__device__ __forceinline__ float4 q4_slot(const Q4Args& a, const uint8_t* from) {
    if (HALF_SLOT || a.x_half) {
        const uint2 r = *reinterpret_cast<const uint2*>(from);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
        return make_float4(f.x, f.y, h.x, h.y);
    }
    return *reinterpret_cast<const float4*>(from);
}

// split(k-block, row, x, store) of a warp's items, two at a time, whose chains of dependent steps overlap.
template <bool HALF_SLOT, class Slot, class Split>
__device__ __forceinline__ void q4_split(const Q4Args& a, const Q4Items& it, int tokens, int blocks, Slot slot, Split split) {
#pragma unroll 1
    for (int m = it.row; m < tokens; m += it.row_step)
#pragma unroll 1
        for (int b = it.block; b < blocks; b += 2 * it.block_step) {
            // Without a second item the first one's is computed again and not stored.
            const bool two = b + it.block_step < blocks;
            const int c = two ? b + it.block_step : b;
            const float4 x0 = q4_slot<HALF_SLOT>(a, slot(b, m)), x1 = q4_slot<HALF_SLOT>(a, slot(c, m));
            __syncwarp();  // every lane has its numbers: the fragments may take their places
            split(b, m, x0, true);
            split(c, m, x1, two);
        }
}

// The greatest magnitude of a warp's numbers, as FP32 bits (a NaN's bits are greater than an infinity's).
__device__ __forceinline__ uint32_t q4_top(float4 x) {
    const uint32_t a = max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu);
    const uint32_t b = max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu);
    return __reduce_max_sync(~0u, max(a, b));
}

// The sums of a warp's numbers, times `up`, over its groups of G, in every lane.
template <int G>
__device__ __forceinline__ float q4_group_sum(float4 x, float up) {
    float s = (x.x * up + x.y * up) + (x.z * up + x.w * up);
#pragma unroll
    for (int o = 1; o < G / 4; o <<= 1) s += __shfl_xor_sync(~0u, s, o);
    return s;
}

// Two FP32 numbers an instruction.
__device__ __forceinline__ uint64_t q4_pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 q4_unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t q4_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t q4_mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t q4_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// ---- operands

// The code nearest to 0 of rows g and g + 8 of a group, z, and what remains there, o = m + d z:
//   value = d (q - z) + o.
// With a minimum z is -m / d rounded and held to the codes, so that |o| <= |d| / 2, or o and all d (q - z) have one
// sign: neither term is far above the value, and a weight of 0 is two zeros.  (With 8 for all, or with d q + m as it
// stands, a great number of x whose weight is 0 would come in twice, with opposite signs.)
struct Q4Zero {
    uint32_t z[2] = {8, 8};
    float o[2] = {0.0f, 0.0f};
    __device__ __forceinline__ void of(float2 d, float2 m) {
        const float ds[2] = {d.x, d.y}, ms[2] = {m.x, m.y};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float inverse;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(ds[r]));
            // (d = 0 makes it infinite or NaN, which the bounds turn into a code)
            const float near = fminf(fmaxf(-ms[r] * inverse, 0.0f), 15.0f) + 12582912.0f;  // its last bits an integer
            z[r] = __float_as_uint(near) & 15u;
            o[r] = fmaf(ds[r], near - 12582912.0f, ms[r]);
        }
    }
};

// An integer below 2^m in the low bits of a number whose mantissa's last bit is worth 1 is that power of two plus
// the integer, so a nibble becomes a number by one logic operation and a subtraction.
// (u & MASK) ^ FLIP: two nibbles, code - 8 in four bits, made codes in such numbers.
template <uint32_t MASK, uint32_t FLIP>
__device__ __forceinline__ uint32_t q4_nibbles(uint32_t u) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(v) : "r"(u), "n"(MASK), "r"(FLIP));
    return v;
}

// FP16: nibbles at bits 0 and 16: 1024 + q, less 1024 + z.
__device__ __forceinline__ uint32_t q4_low(uint32_t u, uint32_t less) {
    uint32_t v;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(v) : "r"(q4_nibbles<0x000f000fu, 0x64086408u>(u)), "r"(less));
    return v;
}
__device__ __forceinline__ uint32_t q4_less_low(uint32_t z) { return 0x64006400u + z * 0x00010001u; }

// At bits 4 and 20: (1024 + 16 q) / 16, less 64 + z.
__device__ __forceinline__ uint32_t q4_high(uint32_t u, uint32_t less) {
    uint32_t v;
    asm("fma.rn.f16x2 %0, %1, %2, %3;"
        : "=r"(v)
        : "r"(q4_nibbles<0x00f000f0u, 0x64806480u>(u)), "r"(0x2c002c00u), "r"(less));
    return v;
}
__device__ __forceinline__ uint32_t q4_less_high(uint32_t z) { return 0xd400d400u + z * 0x00100010u; }

// BF16: nibbles at bits 0 and 16: 128 + q, less 128 + z.
__device__ __forceinline__ uint32_t q4_bf16(uint32_t u, uint32_t less) {
    uint32_t v;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(q4_nibbles<0x000f000fu, 0x43084308u>(u)), "r"(less));
    return v;
}
__device__ __forceinline__ uint32_t q4_less_bf16(uint32_t z) { return 0x43004300u + z * 0x00010001u; }

// c = a b, or c += a b, of FP16 (HALF) or BF16 operands.
template <bool HALF, bool FIRST>
__device__ __forceinline__ void q4_mma(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
    if constexpr (FIRST) c[0] = c[1] = c[2] = c[3] = 0.0f;
    if constexpr (HALF)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

// The operand of 16 columns, q - z, out of words of rows g and g + 8.
__device__ __forceinline__ void q4_bf16_words(uint32_t (&a)[4], uint32_t u0, uint32_t u1, const uint32_t (&less)[2]) {
    a[0] = q4_bf16(u0, less[0]);
    a[1] = q4_bf16(u1, less[1]);
    a[2] = q4_bf16(u0 >> 4, less[0]);
    a[3] = q4_bf16(u1 >> 4, less[1]);
}

// An FP32 row's k-block as three BF16 columns, x = a[0] + a[1] + a[2], whole: each takes the next eight bits at
// least.  Scaled by 2^24, so that the last parts of the smallest numbers too are normal ones; where `top`, the
// greatest number's bits, reaches 2^72, by 2^-24: 128 numbers below 2^72 by codes and a scale of 2^16 sum to less than
// 2^123 either way, and what lies below 2^-86 beside a number of 2^72 may lose bits.
__device__ __forceinline__ bool q4_three_great(uint32_t top) { return top >= 0x63800000u; }
__device__ __forceinline__ float q4_three_up(uint32_t top) { return q4_three_great(top) ? 0x1p-24f : 0x1p24f; }
__device__ __forceinline__ float q4_three_scale(uint32_t top) { return q4_three_great(top) ? 0x1p24f : 0x1p-24f; }

// A lane's four numbers are columns 0..3 or 4..7 of the run of eight that lane t = lane / 2 % 4 of a fragment
// holds: a word of slice 2 (lane / 8), the even columns, and one of the next, 32 bytes on, the odd ones.  `to`: the
// first column.
__device__ __forceinline__ int q4_float_word(int lane) { return (lane >> 3) * 64 + (lane >> 1 & 3) * 8 + (lane & 1) * 4; }
__device__ __forceinline__ void q4_put_three(float4 x, uint32_t top, uint8_t* to, int column) {
    to += q4_float_word(threadIdx.x & 31);
    const float up = q4_three_up(top);
    float v[4] = {x.x * up, x.z * up, x.y * up, x.w * up};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(v[2 * h], v[2 * h + 1]);
            v[2 * h] -= __low2float(a);
            v[2 * h + 1] -= __high2float(a);
            *reinterpret_cast<__nv_bfloat162*>(to + i * column + h * 32) = a;
        }
    }
}

// ---- one row, as digits: six of a product's eight columns

// 2^n as a number, n an exponent of normal numbers.
__device__ __forceinline__ float q4_power(int n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }

// Adding 1.5 * 2^23 rounds a number of up to 2^22 to an integer, which it leaves in the sum's low bits.
constexpr float kQ4Magic = 12582912.0f;
constexpr uint32_t kQ4MagicBits = 0x4b400000u;

// Three signed base-256 digits each of four such integers, a word of each column: adding 128 to the lower two makes
// the digits the integer's bytes.
__device__ __forceinline__ void q4_digits(const float (&n)[4], uint32_t* words) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (__float_as_uint(n[i]) + (0x8080u - kQ4MagicBits)) ^ 0x8080u;
    const uint32_t l01 = __byte_perm(v[0], v[1], 0x5140), l23 = __byte_perm(v[2], v[3], 0x5140);
    words[0] = __byte_perm(l01, l23, 0x5410);
    words[1] = __byte_perm(l01, l23, 0x7632);
    words[2] = __byte_perm(__byte_perm(v[0], v[1], 0x0062), __byte_perm(v[2], v[3], 0x0062), 0x5410);
}

template <bool GATED_>
struct Q4Digits {
    static constexpr bool GATED = GATED_;
    static constexpr int kTokens = 1;
    static constexpr int kTiles = GATED ? 2 : 1;
    static constexpr int kLaneSums = 1;          // of a tile, joined over the digits
    static constexpr int kWarps = !GATED ? 16 : 8;
    static constexpr int kRun = 2, kRing = 3;    // k-blocks of a warp a round; rounds on their way
    static constexpr bool kFinisher = true;      // a warp of its own finishes the sums
    static constexpr bool kWideRows = true;      // rows that digits do not hold are three BF16 columns
    static constexpr int kSlice = 224;           // bytes: six columns of 32 numbers, and a step of 8 banks
    static constexpr int kRow = 4 * kSlice;      // of a k-block
    static constexpr int kWide = 288;            // a column of a row that is not digits

    // Shared memory of `chunk` k-blocks: the columns; the factor, twice; the scale of a k-block that is not digits,
    // else 0; with a minimum the sums over each group of each column's digits and of x, of a k-block that is not digits
    // in that scale.
    static __host__ __device__ int block_bytes(int, int ng) { return kRow + 12 + 28 * ng; }
    // What the lanes of columns 6 and 7 read past the last, their factor, and what aligns the sums.
    static constexpr int kTail = 88;
    uint8_t* frags;
    float2* factors;
    const float2* own;  // the lane's, of columns 2 t and 2 t + 1: 0 for columns 6 and 7
    int own_step;
    float* scales;
    int2* column_sums;  // of a group's three pairs of columns
    float* sums;
    __device__ __forceinline__ Q4Digits(const Q4Args& a, uint8_t* x, int, int ng) {
        frags = x;
        factors = reinterpret_cast<float2*>(x + a.chunk * kRow + 80);
        const bool last = (threadIdx.x & 3) == 3;
        own = last ? factors - 1 : factors;
        own_step = last ? 0 : 1;
        scales = reinterpret_cast<float*>(factors + a.chunk);
        column_sums = reinterpret_cast<int2*>(scales + a.chunk + (a.chunk & 1));
        sums = reinterpret_cast<float*>(column_sums + 3 * ng * a.chunk);
    }

    // A slice of 32 columns of x is the six columns of its digits, 32 bytes each, a lane's four numbers a word of each.
    // read() once the numbers are on their way.  Returns whether the warp saw a row that is not digits.
    template <int G, bool MINIMA, class Read>
    __device__ __forceinline__ bool split(const Q4Args& a, int m0, int tokens, int kb0, int kb1, Read read) const {
        constexpr int NG = 128 / G;
        const int lane = threadIdx.x & 31;
        const Q4Items it(kWarps, tokens);
        bool seen = false;
        auto slot = [&](int b, int) { return frags + b * kRow + lane * 16; };
        q4_fetch<false>(a, it, m0, tokens, kb0, kb1 - kb0, slot);
        if (threadIdx.x == 0) factors[-1] = make_float2(0.0f, 0.0f);
        read();
        asm volatile("cp.async.wait_all;" ::: "memory");
        q4_split<false>(a, it, tokens, kb1 - kb0, slot, [&](int b, int, float4 x, bool store) {
            // The greatest number is below 2^(e - 126), e its exponent field: scaled by 2^(147 - e) all are below
            // 2^21.  Their integers are three digits; what is left of each, by 2^22, is three more, and nothing is
            // left of a number of the greatest's 2^-19 or more.
            const uint32_t top = q4_top(x);
            const int e = static_cast<int>(top >> 23);
            // Not digits: smaller numbers; those whose units or sums pass the ends of FP32's range; infinities, NaN.
            const bool out = e >= 240 || (e < 40 && top != 0);
            const float least = q4_power(max(e, 40) - 146), up = q4_power(147 - max(e, 40));
            const float n[4] = {x.x, x.y, x.z, x.w};
            float first[4], second[4];
            bool left = out;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                first[i] = fmaf(n[i], up, kQ4Magic);
                second[i] = fmaf(fmaf(n[i], up, kQ4Magic - first[i]), 0x1p22f, kQ4Magic);
                left |= fabsf(n[i]) < least && n[i] != 0.0f;
            }
            const bool wide = __any_sync(~0u, left);
            uint32_t words[6];
            q4_digits(first, words);
            q4_digits(second, words + 3);
            uint8_t* row = frags + b * kRow;
            if (store && !wide) {
                uint32_t* to = reinterpret_cast<uint32_t*>(row + (lane >> 3) * kSlice) + (lane & 7);
#pragma unroll
                for (int c = 0; c < 6; ++c) to[8 * c] = words[c];
            } else if (store) {
                q4_put_three(x, top, row, kWide);
            }
            // The factor is that of column 2, with the weights' 1 / 16: 2^16 2^(e - 147) / 16.  (The last two columns
            // are not there: any bytes are integers, and theirs count nothing.)
            if (store && lane == 0) {
                const float f = out || top == 0 ? 0.0f : q4_power(e - 135);
                factors[b] = make_float2(f, f);
                scales[b] = wide ? q4_three_scale(top) : 0.0f;
            }
            seen |= wide;
            if constexpr (MINIMA) {
                const float s = q4_group_sum<G>(x, wide ? q4_three_up(top) : 1.0f);
                // A sum of up to 128 digits has 15 bits: two columns' in a word.
                int pairs[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    pairs[p] = __dp4a(static_cast<int>(words[2 * p]), 0x01010101, 0) +
                               __dp4a(static_cast<int>(words[2 * p + 1]), 0x01010101, 0) * 65536;
                    for (int o = 1; o < G / 4; o <<= 1) pairs[p] += __shfl_xor_sync(~0u, pairs[p], o);
                }
                if (store && lane % (G / 4) == 0) {
                    const int at = b * NG + lane / (G / 4);
                    sums[at] = s;
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const int low = static_cast<short>(pairs[p]);
                        column_sums[3 * at + p] = make_int2(low, (pairs[p] - low) >> 16);
                    }
                }
            }
        });
        return seen;
    }

    uint64_t acc[kTiles][2];  // columns 2 t and 2 t + 1 of rows g, g + 8, in the factors' unit
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) acc[i][0] = acc[i][1] = 0;
    }

    // c = a b + (first, first, first, first), or c += a b.  With a minimum a product begins from what makes its weights
    // q - z: 16 (8 - z) times its column's sum, exact like the rest (|16 (q - z)| <= 240 leaves |sum| < 2^22).
    template <bool FIRST>
    static __device__ __forceinline__ void mma(int (&c)[4], const uint32_t (&a)[4], uint2 b) {
        if constexpr (FIRST)
            asm volatile(
                "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                "{%10, %10, %10, %10};"
                : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0x4b400000));
        else
            asm volatile(
                "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                "{%0, %1, %2, %3};"
                : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    }

    __device__ __forceinline__ bool wide(int at) const { return scales[at] != 0.0f; }

    // A k-block that is not digits, its three BF16 columns one product.  Its sums, whole, take the place of column 7,
    // lane (g, 3).
    template <int G, bool MINIMA>
    __device__ __forceinline__ void wide_product(const Q4Stage<G> (&st)[kTiles], int at) {
        constexpr int NG = 128 / G, SL = 4 / NG;
        const int lane = threadIdx.x & 31;
        const float scale = scales[at];
        // The lanes of columns past the third read the third's: their sums go nowhere.
        const uint8_t* f = frags + at * kRow + min(lane >> 2, 2) * kWide + (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const uint32_t u[2][4] = {{st[i].lo.x, st[i].lo.y, st[i].lo.z, st[i].lo.w},
                                      {st[i].hi.x, st[i].hi.y, st[i].hi.z, st[i].hi.w}};
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float2 d = Q4Stage<G>::pick(st[i].d, g);
                Q4Zero zero;
                if (MINIMA) zero.of(d, Q4Stage<G>::pick(st[i].m, g));
                const uint32_t less[2] = {q4_less_bf16(zero.z[0]), q4_less_bf16(zero.z[1])};
                float c[4];
#pragma unroll
                for (int s = 0; s < 2 * SL; ++s) {
                    const int j = g * SL + s / 2, h = s % 2;
                    uint32_t av[4];
                    q4_bf16_words(av, u[0][j] >> (8 * h), u[1][j] >> (8 * h), less);
                    const uint2 b = *reinterpret_cast<const uint2*>(f + (2 * j + h) * 32);
                    if (s == 0) q4_mma<false, true>(c, av, b);
                    else q4_mma<false, false>(c, av, b);
                }
                // Lane (g, 0) holds columns 0 and 1, lane (g, 1) column 2, lane (g, 3) what the minima add.
                const int t = lane & 3;
                const float part[2] = {t == 0 ? c[0] + c[1] : t == 1 ? c[0] : 0.0f, t == 0 ? c[2] + c[3] : t == 1 ? c[2] : 0.0f};
                const float x = MINIMA && t == 3 ? sums[at * NG + g] : 0.0f;
                sum[0] = fmaf(d.x, part[0], fmaf(zero.o[0], x, sum[0]));
                sum[1] = fmaf(d.y, part[1], fmaf(zero.o[1], x, sum[1]));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(~0u, sum[r], 2);
                sum[r] += __shfl_xor_sync(~0u, sum[r], 1);
                const float2 v = q4_unpair(acc[i][r]);
                acc[i][r] = q4_pair(v.x, (lane & 3) == 3 ? fmaf(scale, sum[r], v.y) : v.y);
            }
        }
    }

    // One k-block, the chunk's at `at`.
    template <int G, bool MINIMA>
    __device__ __forceinline__ void product(const Q4Stage<G> (&st)[kTiles], int at) {
        constexpr int NG = 128 / G, SL = 4 / NG;  // slices of 32 a group
        const int lane = threadIdx.x & 31;
        const uint8_t* f = frags + at * kRow + lane * 8;
        const uint64_t magic = q4_pair(-12582912.0f, -12582912.0f);
        uint64_t part[kTiles][2];  // the k-block's sums, in its rows' scales
        uint32_t w[kTiles][2][4];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            w[i][0][0] = st[i].lo.x; w[i][0][1] = st[i].lo.y; w[i][0][2] = st[i].lo.z; w[i][0][3] = st[i].lo.w;
            w[i][1][0] = st[i].hi.x; w[i][1][1] = st[i].hi.y; w[i][1][2] = st[i].hi.z; w[i][1][3] = st[i].hi.w;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t av[kTiles][SL][4];
            uint64_t d0[kTiles], d1[kTiles];
            Q4Zero zero[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    const uint32_t u0 = w[i][0][g * SL + s], u1 = w[i][1][g * SL + s];
                    av[i][s][0] = u0 << 4 & 0xf0f0f0f0u;
                    av[i][s][1] = u1 << 4 & 0xf0f0f0f0u;
                    av[i][s][2] = u0 & 0xf0f0f0f0u;
                    av[i][s][3] = u1 & 0xf0f0f0f0u;
                }
                const float2 d = Q4Stage<G>::pick(st[i].d, g);
                d0[i] = q4_pair(d.x, d.x);
                d1[i] = q4_pair(d.y, d.y);
                if (MINIMA) zero[i].of(d, Q4Stage<G>::pick(st[i].m, g));
            }
            uint2 b[SL];
#pragma unroll
            for (int s = 0; s < SL; ++s) b[s] = *reinterpret_cast<const uint2*>(f + (g * SL + s) * kSlice);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                int c[4];
                if (MINIMA) {
                    const int2 x = column_sums[3 * (at * NG + g) + min(lane & 3, 2)];
                    const int k0 = 16 * (8 - static_cast<int>(zero[i].z[0])), k1 = 16 * (8 - static_cast<int>(zero[i].z[1]));
                    c[0] = k0 * x.x + 0x4b400000;
                    c[1] = k0 * x.y + 0x4b400000;
                    c[2] = k1 * x.x + 0x4b400000;
                    c[3] = k1 * x.y + 0x4b400000;
                    mma<false>(c, av[i][0], b[0]);
                    // o sum x, whole, in column 7's place.
                    const uint64_t v = q4_pair(0.0f, sums[at * NG + g]);
                    const bool mine = (lane & 3) == 3;
                    acc[i][0] = q4_fma2(q4_pair(0.0f, mine ? zero[i].o[0] : 0.0f), v, acc[i][0]);
                    acc[i][1] = q4_fma2(q4_pair(0.0f, mine ? zero[i].o[1] : 0.0f), v, acc[i][1]);
                } else {
                    mma<true>(c, av[i][0], b[0]);
                }
#pragma unroll
                for (int s = 1; s < SL; ++s) mma<false>(c, av[i][s], b[s]);
                const uint64_t v0 = q4_add2(q4_pair(__int_as_float(c[0]), __int_as_float(c[1])), magic);
                const uint64_t v1 = q4_add2(q4_pair(__int_as_float(c[2]), __int_as_float(c[3])), magic);
                part[i][0] = g == 0 ? q4_mul2(d0[i], v0) : q4_fma2(d0[i], v0, part[i][0]);
                part[i][1] = g == 0 ? q4_mul2(d1[i], v1) : q4_fma2(d1[i], v1, part[i][1]);
            }
        }
        const uint64_t v = *reinterpret_cast<const uint64_t*>(own + at * own_step);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            acc[i][0] = q4_fma2(v, part[i][0], acc[i][0]);
            acc[i][1] = q4_fma2(v, part[i][1], acc[i][1]);
        }
    }

    // The lane's sum of tile i: row lane / 4 (lane odd: + 8).
    __device__ __forceinline__ float lane_sum(int i, int) const {
        // The columns' weights: 2^-16, 2^-8, 1 of the first three, 2^-22 of these of the next; what is whole.
        const int t = threadIdx.x & 3;
        const float lower = q4_power(t == 0 ? -16 : t == 2 ? -30 : 0);
        const float upper = q4_power(t == 0 ? -8 : t == 1 ? -38 : t == 2 ? -22 : 0);
        float sum[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float2 v = q4_unpair(acc[i][r]);
            sum[r] = fmaf(v.x, lower, v.y * upper);
            sum[r] += __shfl_xor_sync(~0u, sum[r], 1);
            sum[r] += __shfl_xor_sync(~0u, sum[r], 2);
        }
        return t & 1 ? sum[1] : sum[0];
    }
    static __device__ __forceinline__ int row_of(int, int lane) { return (lane >> 2) + 8 * (lane & 1); }
    static __device__ __forceinline__ int token_of(int, int lane) { return lane >> 1 & 1; }  // lanes of a second are idle
};

// ---- a few FP32 rows: the three parts of two in each of NP products of eight columns

template <int NP, bool GATED_>
struct Q4Pairs {
    static constexpr bool GATED = GATED_;
    static constexpr int kTokens = 2 * NP;
    static constexpr int kTiles = GATED ? 2 : 1;
    static constexpr int kLaneSums = NP;
    static constexpr int kWarps = !GATED ? 16 : 8;
    static constexpr int kRun = 2, kRing = 3;   // k-blocks of a warp a round; rounds on their way
    static constexpr bool kFinisher = true, kWideRows = false;
    static constexpr int kColumn = 288;         // bytes: 8 slices x 32, and a step of 8 banks

    // Column 2 p + m of a product is part p of its row m.  Held are the rows' first parts, their second and their third
    // ones, of the rows that are there.
    static __host__ __device__ int block_bytes(int tokens, int ng) { return tokens * 3 * kColumn + kTokens * 4 * (1 + ng); }
    static constexpr int kTail = kColumn;  // what the lanes of a row that is not there read past the last
    uint8_t* frags;
    const uint8_t* column;  // the lane's, of the first product
    int part_bytes, x_bytes;
    float* scales;          // of a row's k-block
    float* sums;            // of a row's groups, in its scale
    __device__ __forceinline__ Q4Pairs(const Q4Args& a, uint8_t* x, int tokens, int) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        frags = x;
        part_bytes = tokens * kColumn;
        x_bytes = 3 * part_bytes;
        // The last two columns are the third parts again: their sums go nowhere.
        column = x + min(g >> 1, 2) * part_bytes + (g & 1) * kColumn + (lane & 3) * 8;
        scales = reinterpret_cast<float*>(x + a.chunk * x_bytes + kTail);
        sums = scales + a.chunk * kTokens;
    }

    template <int G, bool MINIMA, class Read>
    __device__ __forceinline__ bool split(const Q4Args& a, int m0, int tokens, int kb0, int kb1, Read read) const {
        constexpr int NG = 128 / G;
        const int lane = threadIdx.x & 31;
        const Q4Items it(kWarps, tokens);
        auto first = [&](int b, int m) { return frags + b * x_bytes + m * kColumn; };
        auto slot = [&](int b, int m) { return first(b, m) + (lane >> 4) * part_bytes + (lane & 15) * 16; };
        q4_fetch<false>(a, it, m0, tokens, kb0, kb1 - kb0, slot);
        read();
        asm volatile("cp.async.wait_all;" ::: "memory");
        q4_split<false>(a, it, tokens, kb1 - kb0, slot, [&](int b, int m, float4 x, bool store) {
            const uint32_t top = q4_top(x);
            if (store) q4_put_three(x, top, first(b, m), part_bytes);
            if (store && lane == 0) scales[b * kTokens + m] = q4_three_scale(top);
            if constexpr (MINIMA) {
                const float s = q4_group_sum<G>(x, q4_three_up(top));
                if (store && lane % (G / 4) == 0) sums[(b * NG + lane / (G / 4)) * kTokens + m] = s;
            }
        });
        return false;
    }

    float acc[kTiles][NP][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int t = 0; t < NP; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][t][c] = 0.0f;
    }

    template <int G, bool MINIMA>
    __device__ __forceinline__ void product(const Q4Stage<G> (&st)[kTiles], int at) {
        constexpr int NG = 128 / G, SL = 4 / NG;
        const int lane = threadIdx.x & 31;
        const uint8_t* f = column + at * x_bytes;
        float part[kTiles][NP][4];  // the k-block's sums, in its rows' scales
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float s[kTiles][NP][4];
            Q4Zero zero[kTiles];
            uint32_t less[kTiles][2];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                if (MINIMA) zero[i].of(Q4Stage<G>::pick(st[i].d, g), Q4Stage<G>::pick(st[i].m, g));
                less[i][0] = q4_less_bf16(zero[i].z[0]);
                less[i][1] = q4_less_bf16(zero[i].z[1]);
            }
#pragma unroll
            for (int j = g * SL; j < (g + 1) * SL; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t av[kTiles][4];
#pragma unroll
                    for (int i = 0; i < kTiles; ++i) {
                        const uint32_t u0 = j == 0 ? st[i].lo.x : j == 1 ? st[i].lo.y : j == 2 ? st[i].lo.z : st[i].lo.w;
                        const uint32_t u1 = j == 0 ? st[i].hi.x : j == 1 ? st[i].hi.y : j == 2 ? st[i].hi.z : st[i].hi.w;
                        q4_bf16_words(av[i], u0 >> (8 * h), u1 >> (8 * h), less[i]);
                    }
#pragma unroll
                    for (int t = 0; t < NP; ++t) {
                        const uint2 b = *reinterpret_cast<const uint2*>(f + (2 * j + h) * 32 + t * (2 * kColumn));
#pragma unroll
                        for (int i = 0; i < kTiles; ++i) {
                            if (j == g * SL && h == 0) q4_mma<false, true>(s[i][t], av[i], b);
                            else q4_mma<false, false>(s[i][t], av[i], b);
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const float2 d = Q4Stage<G>::pick(st[i].d, g);
#pragma unroll
                for (int t = 0; t < NP; ++t)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float scale = c & 2 ? d.y : d.x;
                        part[i][t][c] = g == 0 ? scale * s[i][t][c] : fmaf(scale, s[i][t][c], part[i][t][c]);
                    }
            }
            if (MINIMA) {
                // o sum x, in one of the lanes whose sums meet.
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const float o0 = lane & 3 ? 0.0f : zero[i].o[0], o1 = lane & 3 ? 0.0f : zero[i].o[1];
#pragma unroll
                    for (int t = 0; t < NP; ++t) {
                        const float2 v = *reinterpret_cast<const float2*>(sums + (at * NG + g) * kTokens + 2 * t);
                        part[i][t][0] = fmaf(o0, v.x, part[i][t][0]);
                        part[i][t][1] = fmaf(o0, v.y, part[i][t][1]);
                        part[i][t][2] = fmaf(o1, v.x, part[i][t][2]);
                        part[i][t][3] = fmaf(o1, v.y, part[i][t][3]);
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const float2 v = *reinterpret_cast<const float2*>(scales + at * kTokens + 2 * t);
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][t][c] = fmaf(c & 1 ? v.y : v.x, part[i][t][c], acc[i][t][c]);
        }
    }
    // The lane's sum c of tile i: row lane / 4 (lane odd: + 8) of row 2 c + (lane / 2) % 2 of x, over its parts' lanes.
    __device__ __forceinline__ float lane_sum(int i, int c) const {
        const int lane = threadIdx.x & 31;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = (lane & 3) == 3 ? 0.0f : acc[i][c][k];
            v[k] += __shfl_xor_sync(~0u, v[k], 2);
            v[k] += __shfl_xor_sync(~0u, v[k], 1);
        }
        return lane & 2 ? (lane & 1 ? v[3] : v[1]) : (lane & 1 ? v[2] : v[0]);
    }
    static __device__ __forceinline__ int row_of(int, int lane) { return (lane >> 2) + 8 * (lane & 1); }
    static __device__ __forceinline__ int token_of(int c, int lane) { return 2 * c + (lane >> 1 & 1); }
};

// ---- x as floating-point columns: T products of eight rows of x, HALF: FP16 rows as they are

template <int T, bool HALF, bool GATED_>
struct Q4Floats {
    static constexpr bool GATED = GATED_;
    static constexpr int kTokens = 8 * T;
    static constexpr int kTiles = GATED ? 2 : 1;
    static constexpr int kLaneSums = 4 * T;
    static constexpr int kParts = HALF ? 1 : 3;  // columns of a row
    static constexpr int kProducts = kParts * T;
    static constexpr int kWarps = T <= 2 && !GATED ? 16 : 8;
    static constexpr int kRun = T == 1 && HALF ? 2 : 1, kRing = kRun == 2 || GATED ? 3 : 4;
    static constexpr bool kFinisher = false, kWideRows = false;

    static constexpr int kColumn = 288;  // bytes: 8 slices x 32, and a step of 8 banks

    // The columns: the eight rows' first parts of a product, their second ones, their third ones, then the next
    // eight rows'.  Of a single product's rows only those that are there.
    static __host__ __device__ int columns(int tokens) { return T == 1 ? kParts * tokens : 8 * kProducts; }
    static __host__ __device__ int block_bytes(int tokens, int ng) {
        return columns(tokens) * kColumn + kTokens * 4 * (1 + ng);
    }
    static constexpr int kTail = T == 1 ? 8 * kColumn : 0;  // what the lanes of rows that are not there read past the last
    uint8_t* frags;
    int part_bytes, x_bytes;  // from a part to the next, of a k-block
    float* scales;            // of a row's k-block
    float* sums;              // of a row's groups, in its scale
    __device__ __forceinline__ Q4Floats(const Q4Args& a, uint8_t* x, int tokens, int) {
        frags = x;
        part_bytes = (T == 1 ? tokens : 8) * kColumn;
        x_bytes = columns(tokens) * kColumn;
        scales = reinterpret_cast<float*>(x + a.chunk * x_bytes + kTail);
        sums = scales + a.chunk * kTokens;
    }

    template <int G, bool MINIMA, class Read>
    __device__ __forceinline__ bool split(const Q4Args& a, int m0, int tokens, int kb0, int kb1, Read read) const {
        constexpr int NG = 128 / G;
        const int lane = threadIdx.x & 31;
        const Q4Items it(kWarps, tokens);
        auto column = [&](int b, int m) {
            return frags + b * x_bytes + (T == 1 ? m : m / 8 * (8 * kParts) + m % 8) * kColumn;
        };
        auto slot = [&](int b, int m) {
            return HALF ? column(b, m) + lane * 8 : column(b, m) + (lane >> 4) * part_bytes + (lane & 15) * 16;
        };
        q4_fetch<HALF>(a, it, m0, tokens, kb0, kb1 - kb0, slot);
        read();
        asm volatile("cp.async.wait_all;" ::: "memory");
        q4_split<HALF>(a, it, tokens, kb1 - kb0, slot, [&](int b, int m, float4 x, bool store) {
            uint8_t* to = column(b, m);
            float up = 1.0f;
            if constexpr (HALF) {
                to += q4_float_word(lane);
                if (store) {
                    *reinterpret_cast<__half2*>(to) = __floats2half2_rn(x.x, x.z);
                    *reinterpret_cast<__half2*>(to + 32) = __floats2half2_rn(x.y, x.w);
                }
            } else {
                const uint32_t top = q4_top(x);
                up = q4_three_up(top);
                if (store) q4_put_three(x, top, to, part_bytes);
                if (store && lane == 0) scales[b * kTokens + m] = q4_three_scale(top);
            }
            if constexpr (MINIMA) {
                const float s = q4_group_sum<G>(x, up);
                if (store && lane % (G / 4) == 0) sums[(b * NG + lane / (G / 4)) * kTokens + m] = s;
            }
        });
        return false;
    }

    float acc[kTiles][kLaneSums];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int c = 0; c < kLaneSums; ++c) acc[i][c] = 0.0f;
    }

    template <int G, bool MINIMA>
    __device__ __forceinline__ void product(const Q4Stage<G> (&st)[kTiles], int at) {
        constexpr int NG = 128 / G;
        const int lane = threadIdx.x & 31;
        const uint8_t* f = frags + at * x_bytes + (lane >> 2) * kColumn + (lane & 3) * 8;
        constexpr int kSums = HALF ? 1 : 2;  // the first parts', and the others', which are far smaller
        float part[kTiles][kLaneSums];       // the k-block's sums, in its rows' scales
        float s[kTiles][T][kSums][4];        // a group's sums
        Q4Zero zero[kTiles];
        uint32_t less[kTiles][2], less_high[kTiles][2];
        uint32_t w[kTiles][2][4];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            w[i][0][0] = st[i].lo.x; w[i][0][1] = st[i].lo.y; w[i][0][2] = st[i].lo.z; w[i][0][3] = st[i].lo.w;
            w[i][1][0] = st[i].hi.x; w[i][1][1] = st[i].hi.y; w[i][1][2] = st[i].hi.z; w[i][1][3] = st[i].hi.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j % (4 / NG) == 0 && (j == 0 || MINIMA)) {
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const int g = j / (4 / NG);
                    if (MINIMA) zero[i].of(Q4Stage<G>::pick(st[i].d, g), Q4Stage<G>::pick(st[i].m, g));
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        less[i][r] = HALF ? q4_less_low(zero[i].z[r]) : q4_less_bf16(zero[i].z[r]);
                        if (HALF) less_high[i][r] = q4_less_high(zero[i].z[r]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t av[kTiles][4];
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const uint32_t u0 = w[i][0][j] >> (8 * h), u1 = w[i][1][j] >> (8 * h);
                    if constexpr (HALF) {
                        av[i][0] = q4_low(u0, less[i][0]);
                        av[i][1] = q4_low(u1, less[i][1]);
                        av[i][2] = q4_high(u0, less_high[i][0]);
                        av[i][3] = q4_high(u1, less_high[i][1]);
                    } else {
                        q4_bf16_words(av[i], u0, u1, less[i]);
                    }
                }
                const bool first = j % (4 / NG) == 0 && h == 0;
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        const uint2 b = *reinterpret_cast<const uint2*>(f + (2 * j + h) * 32 + t * (8 * kParts * kColumn) +
                                                                        p * (T == 1 ? part_bytes : 8 * kColumn));
#pragma unroll
                        for (int i = 0; i < kTiles; ++i) {
                            if (first && p < kSums) q4_mma<HALF, true>(s[i][t][p], av[i], b);
                            else q4_mma<HALF, false>(s[i][t][p == 0 ? 0 : kSums - 1], av[i], b);
                        }
                    }
                }
            }
            if ((j + 1) % (4 / NG) != 0) continue;
            const int g = (j + 1) / (4 / NG) - 1;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const float2 d = Q4Stage<G>::pick(st[i].d, g);
#pragma unroll
                for (int c = 0; c < kLaneSums; ++c) {
                    const float scale = c & 2 ? d.y : d.x;
                    const float v = HALF ? s[i][c / 4][0][c % 4] : s[i][c / 4][0][c % 4] + s[i][c / 4][kSums - 1][c % 4];
                    part[i][c] = g == 0 ? scale * v : fmaf(scale, v, part[i][c]);
                }
            }
            if (MINIMA) {
                const float* xs = sums + (at * NG + g) * kTokens + (lane & 3) * 2;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const float o0 = zero[i].o[0], o1 = zero[i].o[1];
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        const float2 v = *reinterpret_cast<const float2*>(xs + t * 8);
                        part[i][4 * t] = fmaf(o0, v.x, part[i][4 * t]);
                        part[i][4 * t + 1] = fmaf(o0, v.y, part[i][4 * t + 1]);
                        part[i][4 * t + 2] = fmaf(o1, v.x, part[i][4 * t + 2]);
                        part[i][4 * t + 3] = fmaf(o1, v.y, part[i][4 * t + 3]);
                    }
                }
            }
        }
        const float* xs = scales + at * kTokens + (lane & 3) * 2;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float2 v = HALF ? make_float2(1.0f, 1.0f) : *reinterpret_cast<const float2*>(xs + t * 8);
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    acc[i][4 * t + c] = fmaf(c & 1 ? v.y : v.x, part[i][4 * t + c], acc[i][4 * t + c]);
        }
    }
    __device__ __forceinline__ float lane_sum(int i, int c) const { return acc[i][c]; }
    static __device__ __forceinline__ int row_of(int c, int lane) { return (lane >> 2) + 4 * (c & 2); }
    static __device__ __forceinline__ int token_of(int c, int lane) { return c / 4 * 8 + (lane & 3) * 2 + (c & 1); }
};

// ---- the kernel

// One output element: the chain, the gate, the store.
__device__ __forceinline__ void q4_finish(const Q4Args& a, int m, long long n, float v, float g, bool gated) {
    const Q4Row row(a, m);
    const long long at = row.at(a.ynb) + n;
    if (a.chain.from_redirect) v += static_cast<const float*>(a.y)[at];
    v = apply_chain(a.chain, v, n, row.i1, row.i2, row.i3);
    if (gated) {
        g = apply_chain(a.chain, g, a.n + n, row.i1, row.i2, row.i3);
        v *= a.act == SDB_GATE_SILU ? silu(g) : gelu(g);
    }
    if (a.y_half) static_cast<__half*>(a.y)[at] = __float2half_rn(v);
    else static_cast<float*>(a.y)[at] = v;
}

// The warps' sums: two buffers where they are small.
template <class F>
constexpr int q4_red_floats() { return F::kWarps * F::kTiles * F::kLaneSums * 32; }
template <class F>
constexpr int q4_red_buffers() { return F::kLaneSums <= 4 ? 2 : 1; }

template <class F>
constexpr int q4_threads() { return 32 * (F::kWarps + 1 + (F::kFinisher ? 1 : 0)); }

// Shared memory but for the k-blocks of x; `block` the bytes of a tile.
template <class F>
int q4_fixed_bytes(int block) {
    return q4_red_buffers<F>() * q4_red_floats<F>() * 4 + F::kRing * (F::kWarps * F::kTiles * F::kRun * block + 16) + 16 +
           F::kTail;
}

// MINIMA: compiled for itself, so that the products of two k-blocks lie side by side without a branch between (one
// row of 8192 -> 28672 without a minimum 27.6 us, with the choice made in the loop 31.8).
template <class F, int G, bool MINIMA>
__global__ void __launch_bounds__(q4_threads<F>(), 1) q4_rows_kernel(const __grid_constant__ Q4Args a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const bool worker = warp < F::kWarps, bringer = warp == F::kWarps;
    const int WK = 1 << a.wk_log, wk = warp & (WK - 1), wr = warp >> a.wk_log, round_blocks = F::kRun << a.wk_log;
    const int cluster = 1 << a.cluster_log, rank = blockIdx.x & (cluster - 1);
    const int groups = a.groups, group0 = blockIdx.x >> a.cluster_log, group_step = gridDim.x >> a.cluster_log;
    const int kb_begin = rank * a.range, kb_end = min(kb_begin + a.range, a.kblocks);
    const int m0 = blockIdx.y * F::kTokens, tokens = min(F::kTokens, a.rows - m0);
    constexpr int block = 1024 + 4096 / G * (MINIMA ? 2 : 1);  // bytes of a tile
    constexpr int place_bytes = F::kWarps * F::kTiles * F::kRun * block;

    float* red = reinterpret_cast<float*>(smem);
    uint8_t* ring = reinterpret_cast<uint8_t*>(red + q4_red_buffers<F>() * q4_red_floats<F>());
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + F::kRing * place_bytes);
    uint64_t* empty = full + F::kRing;
    volatile int* abort = reinterpret_cast<volatile int*>(empty + F::kRing);
    F form(a, reinterpret_cast<uint8_t*>(empty + F::kRing) + 16, tokens, MINIMA ? 128 / G : 0);

    // The rounds in order: over the row tiles, the chunks of x and their k-blocks.
    int next_group = group0, next_kc = kb_begin, next_kb = kb_begin, brought = 0;
    auto bring = [&](int place) {  // the bringer's warp: the next round
        if (next_group >= groups) return;
        const int kc_end = min(next_kc + a.chunk, kb_end), count = min(round_blocks, kc_end - next_kb);
        if (lane == 0) mbar_arrive_expect_tx(full + place, (F::kTiles << a.wr_log) * count * block);
        __syncwarp();
        if (lane < F::kTiles << a.wr_log) {
            const int tile = min((next_group << a.wr_log) + (lane & ((1 << a.wr_log) - 1)), a.tiles - 1);
            const uint8_t* from = F::GATED && lane >> a.wr_log ? a.gate : a.w;
            bulk_load(ring + place * place_bytes + lane * (round_blocks * block),
                      from + (static_cast<long long>(tile) * a.kblocks + next_kb) * block, count * block, full + place);
        }
        ++brought;
        next_kb += count;
        if (next_kb == kc_end) {
            next_kc = kc_end;
            if (kc_end == kb_end) {
                next_kc = kb_begin;
                next_group += group_step;
            }
            next_kb = next_kc;
        }
    };
    if (bringer) {
        if (lane == 0) {
            *abort = 0;
            for (int i = 0; i < F::kRing; ++i) {
                mbar_init(full + i, 1);
                mbar_init(empty + i, F::kWarps);
            }
            fence_barrier_init();
        }
        __syncwarp();
        if (kb_begin < kb_end) {
            // After the working warps' first reads of x, which would else queue behind all of this.
            asm volatile("bar.sync 1, %0;" ::"n"(32 * (F::kWarps + 1)) : "memory");
#pragma unroll 1
            for (int i = 0; i < F::kRing; ++i) bring(i);
        }
    }

    bool started = false, held = false;  // a chunk of x, the only one, is in shared memory
    bool lost = false;                   // a bounded wait ran out
    bool wide = false;                   // the chunk has rows that are not digits
    int parity = 0, place = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (int group = group0; group < groups; group += group_step) {
        form.clear();
#pragma unroll 1
        for (int kc = kb_begin; kc < kb_end; kc += a.chunk) {
            const int kc_end = min(kc + a.chunk, kb_end);
            if (!held) {
                if (started) __syncthreads();  // the chunk before has been read
                if (worker)
                    wide = form.template split<G, MINIMA>(a, m0, tokens, kc, kc_end, [&] {
                        if (!started) asm volatile("bar.arrive 1, %0;" ::"n"(32 * (F::kWarps + 1)) : "memory");
                    });
                started = true;
                if constexpr (F::kWideRows) wide = __syncthreads_or(wide);
                else __syncthreads();
                held = a.chunk >= kb_end - kb_begin;
            }
            if (!worker && !bringer) continue;
#pragma unroll 1
            for (int kb = kc; kb < kc_end && !lost; kb += round_blocks) {
                // A wait that runs out ends the rounds for this warp and, by the abort flag, for the others; the
                // barriers are still met.
                lost = __any_sync(~0u, !mbar_wait((bringer ? empty : full) + place, phase, abort, a.err));
                if (lost) break;
                if (bringer) {
                    bring(place);
                } else {
                    const int at = kb - kc + wk * F::kRun;
                    const uint8_t* tiles = ring + place * place_bytes + warp * (F::kRun * block);
                    const int count = min(kc_end - kc - at, F::kRun);  // less than 1: none
                    auto staged = [&](int i, auto then) {
                        Q4Stage<G> stage[F::kTiles];
#pragma unroll
                        for (int t = 0; t < F::kTiles; ++t)
                            stage[t].read(tiles + t * (F::kWarps * F::kRun * block) + i * block, lane, MINIMA);
                        then(stage, at + i);
                    };
                    auto one = [&](int i) {
                        staged(i, [&](auto& stage, int k) { form.template product<G, MINIMA>(stage, k); });
                    };
                    bool apart = false;  // each k-block by itself
                    if constexpr (F::kWideRows) {
                        apart = wide;
#pragma unroll 1
                        for (int i = 0; apart && i < count; ++i) {
                            if (!form.wide(at + i)) one(i);
                            else staged(i, [&](auto& stage, int k) { form.template wide_product<G, MINIMA>(stage, k); });
                        }
                    }
                    if (!apart && F::kRun == 2 && count == 2) {  // two k-blocks' chains of products side by side
                        one(0);
                        one(1);
                    } else if (!apart && count > 0) {
                        one(0);
                    }
                    __syncwarp();  // every lane has read its part
                    if (lane == 0) mbar_arrive(empty + place);
                }
                if (++place == F::kRing) {
                    place = 0;
                    phase ^= 1;
                }
            }
        }

        // The warps' sums: [sum][tile][warp][lane].  Of two buffers, the one written next has been read by
        // every thread before the barrier in between.
        float* mine = red + parity * q4_red_floats<F>();
        if constexpr (q4_red_buffers<F>() == 2) parity ^= 1;
        if (worker) {
#pragma unroll
            for (int c = 0; c < F::kLaneSums; ++c)
#pragma unroll
                for (int i = 0; i < F::kTiles; ++i)
                    mine[((c * F::kTiles + i) * F::kWarps + warp) * 32 + lane] = form.lane_sum(i, c);
        }
        if (cluster > 1) cooperative_groups::this_cluster().sync();
        else __syncthreads();
        // A warp finishes a sum of a tile: the working warps, or the one that does nothing else.  A cluster's CTAs
        // share the sums.
        const int items = F::kLaneSums << a.wr_log, item_step = F::kFinisher ? 1 : F::kWarps;
        const int item0 = F::kFinisher ? (worker || bringer ? items : 0) : worker ? warp : items;
#pragma unroll 1
        for (int o = (item0 << a.cluster_log) + rank; o < items; o += item_step << a.cluster_log) {
            const int c = o >> a.wr_log, tw = o - (c << a.wr_log);
            const int m = F::token_of(c, lane);
            const long long n = ((static_cast<long long>(group) << a.wr_log) + tw) * 16 + F::row_of(c, lane);
            if (m >= tokens || n >= a.n) continue;
            float v[2] = {0.0f, 0.0f};
            const int at = (c * F::kTiles * F::kWarps + tw * WK) * 32 + lane;
            auto join = [&](const float* from) {
#pragma unroll 4
                for (int j = 0; j < WK; ++j) {
#pragma unroll
                    for (int i = 0; i < F::kTiles; ++i) v[i] += from[at + (i * F::kWarps + j) * 32];
                }
            };
            if (cluster > 1) {
#pragma unroll 4
                for (int k = 0; k < cluster; ++k) join(cooperative_groups::this_cluster().map_shared_rank(mine, k));
            } else {
                join(mine);
            }
            q4_finish(a, m0 + m, n, v[0], v[1], F::GATED);
        }
        if constexpr (q4_red_buffers<F>() == 1) {
            if (cluster > 1) cooperative_groups::this_cluster().sync();
            else __syncthreads();
        }
    }
    if (bringer && lost)  // copies may still be on their way into this CTA's memory: wait for them, with a limit
        for (int i = max(0, brought - F::kRing); i < brought; ++i)
            mbar_wait_quiet(full + i % F::kRing, i / F::kRing & 1, kWaitLimitNs);
    if (cluster > 1) cooperative_groups::this_cluster().sync();  // the others have read this CTA's sums
}

// How a product is cut (q4_linear.cu).
struct Q4Plan {
    int form;      // rows of x a CTA takes: 1 in digits; 2 or 4 in pairs; 8, 16, or 32 of FP16, in floats
    int wk_log;    // warps that share a row tile's k-blocks (fewer where their k-blocks of x do not fit)
    int cluster_log;  // CTAs that do
    int shared;    // bytes of shared memory a CTA may take
};

// Launches the kernel for rows in FP16 or FP32, plain or gated, groups of G with MINIMA or without.
template <int G, bool MINIMA>
int q4_launch(const Q4Args& a, const Q4Plan& p, cudaStream_t st);

}  // namespace sdb
