// The kernel of the linear layers of a few rows with 4-bit weights (q4.cuh).
//
//   y[m][n] = sum_g d[n][g] S + (min[n][g] + 8 d[n][g]) sum_{k in g} x[m][k],
//   S = sum_{k in g} (q[n][k] - 8) x[m][k]
//
// The weights' bytes are the work: each is read once for up to 32 rows of x.
// The 16 weight rows of a tile are the M of mma.m16n8k16 and the rows of x its
// N, so that one instruction turns 8 bytes a lane into sums for 8 columns; S
// is summed over one group by the tensor core, from zero, and joins the FP32
// sum with the group's scale.  q - 8 is exact in FP16 (0x6400 | q is 1024 + q;
// a subtraction, or for a nibble four bits up a multiply-add, leaves q - 8).
//
// FP32 rows of x are made FP16 pairs: a row's 128 numbers of a k-block are
// scaled by a power of two that brings the greatest just under 2^15, x = hi + lo
// with both FP16 -- off by 2^-24 of x at most, or 2^-40 of the k-block's
// greatest number -- and the sum over the k-block is scaled back.  So the
// products see x whole at any magnitude.  With up to four rows hi and lo are
// two columns of one product (PAIRED), else two products.  FP16 rows are taken
// as they are.
//
// A CTA is eight warps: WR tiles of rows side by side, WK = 8 / WR warps to a
// tile that share its k-blocks, and up to eight CTAs of a cluster that share
// them again.  x is split once into shared memory, each column of the products
// a run of its eight k-slices' fragments (4 lanes of 8 bytes a slice) and 288
// bytes to the next column, so that neither a column's stores nor a slice's
// loads over eight columns meet a bank twice, and stays there for all the row
// tiles the CTA walks.  A product's unused columns are not stored: their lanes
// read what lies there and their sums go nowhere.  Weights go from memory to
// registers, two k-blocks ahead.  The warps' sums meet in shared memory and are added in one order, so
// a result does not turn on timing; the sums of a cluster's other CTAs are read
// where they lie.
#pragma once

#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "chain.cuh"
#include "q4.cuh"

namespace sdb {

constexpr int kQ4Warps = 8;
constexpr int kQ4Threads = 32 * kQ4Warps;
constexpr int kQ4MaxShared = 227 * 1024;
constexpr int kQ4Column = 288;  // bytes of a column's k-block in shared memory: 8 slices x 32, and a step of 8 banks

struct Q4Args {
    Q4View w, gate;            // gate: the gated form's second matrix
    const void* x;
    void* y;
    long long xnb[3], ynb[3];  // strides of rows in elements (dims 1..3)
    int ne1, ne2;
    int rows;                  // of x
    int x_vec;                 // x's runs of four numbers are aligned
    int y_half;                // FP16 output
    int act;                   // SDB_GATE_*
    int wk_log;                // WK = 1 << wk_log
    int cluster;               // CTAs that share a tile's k-blocks
    int range;                 // k-blocks of a CTA (the last of a cluster may have fewer)
    int chunk;                 // k-blocks of x held at a time, a multiple of WK
    Chain chain;
};

// What a variant's shared memory holds.
template <int T, bool PAIRED, bool HALF, bool GATED>
struct Q4Shape {
    static constexpr int kTokens = PAIRED ? 4 : 8 * T;            // rows of x of a CTA
    static constexpr int kProducts = HALF || PAIRED ? T : 2 * T;  // products of a k-slice
    static constexpr int kTiles = GATED ? 2 : 1;
    static constexpr int kSums = PAIRED ? 2 : 4 * T;              // FP32 sums a lane has of a tile
    static constexpr int kRedBuffers = T == 1 ? 2 : 1;
    static constexpr int kRedFloats = kQ4Warps * kTiles * kSums * 32;
    // Bytes of x a k-block with `tokens` rows: the columns of the products, the rows' scales and their sums
    // over its groups; and after all k-blocks, what the lanes of unused columns read past the last.
    static __host__ __device__ constexpr int columns(int tokens) { return PAIRED ? 2 * tokens : 8 * kProducts; }
    static constexpr int block_bytes(int tokens, int ng) { return kQ4Column * columns(tokens) + kTokens * 4 * (1 + ng); }
    static constexpr int fixed_bytes() { return kRedBuffers * kRedFloats * 4 + kTokens * 8 + 8 * kQ4Column; }
};

// c = a b, or c += a b.
template <bool FIRST>
__device__ __forceinline__ void q4_mma(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
    if constexpr (FIRST)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(0.0f));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

// u & mask | 0x64006400: two nibbles in the low bits of FP16 numbers from 1024 on.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t q4_nibbles(uint32_t u) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(u), "n"(MASK), "r"(0x64006400u));
    return v;
}

__device__ __forceinline__ uint32_t q4_low(uint32_t u) {  // nibbles at bits 0 and 16: 1024 + q, less 1032
    uint32_t v;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(v) : "r"(q4_nibbles<0x000f000fu>(u)), "r"(0x64086408u));
    return v;
}

__device__ __forceinline__ uint32_t q4_high(uint32_t u) {  // at bits 4 and 20: (1024 + 16 q) / 16, less 72
    uint32_t v;
    asm("fma.rn.f16x2 %0, %1, %2, %3;"
        : "=r"(v)
        : "r"(q4_nibbles<0x00f000f0u>(u)), "r"(0x2c002c00u), "r"(0xd480d480u));
    return v;
}

// Weights pass through: not kept in L1, kept in L2 as any line (a next call may find them there).
__device__ __forceinline__ uint4 q4_load(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 q4_load(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ unsigned q4_load(const unsigned* p) {
    unsigned v;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// A k-block of a row tile as a lane holds it: the words of rows g and g + 8, the scales, the minima.
template <int G>
struct Q4Stage {
    static constexpr int kNg = 128 / G;
    uint4 lo, hi;
    uint32_t d[kNg], m[kNg];

    static __device__ __forceinline__ void load_run(uint32_t (&r)[kNg], const uint8_t* p) {
        if constexpr (kNg == 4) {
            const uint4 v = q4_load(reinterpret_cast<const uint4*>(p));
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
        } else if constexpr (kNg == 2) {
            const uint2 v = q4_load(reinterpret_cast<const uint2*>(p));
            r[0] = v.x; r[1] = v.y;
        } else {
            r[0] = q4_load(reinterpret_cast<const unsigned*>(p));
        }
    }
    // Group i's numbers of rows g and g + 8.
    static __device__ __forceinline__ float2 pick(const uint32_t (&r)[kNg], int i) {
        if constexpr (kNg == 1) return __half22float2(*reinterpret_cast<const __half2*>(&r[0]));
        const __half2 a = *reinterpret_cast<const __half2*>(&r[i / 2]);
        const __half2 b = *reinterpret_cast<const __half2*>(&r[kNg / 2 + i / 2]);
        return i & 1 ? make_float2(__high2float(a), __high2float(b)) : make_float2(__low2float(a), __low2float(b));
    }
};

// Where a lane's next k-block of a matrix lies; steps are counted in k-blocks.
template <int G>
struct Q4Walk {
    const uint8_t *codes, *scales, *minima;
    __device__ __forceinline__ void start(const Q4View& w, long long block, int lane) {
        codes = w.codes + block * 1024 + lane * 16;
        scales = reinterpret_cast<const uint8_t*>(w.scales) + (block * 8 + lane / 4) * (512 / G);
        minima = w.minima ? reinterpret_cast<const uint8_t*>(w.minima) + (block * 8 + lane / 4) * (512 / G) : nullptr;
    }
    __device__ __forceinline__ void step(long long blocks) {
        codes += blocks * 1024;
        scales += blocks * (4096 / G);
        if (minima) minima += blocks * (4096 / G);
    }
    __device__ __forceinline__ void load(Q4Stage<G>& s) const {
        s.lo = q4_load(reinterpret_cast<const uint4*>(codes));
        s.hi = q4_load(reinterpret_cast<const uint4*>(codes) + 32);
        Q4Stage<G>::load_run(s.d, scales);
        if (minima) Q4Stage<G>::load_run(s.m, minima);
    }
};

// Splits the CTA's rows of x for k-blocks [kb0, kb1) into shared memory: a warp takes a row's k-block, a
// lane four numbers (columns 4 lane..): slice 2 (lane / 8) + lane % 2, and there lane / 2 % 4 of the column.
template <int T, bool PAIRED, bool HALF, int G>
__device__ __forceinline__ void q4_split(const Q4Args& a, const long long* row_at, int tokens, int kb0, int kb1,
                                         uint8_t* frags, float* scales, float* sums) {
    using S = Q4Shape<T, PAIRED, HALF, false>;
    constexpr int NG = 128 / G;
    const int lane = threadIdx.x & 31;
    const int slice = (lane >> 3) * 2 + (lane & 1), t = (lane >> 1) & 3;
    const int items = tokens * (kb1 - kb0), block = kQ4Column * S::columns(tokens);
    for (int i = threadIdx.x / 32; i < items; i += kQ4Warps) {
        const int b = i / tokens, m = i - b * tokens;
        const long long k = (kb0 + b) * 128LL + lane * 4;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint2 raw = make_uint2(0, 0);
        if constexpr (HALF) {
            const __half* p = static_cast<const __half*>(a.x) + row_at[m] + k;
            if (a.x_vec && k + 4 <= a.w.k) {
                raw = __ldg(reinterpret_cast<const uint2*>(p));
            } else {
                unsigned short h[4];
                for (int c = 0; c < 4; ++c) h[c] = k + c < a.w.k ? __half_as_ushort(p[c]) : 0;
                raw.x = h[0] | static_cast<uint32_t>(h[1]) << 16;
                raw.y = h[2] | static_cast<uint32_t>(h[3]) << 16;
            }
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
            x[0] = f0.x; x[1] = f0.y; x[2] = f1.x; x[3] = f1.y;
        } else {
            const float* p = static_cast<const float*>(a.x) + row_at[m] + k;
            if (a.x_vec && k + 4 <= a.w.k) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(p));
                x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
            } else {
                for (int c = 0; c < 4; ++c) x[c] = k + c < a.w.k ? p[c] : 0.0f;
            }
        }
        uint8_t* base = frags + b * block + slice * 32 + t * 8;
        auto slot = [&](int col) { return reinterpret_cast<uint2*>(base + col * kQ4Column); };
        if constexpr (HALF) {
            *slot(m) = raw;
        } else {
            float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            // top < 2^(e - 126), e its exponent field: scaled by 2^(141 - e) it is below 2^15.  The field of
            // that power is 268 - e, kept a normal number's; infinities (and NaN, which fmaxf passes over)
            // stay what they are.
            const int e = static_cast<int>(__float_as_uint(top) >> 23);
            const int f = min(268 - e, 253);
            const float up = __uint_as_float(static_cast<uint32_t>(f) << 23);
            const float down = __uint_as_float(static_cast<uint32_t>(254 - f) << 23);
            uint2 hi, lo;
            for (int c = 0; c < 4; c += 2) {
                const float u = x[c] * up, v = x[c + 1] * up;
                const __half2 h = __floats2half2_rn(u, v);
                const float2 r = __half22float2(h);
                const __half2 l = __floats2half2_rn(u - r.x, v - r.y);
                (c ? hi.y : hi.x) = *reinterpret_cast<const uint32_t*>(&h);
                (c ? lo.y : lo.x) = *reinterpret_cast<const uint32_t*>(&l);
            }
            if constexpr (PAIRED) {
                *slot(2 * m) = hi;
                *slot(2 * m + 1) = lo;
            } else {
                *slot(m / 8 * 16 + m % 8) = hi;
                *slot(m / 8 * 16 + m % 8 + 8) = lo;
            }
            if (lane == 0) scales[b * S::kTokens + m] = down;
        }
        if (a.w.minima) {
            float s = (x[0] + x[1]) + (x[2] + x[3]);
            for (int o = 1; o < G / 4; o <<= 1) s += __shfl_xor_sync(~0u, s, o);
            if (lane % (G / 4) == 0) sums[(b * NG + lane / (G / 4)) * S::kTokens + m] = s;
        }
    }
}

// One output element: the chain, the gate, the store.
__device__ __forceinline__ void q4_finish(const Q4Args& a, int m, long long n, float v, float g, bool gated) {
    const int q = m / a.ne1, i1 = m - q * a.ne1, i3 = q / a.ne2, i2 = q - i3 * a.ne2;
    const long long at = n + i1 * a.ynb[0] + i2 * a.ynb[1] + i3 * a.ynb[2];
    if (a.chain.from_redirect) v += static_cast<const float*>(a.y)[at];
    v = apply_chain(a.chain, v, n, i1, i2, i3);
    if (gated) {
        g = apply_chain(a.chain, g, a.w.n + n, i1, i2, i3);
        v *= a.act == SDB_GATE_SILU ? silu(g) : gelu(g);
    }
    if (a.y_half) static_cast<__half*>(a.y)[at] = __float2half_rn(v);
    else static_cast<float*>(a.y)[at] = v;
}

template <int T, bool PAIRED, bool HALF, bool GATED, int G>
__global__ void __launch_bounds__(kQ4Threads, T == 1 ? 2 : 1) q4_rows_kernel(const __grid_constant__ Q4Args a) {
    using S = Q4Shape<T, PAIRED, HALF, GATED>;
    constexpr int NG = 128 / G;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int wk = warp & ((1 << a.wk_log) - 1), wr = warp >> a.wk_log, WK = 1 << a.wk_log, WR = kQ4Warps >> a.wk_log;
    const int rank = blockIdx.x % a.cluster;
    const int groups = (a.w.tiles + WR - 1) / WR;                  // of WR row tiles
    const int group0 = blockIdx.x / a.cluster, group_step = gridDim.x / a.cluster;
    const int m0 = blockIdx.y * S::kTokens, tokens = min(S::kTokens, a.rows - m0);
    const int kb_begin = rank * a.range, kb_end = min(kb_begin + a.range, a.w.kblocks);

    float* red = reinterpret_cast<float*>(smem);
    long long* row_at = reinterpret_cast<long long*>(red + S::kRedBuffers * S::kRedFloats);
    uint8_t* frags = reinterpret_cast<uint8_t*>(row_at + S::kTokens);
    const int block_bytes = kQ4Column * S::columns(tokens);
    float* scales = reinterpret_cast<float*>(frags + a.chunk * block_bytes + 8 * kQ4Column);
    float* sums = scales + a.chunk * S::kTokens;

    // The warp's k-blocks in the order they are taken: over its row tiles, kb_begin + wk, + WK, ...  A warp
    // past the last tile walks the last one again and stores nothing.
    Q4Stage<G> stage[2][S::kTiles];
    Q4Walk<G> walk[S::kTiles];
    const int steps = kb_end - kb_begin > wk ? (kb_end - kb_begin - wk + WK - 1) >> a.wk_log : 0;  // of a tile
    int load_group = group0, load_step = 0;
    auto tile_of = [&](int group) { return min(group * WR + wr, a.w.tiles - 1); };
    {
        const long long block = static_cast<long long>(tile_of(group0)) * a.w.kblocks + kb_begin + wk;
        walk[0].start(a.w, block, lane);
        if constexpr (GATED) walk[1].start(a.gate, block, lane);
    }
    auto load = [&](Q4Stage<G> (&to)[S::kTiles]) {
        if (load_group >= groups) return;
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) walk[i].load(to[i]);
        long long blocks = WK;
        if (++load_step == steps) {
            load_step = 0;
            const int next = load_group + group_step;
            if (next < groups)
                blocks = static_cast<long long>(tile_of(next) - tile_of(load_group)) * a.w.kblocks -
                         static_cast<long long>(steps - 1) * WK;
            load_group = next;
        }
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) walk[i].step(blocks);
    };
    if (steps == 0) load_group = groups;
    load(stage[0]);
    load(stage[1]);

    if (threadIdx.x < tokens) {
        const int m = m0 + threadIdx.x, q = m / a.ne1, i1 = m - q * a.ne1, i3 = q / a.ne2, i2 = q - i3 * a.ne2;
        row_at[threadIdx.x] = i1 * a.xnb[0] + i2 * a.xnb[1] + i3 * a.xnb[2];
    }
    __syncthreads();

    const uint8_t* lane_frags = frags + (lane >> 2) * kQ4Column + (lane & 3) * 8;
    float acc[S::kTiles][S::kSums];
    // One k-block, the chunk's at `at`.
    auto product = [&](const Q4Stage<G> (&st)[S::kTiles], int at) {
        const uint8_t* f = lane_frags + at * block_bytes;
        float part[S::kTiles][S::kSums];  // the k-block's sums, in its rows' scales
        float s[S::kTiles][T][4];         // a group's sums
        uint32_t w[S::kTiles][2][4];
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) {
            w[i][0][0] = st[i].lo.x; w[i][0][1] = st[i].lo.y; w[i][0][2] = st[i].lo.z; w[i][0][3] = st[i].lo.w;
            w[i][1][0] = st[i].hi.x; w[i][1][1] = st[i].hi.y; w[i][1][2] = st[i].hi.z; w[i][1][3] = st[i].hi.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t av[S::kTiles][4];
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i) {
                    const uint32_t u0 = w[i][0][j] >> (8 * h), u1 = w[i][1][j] >> (8 * h);
                    av[i][0] = q4_low(u0);
                    av[i][1] = q4_low(u1);
                    av[i][2] = q4_high(u0);
                    av[i][3] = q4_high(u1);
                }
                const int slice = 2 * j + h;
#pragma unroll
                for (int p = 0; p < S::kProducts; ++p) {
                    const uint2 b = *reinterpret_cast<const uint2*>(f + slice * 32 + p * (8 * kQ4Column));
                    const int t = HALF || PAIRED ? p : p / 2;
                    const bool first = j % (4 / NG) == 0 && h == 0 && (HALF || PAIRED || p % 2 == 0);
#pragma unroll
                    for (int i = 0; i < S::kTiles; ++i) {
                        if (first) q4_mma<true>(s[i][t], av[i], b);
                        else q4_mma<false>(s[i][t], av[i], b);
                    }
                }
            }
            if ((j + 1) % (4 / NG) != 0) continue;
            const int g = (j + 1) / (4 / NG) - 1;
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) {
                const float2 d = Q4Stage<G>::pick(st[i].d, g);
                auto join = [&](int c, float scale, float v) {
                    part[i][c] = g == 0 ? scale * v : fmaf(scale, v, part[i][c]);
                };
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    if constexpr (PAIRED) {
                        join(0, d.x, s[i][0][0] + s[i][0][1]);
                        join(1, d.y, s[i][0][2] + s[i][0][3]);
                    } else {
                        join(4 * t, d.x, s[i][t][0]);
                        join(4 * t + 1, d.x, s[i][t][1]);
                        join(4 * t + 2, d.y, s[i][t][2]);
                        join(4 * t + 3, d.y, s[i][t][3]);
                    }
                }
            }
            if (a.w.minima) {
                const float* xs = sums + (at * NG + g) * S::kTokens;
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i) {
                    const float2 d = Q4Stage<G>::pick(st[i].d, g), mn = Q4Stage<G>::pick(st[i].m, g);
                    const float o0 = fmaf(8.0f, d.x, mn.x), o1 = fmaf(8.0f, d.y, mn.y);
                    if constexpr (PAIRED) {
                        const float v = xs[lane & 3];
                        acc[i][0] = fmaf(o0, v, acc[i][0]);
                        acc[i][1] = fmaf(o1, v, acc[i][1]);
                    } else {
#pragma unroll
                        for (int t = 0; t < T; ++t) {
                            const float2 v = *reinterpret_cast<const float2*>(xs + t * 8 + (lane & 3) * 2);
                            acc[i][4 * t] = fmaf(o0, v.x, acc[i][4 * t]);
                            acc[i][4 * t + 1] = fmaf(o0, v.y, acc[i][4 * t + 1]);
                            acc[i][4 * t + 2] = fmaf(o1, v.x, acc[i][4 * t + 2]);
                            acc[i][4 * t + 3] = fmaf(o1, v.y, acc[i][4 * t + 3]);
                        }
                    }
                }
            }
        }
        const float* xs = scales + at * S::kTokens;
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) {
            if constexpr (HALF) {
#pragma unroll
                for (int c = 0; c < S::kSums; ++c) acc[i][c] += part[i][c];
            } else if constexpr (PAIRED) {
                const float v = xs[lane & 3];
                acc[i][0] = fmaf(v, part[i][0], acc[i][0]);
                acc[i][1] = fmaf(v, part[i][1], acc[i][1]);
            } else {
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const float2 v = *reinterpret_cast<const float2*>(xs + t * 8 + (lane & 3) * 2);
                    acc[i][4 * t] = fmaf(v.x, part[i][4 * t], acc[i][4 * t]);
                    acc[i][4 * t + 1] = fmaf(v.y, part[i][4 * t + 1], acc[i][4 * t + 1]);
                    acc[i][4 * t + 2] = fmaf(v.x, part[i][4 * t + 2], acc[i][4 * t + 2]);
                    acc[i][4 * t + 3] = fmaf(v.y, part[i][4 * t + 3], acc[i][4 * t + 3]);
                }
            }
        }
    };

    bool held = false;  // the one chunk of x is in shared memory
    int parity = 0;
    for (int group = group0; group < groups; group += group_step) {
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
            for (int c = 0; c < S::kSums; ++c) acc[i][c] = 0.0f;
        for (int kc = kb_begin; kc < kb_end; kc += a.chunk) {
            const int kc_end = min(kc + a.chunk, kb_end);
            if (!held) {
                if (kc != kb_begin || group != group0) __syncthreads();  // the chunk before has been read
                q4_split<T, PAIRED, HALF, G>(a, row_at, tokens, kc, kc_end, frags, scales, sums);
                __syncthreads();
                held = a.chunk >= kb_end - kb_begin;
            }
            int at = wk;
            for (; at + WK < kc_end - kc; at += 2 * WK) {
                product(stage[0], at);
                load(stage[0]);
                product(stage[1], at + WK);
                load(stage[1]);
            }
            if (at < kc_end - kc) {
                product(stage[0], at);
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i) stage[0][i] = stage[1][i];
                load(stage[1]);
            }
        }

        // The warps' sums: [warp][tile][sum][lane].
        float* mine = red + parity * S::kRedFloats;
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
            for (int c = 0; c < S::kSums; ++c) mine[((warp * S::kTiles + i) * S::kSums + c) * 32 + lane] = acc[i][c];
        if (a.cluster > 1) cooperative_groups::this_cluster().sync();
        else __syncthreads();
        // An output's sums lie WK (of each CTA) apart; a cluster's CTAs share the outputs.
        const int outs = WR * 16 * tokens;
        for (int o = threadIdx.x * a.cluster + rank; o < outs; o += kQ4Threads * a.cluster) {
            const int r = o & 15, q = o >> 4, m = q / WR, tw = q - m * WR;
            const long long n = (static_cast<long long>(group) * WR + tw) * 16 + r;
            if (n >= a.w.n) continue;
            int c, l;
            if constexpr (PAIRED) {
                c = r >> 3;
                l = (r & 7) * 4 + m;
            } else {
                c = (m >> 3) * 4 + (r >> 3) * 2 + (m & 1);
                l = (r & 7) * 4 + ((m & 7) >> 1);
            }
            float v[2] = {0.0f, 0.0f};
            for (int k = 0; k < a.cluster; ++k) {
                const float* from =
                    a.cluster > 1 ? cooperative_groups::this_cluster().map_shared_rank(mine, k) : mine;
                for (int j = 0; j < WK; ++j) {
#pragma unroll
                    for (int i = 0; i < S::kTiles; ++i)
                        v[i] += from[(((tw * WK + j) * S::kTiles + i) * S::kSums + c) * 32 + l];
                }
            }
            q4_finish(a, m0 + m, n, v[0], v[1], GATED);
        }
        if constexpr (S::kRedBuffers == 2) {
            parity ^= 1;  // the buffer is written again after the next barrier
        } else {
            if (a.cluster > 1) cooperative_groups::this_cluster().sync();
            else __syncthreads();
        }
    }
    if (a.cluster > 1) cooperative_groups::this_cluster().sync();  // the others have read this CTA's sums
}

// How a product is cut: see q4_linear.cu.
struct Q4Plan {
    int form;      // 0: PAIRED; else T = 1, 2 or 4
    int blocks;    // grid x
    int chunks;    // grid y: rows of x in runs of the form's tokens
};

// Launches the kernel for FP16 or FP32 rows, plain or gated, groups of G; cudaGetLastError() says how it went.
template <int G>
int q4_launch(const Q4Args& a, const Q4Plan& p, bool half, cudaStream_t st);

}  // namespace sdb
