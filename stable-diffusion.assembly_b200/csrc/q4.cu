// 4-bit matrices: made from FP16 / FP32 numbers, from 4-bit numbers and group
// scales, or from ggml's Q4_0 / Q4_1 blocks, and turned back into FP32.
//
// All four are one pass over the matrix, a lane to a word of eight columns
// (q4.cuh), bound by memory; quantizing by its instructions.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/sdb.h"
#include "q4.cuh"
#include "runtime.cuh"

namespace sdb {

namespace {

// A warp takes 1024 columns of a row, four runs of 256, a lane a word of eight columns of each: no division to
// find them, and four loads on their way.
constexpr int kRuns = 4;

__host__ inline dim3 word_grid(const Q4View& v, long long rows) {
    return dim3(static_cast<unsigned>((rows + 7) / 8), static_cast<unsigned>((v.kblocks + 7) / 8));
}

__device__ __forceinline__ long long word_row() { return blockIdx.x * 8LL + threadIdx.x / 32; }
__device__ __forceinline__ int word_column(int run) {
    return static_cast<int>(blockIdx.y) * 1024 + run * 256 + (threadIdx.x & 31) * 8;
}

__device__ __forceinline__ float saturate_half(float v) { return fminf(fmaxf(v, -65504.0f), 65504.0f); }

// Quantizes eight columns a thread; the extremes of a group come from the
// group / 8 neighbouring lanes that hold it.  Every step is a rounded FP32
// operation of its own (no contraction), so that the numbers chosen are those
// of the formulas:
//   symmetric  s = the group's number of greatest magnitude (max when both are equal),
//              d = f16(s / -8), q = clamp(floor(w / d + 8.5), 0, 15), all 8 where d = 0
//   minimum    d = f16((max - min) / 15), m = f16(min),
//              q = clamp(floor((w - m) / d + 0.5), 0, 15), all 0 where d = 0
// d and m saturate at FP16's range.  A group that holds an infinity or a NaN
// stands for NaN throughout.
template <typename T, bool MINIMUM>
__global__ void __launch_bounds__(256) q4_quantize_kernel(const T* __restrict__ w, long long ld, Q4View v) {
    const int lanes = v.group / 8, k = static_cast<int>(v.k);
    const long long row = word_row();
    const Q4RowAt to(v, row);
    float xs[kRuns][8];
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
        const int k0 = word_column(r), cols = row < v.n ? k - k0 : 0;
        float (&x)[8] = xs[r];
        const T* src = w + row * ld + k0;
        if (cols >= 8 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            if constexpr (sizeof(T) == 4) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(src));
                const float4 b = __ldg(reinterpret_cast<const float4*>(src) + 1);
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
                const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
                const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[p]));
                    x[2 * p] = f.x;
                    x[2 * p + 1] = f.y;
                }
            }
        } else {
            // Past the row's end its last number again, which changes neither extreme.
#pragma unroll
            for (int c = 0; c < 8; ++c) x[c] = cols > 0 ? static_cast<float>(src[min(c, cols - 1)]) : 0.0f;
        }
    }
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
        const int k0 = word_column(r);
        if (k0 >= v.kblocks * 128) break;  // whole groups of lanes leave together: k-blocks are 16 lanes
        const bool in = row < v.n && k0 < k;
        const float (&x)[8] = xs[r];
        float hi = in ? x[0] : -INFINITY, lo = in ? x[0] : INFINITY, zero = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            hi = in ? fmaxf(hi, x[c]) : hi;
            lo = in ? fminf(lo, x[c]) : lo;
            zero = fmaf(x[c], 0.0f, zero);  // NaN from an infinity or a NaN
        }
        // The group's own lanes: all of them are here.
        const unsigned mask = ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
        for (int o = 1; o < lanes; o <<= 1) {
            hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
            lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
            zero += __shfl_xor_sync(mask, zero, o);
        }
        const bool bad = zero != 0.0f;
        // A group of padding.  Its numbers do not tell: a short last group of NaN alone has no extremes either.
        const bool empty = row >= v.n || (k0 & ~(v.group - 1)) >= k;
        __half dh = __float2half_rn(0.0f), mh = dh;
        if (!empty) {
            if (MINIMUM) {
                dh = __float2half_rn(saturate_half(__fdiv_rn(__fsub_rn(hi, lo), 15.0f)));
                mh = __float2half_rn(saturate_half(lo));
            } else {
                dh = __float2half_rn(saturate_half((hi >= -lo ? hi : lo) * -0.125f));  // s / -8
            }
            if (bad) dh = __ushort_as_half(0x7fff);
        }
        const float d = __half2float(dh), m = __half2float(mh);
        // With 1 / d for the division, t is off by under 3e-6: where that is far from the next integer the number
        // is the formula's; else (one word in thousands) the word is made again by true divisions.  t is clamped
        // first, and 2^23 + t rounded towards zero ends in its floor.
        constexpr float add = MINIMUM ? 0.5f : 8.5f;
        uint32_t word = MINIMUM ? 0u : 0x88888888u;
        if (d != 0.0f) {
            const float inverse = __fdiv_rn(1.0f, d);
            bool near = !(fabsf(inverse) < INFINITY);
            word = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float n = MINIMUM ? __fsub_rn(x[c], m) : x[c];
                const float t = fminf(fmaxf(__fadd_rn(__fmul_rn(n, inverse), add), 0.0f), 15.5f);
                const float f = __fadd_rz(t, 8388608.0f);
                near |= fabsf(t - (f - 8388608.0f) - 0.5f) > 0.4999f;
                word |= (__float_as_uint(f) & 15u) << q4_bit(c);
            }
            if (near) {
                word = 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float n = MINIMUM ? __fsub_rn(x[c], m) : x[c];
                    const float q = fminf(fmaxf(floorf(__fadd_rn(__fdiv_rn(n, d), add)), 0.0f), 15.0f);
                    word |= static_cast<uint32_t>(static_cast<int>(q)) << q4_bit(c);
                }
            }
        }
        *to.word(k0) = word ^ 0x88888888u;
        if ((k0 & (v.group - 1)) == 0) {
            __half* s = to.scale(k0);
            *s = dh;
            if (MINIMUM) s[16 * v.ng] = mh;
        }
    }
}

// 4-bit numbers two a byte (the even column low) and scales [n][groups].
__global__ void __launch_bounds__(256) q4_import_kernel(const uint8_t* __restrict__ codes, long long code_row,
                                                        const __half* __restrict__ scales,
                                                        const __half* __restrict__ minima, long long groups,
                                                        Q4View v) {
    struct {
        long long row;
        int k0;
    } at;
    at.row = word_row();
    const Q4RowAt to(v, at.row);
    for (int r = 0; r < kRuns; ++r) {
        at.k0 = word_column(r);
        if (at.k0 >= v.kblocks * 128) break;
        const bool row_in = at.row < v.n;
        uint32_t word = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            uint32_t q = minima ? 0 : 8;
            if (row_in && at.k0 + c < v.k) {
                const uint32_t b = __ldg(codes + at.row * code_row + (at.k0 + c) / 2);
                q = (c & 1) ? b >> 4 : b & 15;
            }
            word |= q << q4_bit(c);
        }
        *to.word(at.k0) = word ^ 0x88888888u;
        if (at.k0 % v.group == 0) {
            __half* s = to.scale(at.k0);
            const bool in = row_in && at.k0 < v.k;
            const long long from = at.row * groups + at.k0 / v.group;
            *s = in ? scales[from] : __float2half_rn(0.0f);
            if (minima) s[16 * v.ng] = in ? minima[from] : __float2half_rn(0.0f);
        }
    }
}

// ggml's blocks of 32 numbers: the FP16 scale, with Q4_1 the FP16 minimum,
// then 16 bytes, byte i numbers i (low) and i + 16 (high).
__global__ void __launch_bounds__(256) q4_blocks_kernel(const uint8_t* __restrict__ blocks, long long row_bytes,
                                                        Q4View v) {
    const int header = v.minimum ? 4 : 2, size = header + 16;
    struct {
        long long row;
        int k0;
    } at;
    at.row = word_row();
    const Q4RowAt to(v, at.row);
    for (int r = 0; r < kRuns; ++r) {
        at.k0 = word_column(r);
        if (at.k0 >= v.kblocks * 128) break;
        const bool in = at.row < v.n && at.k0 < v.k;
        const uint8_t* b = blocks + at.row * row_bytes + at.k0 / 32 * size;
        const int first = static_cast<int>(at.k0) & 31;
        uint32_t word = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            uint32_t q = v.minimum ? 0 : 8;
            if (in) {
                const uint32_t two = __ldg(b + header + (first & 15) + c);
                q = first < 16 ? two & 15 : two >> 4;
            }
            word |= q << q4_bit(c);
        }
        *to.word(at.k0) = word ^ 0x88888888u;
        if (first == 0) {
            __half* s = to.scale(at.k0);
            uint32_t d = 0, m = 0;
            if (in) {
                d = b[0] | static_cast<uint32_t>(b[1]) << 8;
                if (v.minimum) m = b[2] | static_cast<uint32_t>(b[3]) << 8;
            }
            *s = __ushort_as_half(static_cast<unsigned short>(d));
            if (v.minimum) s[16 * v.ng] = __ushort_as_half(static_cast<unsigned short>(m));
        }
    }
}

// A run's numbers cross shared memory, so that a store's lanes write neighbours.
__global__ void __launch_bounds__(256) q4_dequantize_kernel(Q4View v, float* __restrict__ w, long long ld) {
    __shared__ __align__(16) float turned[8][256];
    float* own = turned[threadIdx.x / 32];
    const int lane = threadIdx.x & 31;
    const long long row = word_row();
    const Q4RowAt from(v, row);
    const int k = static_cast<int>(v.k);
    uint32_t words[kRuns];
    float ds[kRuns], ms[kRuns];
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
        const int k0 = word_column(r);
        words[r] = 0;
        ds[r] = ms[r] = 0.0f;
        if (row < v.n && k0 < k) {
            words[r] = __ldg(from.word(k0)) ^ 0x88888888u;
            const __half* s = from.scale(k0);
            ds[r] = __half2float(s[0]);
            if (v.minimum) ms[r] = __half2float(s[16 * v.ng]);
        }
    }
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
        const int first = word_column(r) - lane * 8;  // the warp's run
        if (row >= v.n || first >= k) break;
        float x[8];
        // d q and d (q - 8) are exact in FP32 (11 and 4 bits).
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float code = static_cast<float>(words[r] >> q4_bit(c) & 15u);
            x[c] = v.minimum ? fmaf(ds[r], code, ms[r]) : ds[r] * (code - 8.0f);
        }
        __syncwarp();  // the run before has been read
        reinterpret_cast<float4*>(own)[lane * 2] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(own)[lane * 2 + 1] = make_float4(x[4], x[5], x[6], x[7]);
        __syncwarp();
        float* dst = w + row * ld + first;
        if (first + 256 <= k && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                reinterpret_cast<float4*>(dst)[i * 32 + lane] = reinterpret_cast<const float4*>(own)[i * 32 + lane];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (first + i * 32 + lane < k) dst[i * 32 + lane] = own[i * 32 + lane];
        }
    }
}

// What every maker of a matrix does first: the products' error word is allocated with the matrix, not by a first
// product that a stream capture records.
void prepare_device() { device_error_word(); }

// A matrix [k, n] with contiguous rows of the 4-bit matrix's extents.
bool matrix_of(const sdb_tensor* w, const sdb_q4* q, bool f16) {
    if (w == nullptr || w->data == nullptr) return false;
    if (w->type != SDB_TYPE_F32 && !(f16 && w->type == SDB_TYPE_F16)) return false;
    const int64_t es = w->type == SDB_TYPE_F16 ? 2 : 4;
    return w->ne[0] == q->k && w->ne[1] == q->n && w->ne[2] == 1 && w->ne[3] == 1 && (w->nb[0] == es || w->ne[0] == 1) &&
           w->nb[1] % es == 0 && (w->ne[1] == 1 || w->nb[1] >= es * w->ne[0]) &&
           reinterpret_cast<uintptr_t>(w->data) % es == 0;
}

}  // namespace

}  // namespace sdb

using namespace sdb;

extern "C" {

int64_t sdb_q4_bytes(int64_t k, int64_t n, int32_t group, int32_t minimum) {
    if (!q4_valid_form(k, n, group, minimum)) return 0;
    const int64_t blocks = (n + 15) / 16 * ((k + 127) / 128);
    return blocks * (1024 + 32 * (128 / group) * (minimum ? 2 : 1));
}

int sdb_q4_quantize(const sdb_tensor* w, const sdb_q4* q, void* stream) {
    if (!q4_valid(q)) return fail(SDB_INVALID, "sdb_q4_quantize: no such 4-bit matrix");
    if (!matrix_of(w, q, true))
        return fail(SDB_INVALID, "sdb_q4_quantize: w must be an FP32 or FP16 matrix [k, n] with contiguous rows");
    prepare_device();
    const Q4View v = q4_view(q);
    const auto st = static_cast<cudaStream_t>(stream);
    const dim3 blocks = word_grid(v, v.tiles * 16LL);
    if (w->type == SDB_TYPE_F32) {
        const auto* src = static_cast<const float*>(w->data);
        if (v.minimum) q4_quantize_kernel<float, true><<<blocks, 256, 0, st>>>(src, w->nb[1] / 4, v);
        else q4_quantize_kernel<float, false><<<blocks, 256, 0, st>>>(src, w->nb[1] / 4, v);
    } else {
        const auto* src = static_cast<const __half*>(w->data);
        if (v.minimum) q4_quantize_kernel<__half, true><<<blocks, 256, 0, st>>>(src, w->nb[1] / 2, v);
        else q4_quantize_kernel<__half, false><<<blocks, 256, 0, st>>>(src, w->nb[1] / 2, v);
    }
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}

int sdb_q4_import(const void* codes, const void* scales, const void* minima, const sdb_q4* q, void* stream) {
    if (!q4_valid(q)) return fail(SDB_INVALID, "sdb_q4_import: no such 4-bit matrix");
    if (codes == nullptr || scales == nullptr || (minima != nullptr) != (q->minimum != 0) ||
        reinterpret_cast<uintptr_t>(scales) % 2 != 0 || reinterpret_cast<uintptr_t>(minima) % 2 != 0)
        return fail(SDB_INVALID, "sdb_q4_import: codes, FP16 scales and (with `minimum`, only then) FP16 minima");
    prepare_device();
    const Q4View v = q4_view(q);
    q4_import_kernel<<<word_grid(v, v.tiles * 16LL), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(codes), (q->k + 1) / 2, static_cast<const __half*>(scales),
        static_cast<const __half*>(minima), (q->k + q->group - 1) / q->group, v);
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}

int sdb_q4_from_blocks(const void* blocks, int64_t row_bytes, const sdb_q4* q, void* stream) {
    if (!q4_valid(q)) return fail(SDB_INVALID, "sdb_q4_from_blocks: no such 4-bit matrix");
    if (q->group != 32 || q->k % 32 != 0)
        return fail(SDB_INVALID, "sdb_q4_from_blocks: ggml's blocks are groups of 32, k a multiple of 32");
    if (blocks == nullptr || row_bytes < q->k / 32 * (q->minimum ? 20 : 18))
        return fail(SDB_INVALID, "sdb_q4_from_blocks: no blocks, or rows shorter than k / 32 blocks");
    prepare_device();
    const Q4View v = q4_view(q);
    q4_blocks_kernel<<<word_grid(v, v.tiles * 16LL), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(blocks), row_bytes, v);
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}

int sdb_q4_dequantize(const sdb_q4* q, const sdb_tensor* w, void* stream) {
    if (!q4_valid(q)) return fail(SDB_INVALID, "sdb_q4_dequantize: no such 4-bit matrix");
    if (!matrix_of(w, q, false))
        return fail(SDB_INVALID, "sdb_q4_dequantize: w must be an FP32 matrix [k, n] with contiguous rows");
    const Q4View v = q4_view(q);
    q4_dequantize_kernel<<<word_grid(v, v.n), 256, 0, static_cast<cudaStream_t>(stream)>>>(v, static_cast<float*>(w->data),
                                                                                w->nb[1] / 4);
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}

}  // extern "C"
