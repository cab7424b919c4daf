// The residual block of a transformer in one pass over its rows:
//   h   = keep x + scale gate post(y)
//   out = pre(h) (1 + mul) + add
// post and pre are nothing, a LayerNorm or an RMS norm of the row; gate, mul
// and add are operands of the output's extents or broadcast along any of them.
//
// Bound by memory: x and y are read once and h and out written once, the row's
// numbers in registers in between, both statistics and the normalisations from
// there -- a warp a row up to 512 numbers, a CTA up to 16384 (residual_kernel);
// wider rows are read again for each pass (residual_rows_kernel).  The mean of a
// LayerNorm comes from a first sum, the variance from the sum of d^2 about that
// float mean less the square of d's own mean (d = v - mean), so that rows far
// from 0 lose nothing; sums are FP32, a thread's share of a row and a tree.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/sdb.h"
#include "runtime.cuh"

namespace sdb {

namespace {

struct NormForm {
    int kind;
    float eps;
    const float* weight;
    const float* bias;
};

struct Operand {
    const float* data;
    long long nb[4];  // in elements
};

struct ResidualArgs {
    const void* x;
    const void* y;
    void* h;
    void* out;
    long long xnb[3], ynb[3], hnb[3], onb[3];  // strides of rows in elements (dims 1..3)
    long long ne1, ne2, rows;
    int c;
    float keep, scale;
    NormForm post, pre;
    Operand gate, mul, add;
};

template <typename T>
__device__ __forceinline__ float get(const T* p, long long i) {
    return static_cast<float>(p[i]);
}
__device__ __forceinline__ void put(float* p, long long i, float v) { p[i] = v; }
__device__ __forceinline__ void put(__half* p, long long i, float v) { p[i] = __float2half_rn(v); }

constexpr int kRowThreads = 256;

__device__ __forceinline__ float2 block_sum(float2 v) {
    __shared__ float2 part[kRowThreads / 32];
    for (int o = 16; o; o >>= 1) {
        v.x += __shfl_xor_sync(~0u, v.x, o);
        v.y += __shfl_xor_sync(~0u, v.y, o);
    }
    __syncthreads();  // a sum before has been read
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    float2 s = part[0];
    for (int w = 1; w < kRowThreads / 32; ++w) {
        s.x += part[w].x;
        s.y += part[w].y;
    }
    return s;
}

// A row's norm as v -> (v - mean - shift) * rstd, the two subtractions apart.
struct Stat {
    float mean, shift, rstd;
};

// 1 / sqrt(var + eps).  A rounded variance may come out below 0; a NaN stays one, so that it fills its row.
__device__ __forceinline__ float reciprocal_root(float var, float eps) {
    return 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);
}

// value(i) is the row's number i.
template <typename F>
__device__ __forceinline__ Stat row_stat(const NormForm& n, int c, F value) {
    Stat s{0.0f, 0.0f, 1.0f};
    if (n.kind == SDB_NORM_NONE) return s;
    const float inv = 1.0f / static_cast<float>(c);
    if (n.kind == SDB_NORM_LAYER) {
        float2 t{0.0f, 0.0f};
        for (int i = threadIdx.x; i < c; i += kRowThreads) t.x += value(i);
        s.mean = block_sum(t).x * inv;
    }
    float2 t{0.0f, 0.0f};
    for (int i = threadIdx.x; i < c; i += kRowThreads) {
        const float d = value(i) - s.mean;
        t.x += d;
        t.y = fmaf(d, d, t.y);
    }
    t = block_sum(t);
    if (n.kind == SDB_NORM_LAYER) s.shift = t.x * inv;
    s.rstd = reciprocal_root(t.y * inv - s.shift * s.shift, n.eps);
    return s;
}

__device__ __forceinline__ float normed(const NormForm& n, const Stat& s, float v, int i) {
    if (n.kind == SDB_NORM_NONE) return v;
    v = (v - s.mean - s.shift) * s.rstd;
    if (n.weight) v *= __ldg(n.weight + i);
    if (n.bias) v += __ldg(n.bias + i);
    return v;
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kRowThreads) residual_rows_kernel(const ResidualArgs a) {
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long i1 = row % a.ne1, q = row / a.ne1, i2 = q % a.ne2, i3 = q / a.ne2;
        const TX* x = a.x ? static_cast<const TX*>(a.x) + i1 * a.xnb[0] + i2 * a.xnb[1] + i3 * a.xnb[2] : nullptr;
        const TY* y = a.y ? static_cast<const TY*>(a.y) + i1 * a.ynb[0] + i2 * a.ynb[1] + i3 * a.ynb[2] : nullptr;
        auto operand = [&](const Operand& o) {
            return o.data ? o.data + i1 * o.nb[1] + i2 * o.nb[2] + i3 * o.nb[3] : nullptr;
        };
        const float* gate = operand(a.gate);
        const float* mul = operand(a.mul);
        const float* add = operand(a.add);
        Stat ps{};
        if (y) ps = row_stat(a.post, a.c, [&](int i) { return get(y, i); });
        auto stream = [&](int i) {
            float v = x ? a.keep * get(x, i) : 0.0f;
            if (y) {
                float u = normed(a.post, ps, get(y, i), i);
                if (gate) u *= __ldg(gate + i * a.gate.nb[0]);
                v = fmaf(a.scale, u, v);
            }
            return v;
        };
        Stat hs{};
        if (a.out) hs = row_stat(a.pre, a.c, stream);
        TX* h = a.h ? static_cast<TX*>(a.h) + i1 * a.hnb[0] + i2 * a.hnb[1] + i3 * a.hnb[2] : nullptr;
        TY* out = a.out ? static_cast<TY*>(a.out) + i1 * a.onb[0] + i2 * a.onb[1] + i3 * a.onb[2] : nullptr;
        for (int i = threadIdx.x; i < a.c; i += kRowThreads) {
            const float v = stream(i);  // x and y at i are read before h and out there are written
            if (h) put(h, i, v);
            if (out) {
                float w = normed(a.pre, hs, v, i);
                if (mul) w *= 1.0f + __ldg(mul + i * a.mul.nb[0]);
                if (add) w += __ldg(add + i * a.add.nb[0]);
                put(out, i, w);
            }
        }
    }
}

// ---- rows in registers

// Four numbers at p[0..3] (16 or 8 bytes at a time); plain loads, since h and out may be the same memory.
__device__ __forceinline__ float4 get4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 get4(const __half* p) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void put4(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put4(__half* p, const float (&v)[4]) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// The sum over the T threads of a row, in all of them; *buffer alternates, so that a sum's partial sums are not
// overwritten before every warp has read them.
template <int T>
__device__ __forceinline__ float2 row_sum(float2 v, int* buffer) {
    for (int o = 16; o; o >>= 1) {
        v.x += __shfl_xor_sync(~0u, v.x, o);
        v.y += __shfl_xor_sync(~0u, v.y, o);
    }
    if constexpr (T > 32) {
        __shared__ float2 part[2][T / 32];
        float2* p = part[*buffer];
        *buffer ^= 1;
        if ((threadIdx.x & 31) == 0) p[threadIdx.x / 32] = v;
        __syncthreads();
        v = p[0];
#pragma unroll
        for (int w = 1; w < T / 32; ++w) {
            v.x += p[w].x;
            v.y += p[w].y;
        }
    }
    return v;
}

// T threads a row (32: eight rows a CTA), 4 V numbers a thread: with VEC, runs of four (rows of a multiple of four
// numbers, aligned), else one by one.  A thread's numbers lie T (runs) apart.
template <typename TX, typename TY, int V, int T, bool VEC>
// Registers for 1024 threads an SM: 64 a thread (rows of 8193 to 16384 numbers: 128), more rows at once being worth
// more than what spills -- with VEC 24 bytes at most, number by number 8 to 32, 120 (513 to 1280 numbers of FP16) and
// 192 (4097 to 8192) -- 8 x 4096 x 320 35.7 us, unbounded 40.0; 2 x 4096 x 1280 30.1 and 30.8.
__global__ void __launch_bounds__(T == 32 ? 256 : T, (V == 8 ? 512 : 1024) / (T == 32 ? 256 : T)) residual_kernel(const __grid_constant__ ResidualArgs a) {
    const int t = T == 32 ? threadIdx.x & 31 : threadIdx.x;
    constexpr int kRows = T == 32 ? 8 : 1;
    int buffer = 0;
    auto at = [&](int v, int e) { return VEC ? (v * T + t) * 4 + e : (v * 4 + e) * T + t; };
    for (long long row = blockIdx.x * static_cast<long long>(kRows) + (T == 32 ? threadIdx.x / 32 : 0); row < a.rows;
         row += gridDim.x * static_cast<long long>(kRows)) {
        const int q = static_cast<int>(row) / static_cast<int>(a.ne1), i1 = static_cast<int>(row) - q * static_cast<int>(a.ne1);
        const int i3 = q / static_cast<int>(a.ne2), i2 = q - i3 * static_cast<int>(a.ne2);
        auto base = [&](const long long (&nb)[3]) { return i1 * nb[0] + i2 * nb[1] + i3 * nb[2]; };
        float h[V][4], u[V][4];
        // f(v, e) for the thread's numbers, a run that ends the row early passed over as a whole.
        auto each = [&](auto f) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (VEC) {
                    if (at(v, 0) < a.c) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) f(v, e);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at(v, e) < a.c) f(v, e);
                }
            }
        };
        auto load = [&](float (&to)[V][4], const auto* p) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (VEC) {
                    if (at(v, 0) < a.c) {
                        const float4 f = get4(p + at(v, 0));
                        to[v][0] = f.x; to[v][1] = f.y; to[v][2] = f.z; to[v][3] = f.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at(v, e) < a.c) to[v][e] = get(p, at(v, e));
                }
            }
        };
        // f(v, e, operand's number) over the row, the operand's numbers nb apart.
        auto with = [&](const float* p, long long nb, auto f) {
            if (VEC && nb == 1 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (at(v, 0) < a.c) {
                        const float4 o = __ldg(reinterpret_cast<const float4*>(p + at(v, 0)));
                        f(v, 0, o.x);
                        f(v, 1, o.y);
                        f(v, 2, o.z);
                        f(v, 3, o.w);
                    }
                }
            } else {
                each([&](int v, int e) { f(v, e, __ldg(p + at(v, e) * nb)); });
            }
        };
        auto normalise = [&](const NormForm& n, float (&to)[V][4]) {
            if (n.kind == SDB_NORM_NONE) return;
            const float inv = 1.0f / static_cast<float>(a.c);
            float2 s{0.0f, 0.0f};
            float shift = 0.0f;
            if (n.kind == SDB_NORM_LAYER) {
                each([&](int v, int e) { s.x += to[v][e]; });
                const float mean = row_sum<T>(s, &buffer).x * inv;
                s.x = 0.0f;
                each([&](int v, int e) {
                    to[v][e] -= mean;
                    s.x += to[v][e];
                    s.y = fmaf(to[v][e], to[v][e], s.y);
                });
            } else {
                each([&](int v, int e) { s.y = fmaf(to[v][e], to[v][e], s.y); });
            }
            s = row_sum<T>(s, &buffer);
            if (n.kind == SDB_NORM_LAYER) shift = s.x * inv;
            const float rstd = reciprocal_root(s.y * inv - shift * shift, n.eps);
            each([&](int v, int e) { to[v][e] = (to[v][e] - shift) * rstd; });
            if (n.weight) with(n.weight, 1, [&](int v, int e, float w) { to[v][e] *= w; });
            if (n.bias) with(n.bias, 1, [&](int v, int e, float b) { to[v][e] += b; });
        };
        auto store = [&](auto* p, const float (&from)[V][4]) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (VEC) {
                    if (at(v, 0) < a.c) put4(p + at(v, 0), from[v]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at(v, e) < a.c) put(p, at(v, e), from[v][e]);
                }
            }
        };
        auto operand = [&](const Operand& o) { return o.data + i1 * o.nb[1] + i2 * o.nb[2] + i3 * o.nb[3]; };

        if (a.y) load(u, static_cast<const TY*>(a.y) + base(a.ynb));
        if (a.x) load(h, static_cast<const TX*>(a.x) + base(a.xnb));
        if (a.y) {
            normalise(a.post, u);
            if (a.gate.data) with(operand(a.gate), a.gate.nb[0], [&](int v, int e, float g) { u[v][e] *= g; });
        }
        each([&](int v, int e) {
            float s = a.x ? a.keep * h[v][e] : 0.0f;
            if (a.y) s = fmaf(a.scale, u[v][e], s);
            h[v][e] = s;
        });
        if (a.h) store(static_cast<TX*>(a.h) + base(a.hnb), h);
        if (a.out) {
            normalise(a.pre, h);
            if (a.mul.data) with(operand(a.mul), a.mul.nb[0], [&](int v, int e, float m) { h[v][e] *= 1.0f + m; });
            if (a.add.data) with(operand(a.add), a.add.nb[0], [&](int v, int e, float m) { h[v][e] += m; });
            store(static_cast<TY*>(a.out) + base(a.onb), h);
        }
    }
}

template <typename TX, typename TY, int V, int T>
void launch_rows(const ResidualArgs& a, bool vec, cudaStream_t st) {
    constexpr int rows = T == 32 ? 8 : 1, threads = T == 32 ? 256 : T;
    const unsigned blocks = static_cast<unsigned>(std::min<long long>((a.rows + rows - 1) / rows, 1LL << 20));
    if (vec) residual_kernel<TX, TY, V, T, true><<<blocks, threads, 0, st>>>(a);
    else residual_kernel<TX, TY, V, T, false><<<blocks, threads, 0, st>>>(a);
}

template <typename TX, typename TY>
void launch(const ResidualArgs& a, bool vec, cudaStream_t st) {
    if (a.c <= 256) launch_rows<TX, TY, 2, 32>(a, vec, st);
    else if (a.c <= 512) launch_rows<TX, TY, 4, 32>(a, vec, st);
    else if (a.c <= 1280) launch_rows<TX, TY, 5, 64>(a, vec, st);
    else if (a.c <= 2048) launch_rows<TX, TY, 4, 128>(a, vec, st);
    else if (a.c <= 4096) launch_rows<TX, TY, 4, 256>(a, vec, st);
    else if (a.c <= 8192) launch_rows<TX, TY, 4, 512>(a, vec, st);
    else if (a.c <= 16384) launch_rows<TX, TY, 8, 512>(a, vec, st);
    else
        residual_rows_kernel<TX, TY>
            <<<static_cast<unsigned>(std::min<long long>(a.rows, current_sm_count() * 32LL)), kRowThreads, 0, st>>>(a);
}

bool rows_of(const sdb_tensor* t, bool written) {
    if (t->type != SDB_TYPE_F32 && t->type != SDB_TYPE_F16) return false;
    const int64_t es = t->type == SDB_TYPE_F16 ? 2 : 4;
    for (int d = 0; d < 4; ++d)
        if (t->ne[d] < 0 || t->nb[d] < 0 || t->nb[d] % es != 0) return false;
    for (int d = 1; written && d < 4; ++d)
        if (t->ne[d] > 1 && t->nb[d] == 0) return false;
    return (t->nb[0] == es || t->ne[0] == 1) && t->data != nullptr && reinterpret_cast<uintptr_t>(t->data) % es == 0;
}

bool norm_ok(const sdb_norm_form& n) {
    return n.kind == SDB_NORM_NONE || ((n.kind == SDB_NORM_LAYER || n.kind == SDB_NORM_RMS) && n.eps >= 0.0f);
}

}  // namespace

}  // namespace sdb

using namespace sdb;

extern "C" int sdb_residual_norm(const sdb_tensor* x, const sdb_tensor* y, const sdb_tensor* h,
                                 const sdb_tensor* out, const sdb_residual* p, void* stream) {
    if (p == nullptr || (x == nullptr && y == nullptr) || (h == nullptr && out == nullptr))
        return fail(SDB_INVALID, "sdb_residual_norm: parameters, one of x and y, one of h and out");
    const sdb_tensor* ref = x ? x : y;
    for (const sdb_tensor* t : {x, y, h, out}) {
        if (t == nullptr) continue;
        for (int d = 0; d < 4; ++d)
            if (t->ne[d] != ref->ne[d]) return fail(SDB_INVALID, "sdb_residual_norm: extents differ");
    }
    const int64_t limit = 1LL << 30;
    for (int d = 0; d < 4; ++d)
        if (ref->ne[d] < 0 || ref->ne[d] > limit) return fail(SDB_INVALID, "sdb_residual_norm: extents");
    if (ref->ne[0] == 0) return fail(SDB_INVALID, "sdb_residual_norm: rows of no numbers");
    const double rows = static_cast<double>(ref->ne[1]) * ref->ne[2] * ref->ne[3];
    if (rows > static_cast<double>(limit)) return fail(SDB_INVALID, "sdb_residual_norm: too many rows");
    if (rows == 0) return SDB_OK;
    for (const sdb_tensor* t : {x, y, h, out})
        if (t && !rows_of(t, t == h || t == out))
            return fail(SDB_INVALID, "sdb_residual_norm: FP32 or FP16 tensors with contiguous rows");
    if ((x && h && x->type != h->type) || (y && out && y->type != out->type))
        return fail(SDB_INVALID, "sdb_residual_norm: h has x's type, out has y's");
    if (!norm_ok(p->post) || !norm_ok(p->pre))
        return fail(SDB_INVALID, "sdb_residual_norm: a norm is none, LayerNorm or RMS, eps not negative");
    if (y == nullptr && (p->post.kind != SDB_NORM_NONE || p->gate.data))
        return fail(SDB_INVALID, "sdb_residual_norm: a norm or gate of no y");
    if (out == nullptr && (p->pre.kind != SDB_NORM_NONE || p->mul.data || p->add.data))
        return fail(SDB_INVALID, "sdb_residual_norm: a norm or modulation of no out");
    for (const sdb_operand* o : {&p->gate, &p->mul, &p->add})
        for (int d = 0; o->data && d < 4; ++d)
            if (o->nb[d] < 0 || reinterpret_cast<uintptr_t>(o->data) % 4 != 0)
                return fail(SDB_INVALID, "sdb_residual_norm: operand strides");

    ResidualArgs a{};
    auto strides = [](const sdb_tensor* t, long long (&nb)[3]) {
        if (t)
            for (int d = 0; d < 3; ++d) nb[d] = t->nb[d + 1] / (t->type == SDB_TYPE_F16 ? 2 : 4);
    };
    a.x = x ? x->data : nullptr;
    a.y = y ? y->data : nullptr;
    a.h = h ? h->data : nullptr;
    a.out = out ? out->data : nullptr;
    strides(x, a.xnb);
    strides(y, a.ynb);
    strides(h, a.hnb);
    strides(out, a.onb);
    a.ne1 = ref->ne[1];
    a.ne2 = ref->ne[2];
    a.rows = static_cast<long long>(rows);
    a.c = static_cast<int>(ref->ne[0]);
    a.keep = p->keep;
    a.scale = p->scale;
    auto form = [](const sdb_norm_form& n) { return NormForm{n.kind, n.eps, n.weight, n.bias}; };
    a.post = form(p->post);
    a.pre = form(p->pre);
    auto operand = [](const sdb_operand& o) {
        Operand k{o.data, {0, 0, 0, 0}};
        for (int d = 0; d < 4; ++d) k.nb[d] = o.nb[d];
        return k;
    };
    a.gate = operand(p->gate);
    a.mul = operand(p->mul);
    a.add = operand(p->add);

    // The stream's type (x and h) and the block's (y and out).
    const sdb_tensor* tx = x ? x : h;
    const sdb_tensor* ty = y ? y : out;
    const bool xh = tx && tx->type == SDB_TYPE_F16, yh = ty && ty->type == SDB_TYPE_F16;
    const auto st = static_cast<cudaStream_t>(stream);
    bool vec = a.c % 4 == 0;
    for (const sdb_tensor* t : {x, y, h, out}) {
        if (t == nullptr) continue;
        const int64_t run = t->type == SDB_TYPE_F16 ? 8 : 16;
        if (reinterpret_cast<uintptr_t>(t->data) % run != 0) vec = false;
        for (int d = 1; d < 4; ++d)
            if (t->ne[d] > 1 && t->nb[d] % run != 0) vec = false;
    }
    if (xh && yh) launch<__half, __half>(a, vec, st);
    else if (xh) launch<__half, float>(a, vec, st);
    else if (yh) launch<float, __half>(a, vec, st);
    else launch<float, float>(a, vec, st);
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}
