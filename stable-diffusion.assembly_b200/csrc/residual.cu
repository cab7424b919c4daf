// The residual block of a transformer in one pass over its rows:
//   h   = keep x + scale gate post(y)
//   out = pre(h) (1 + mul) + add
// post and pre are nothing, a LayerNorm or an RMS norm of the row; gate, mul
// and add are operands of the output's extents or broadcast along any of them.
//
// A CTA per row. The mean of a LayerNorm comes from a first sum, the variance
// from the sum of d^2 about that float mean less the square of d's own mean
// (d = v - mean), so that rows far from 0 lose nothing. Sums are FP32 in a
// thread (a thread's share of a row) and across threads.
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
    const float var = fmaxf(t.y * inv - s.shift * s.shift, 0.0f);
    s.rstd = 1.0f / sqrtf(var + n.eps);
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
    const int blocks = static_cast<int>(std::min<long long>(a.rows, 148LL * 32));
    if (xh && yh) residual_rows_kernel<__half, __half><<<blocks, kRowThreads, 0, st>>>(a);
    else if (xh) residual_rows_kernel<__half, float><<<blocks, kRowThreads, 0, st>>>(a);
    else if (yh) residual_rows_kernel<float, __half><<<blocks, kRowThreads, 0, st>>>(a);
    else residual_rows_kernel<float, float><<<blocks, kRowThreads, 0, st>>>(a);
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}
