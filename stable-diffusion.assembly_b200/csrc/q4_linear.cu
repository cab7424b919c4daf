// Linear layers of a few rows with 4-bit weights (q4.cuh), plain and gated:
//   y[m][n] = sum_k x[m][k] W[n][k], then the chain;
//   gated: out[m][j] = a[m][j] act(b[m][j]) of two such products.
//
// A warp per output column j: the lanes share the row's words, and FP32 sums
// of four rows of x at a time are joined across the lanes.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/sdb.h"
#include "chain.cuh"
#include "q4.cuh"
#include "runtime.cuh"

namespace sdb {

namespace {

struct Q4Args {
    Q4View w, gate;          // gate.codes null: a plain product
    const void* x;
    void* y;
    long long xnb[3], ynb[3];  // strides of rows in elements (dims 1..3)
    long long ne1, ne2;
    long long rows;
    int x_half, y_half, act;
    Chain chain;
};

__device__ __forceinline__ float load_x(const Q4Args& a, long long at) {
    return a.x_half ? __half2float(static_cast<const __half*>(a.x)[at]) : static_cast<const float*>(a.x)[at];
}

// One output element: the chain (columns of the value at n, of the gate at w.n + n), the gate, the store.
__device__ __forceinline__ void finish(const Q4Args& a, long long m, long long n, float v, float g) {
    const long long i1 = m % a.ne1, q = m / a.ne1, i2 = q % a.ne2, i3 = q / a.ne2;
    const long long at = n + i1 * a.ynb[0] + i2 * a.ynb[1] + i3 * a.ynb[2];
    if (a.chain.from_redirect) v += static_cast<const float*>(a.y)[at];
    v = apply_chain(a.chain, v, n, i1, i2, i3);
    if (a.gate.codes) {
        g = apply_chain(a.chain, g, a.w.n + n, i1, i2, i3);
        v *= a.act == SDB_GATE_SILU ? silu(g) : gelu(g);
    }
    if (a.y_half) static_cast<__half*>(a.y)[at] = __float2half_rn(v);
    else static_cast<float*>(a.y)[at] = v;
}

__device__ __forceinline__ void product(const Q4Args& a, const Q4View& w, long long n, long long m0, int rows,
                                        float (&sum)[4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = 0.0f;
    for (long long k0 = lane * 8; k0 < w.k; k0 += 256) {
        const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(w.codes) + q4_word(w, n, k0));
        const long long s = q4_scale(w, n, k0);
        const float d = __half2float(w.scales[s]);
        const float off = w.minima ? fmaf(8.0f, d, __half2float(w.minima[s])) : 0.0f;
        const int cols = static_cast<int>(min(8LL, w.k - k0));
        for (int r = 0; r < rows; ++r) {
            const long long m = m0 + r, i1 = m % a.ne1, q = m / a.ne1;
            const long long at = i1 * a.xnb[0] + q % a.ne2 * a.xnb[1] + q / a.ne2 * a.xnb[2] + k0;
            float p = 0.0f, t = 0.0f;
            for (int c = 0; c < cols; ++c) {
                const float x = load_x(a, at + c);
                p = fmaf(x, static_cast<float>(static_cast<int>(word >> q4_bit(c) & 15u) - 8), p);
                t += x;
            }
            sum[r] = fmaf(d, p, sum[r]);
            if (w.minima) sum[r] = fmaf(off, t, sum[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        for (int o = 16; o; o >>= 1) sum[r] += __shfl_xor_sync(~0u, sum[r], o);
}

__global__ void __launch_bounds__(256) q4_rows_kernel(const Q4Args a) {
    const long long n = blockIdx.x * 8LL + threadIdx.x / 32;
    if (n >= a.w.n) return;
    for (long long m0 = blockIdx.y * 4LL; m0 < a.rows; m0 += gridDim.y * 4LL) {
        const int rows = static_cast<int>(min(4LL, a.rows - m0));
        float v[4], g[4] = {};
        product(a, a.w, n, m0, rows, v);
        if (a.gate.codes) product(a, a.gate, n, m0, rows, g);
        if ((threadIdx.x & 31) == 0)
            for (int r = 0; r < rows; ++r) finish(a, m0 + r, n, v[r], g[r]);
    }
}

bool activation(const sdb_tensor* t) {
    if (t == nullptr || (t->type != SDB_TYPE_F32 && t->type != SDB_TYPE_F16)) return false;
    const int64_t es = t->type == SDB_TYPE_F16 ? 2 : 4;
    for (int d = 0; d < 4; ++d)
        if (t->ne[d] < 0 || t->nb[d] < 0 || t->nb[d] % es != 0) return false;
    return (t->nb[0] == es || t->ne[0] == 1) && reinterpret_cast<uintptr_t>(t->data) % es == 0;
}

bool product_shapes(const sdb_q4* w, const sdb_tensor* x, const sdb_tensor* dst) {
    if (!q4_valid(w) || !activation(x) || !activation(dst)) return false;
    if (x->ne[0] != w->k || dst->ne[0] != w->n) return false;
    for (int d = 1; d < 4; ++d)
        if (dst->ne[d] != x->ne[d] || (dst->ne[d] > 1 && dst->nb[d] == 0)) return false;
    // Rows as 32-bit numbers; each extent on its own first, so that the product cannot overflow.
    const int64_t limit = 1LL << 30;
    if (x->ne[1] > limit || x->ne[2] > limit || x->ne[3] > limit) return false;
    const double rows = static_cast<double>(x->ne[1]) * x->ne[2] * x->ne[3];
    if (rows > static_cast<double>(limit)) return false;
    return rows == 0 || (x->data != nullptr && dst->data != nullptr);
}

bool chain_ok(const sdb_chain* c, const sdb_tensor* dst, bool gated) {
    if (c == nullptr) return true;
    if (c->count < 0 || c->count > SDB_MAX_STEPS) return false;
    for (int s = 0; s < c->count; ++s) {
        const int k = c->steps[s].kind;
        if (k != SDB_STEP_ADD && k != SDB_STEP_MUL && k != SDB_STEP_SILU) return false;
        if (k != SDB_STEP_SILU && c->steps[s].operand == nullptr) return false;
        if (c->from_redirect && k != SDB_STEP_ADD) return false;
    }
    if (c->from_redirect && c->redirect == nullptr) return false;
    return c->redirect == nullptr || (!gated && dst->type == SDB_TYPE_F32);
}

int run(const sdb_q4* w, const sdb_q4* gate, const sdb_tensor* x, const sdb_tensor* dst, int act,
        const sdb_chain* chain, cudaStream_t st) {
    Q4Args a{};
    a.w = q4_view(w);
    if (gate) a.gate = q4_view(gate);
    a.x = x->data;
    a.y = chain && chain->redirect ? chain->redirect : dst->data;
    a.x_half = x->type == SDB_TYPE_F16;
    a.y_half = dst->type == SDB_TYPE_F16;
    for (int d = 0; d < 3; ++d) {
        a.xnb[d] = x->nb[d + 1] / (a.x_half ? 2 : 4);
        a.ynb[d] = dst->nb[d + 1] / (a.y_half ? 2 : 4);
    }
    a.ne1 = x->ne[1];
    a.ne2 = x->ne[2];
    a.rows = x->ne[1] * x->ne[2] * x->ne[3];
    a.act = act;
    a.chain = make_chain(chain);
    if (a.rows == 0) return SDB_OK;
    const dim3 grid(static_cast<unsigned>((w->n + 7) / 8), static_cast<unsigned>(std::min<long long>((a.rows + 3) / 4, 65535)));
    q4_rows_kernel<<<grid, 256, 0, st>>>(a);
    count_launch();
    SDB_CUDA(cudaGetLastError());
    return SDB_OK;
}

}  // namespace

}  // namespace sdb

using namespace sdb;

extern "C" {

int sdb_mul_mat_q4_supported(const sdb_q4* w, const sdb_tensor* x, const sdb_tensor* dst) {
    return product_shapes(w, x, dst) ? 1 : 0;
}

int sdb_mul_mat_q4(const sdb_q4* w, const sdb_tensor* x, const sdb_tensor* dst, const sdb_chain* chain,
                   void* stream) {
    if (!product_shapes(w, x, dst)) return fail(SDB_NOT_SUPPORTED, "sdb_mul_mat_q4: shapes not supported");
    if (!chain_ok(chain, dst, false)) return fail(SDB_INVALID, "sdb_mul_mat_q4: invalid chain");
    return run(w, nullptr, x, dst, 0, chain, static_cast<cudaStream_t>(stream));
}

int sdb_mul_mat_q4_gated_supported(const sdb_q4* w, const sdb_q4* gate, const sdb_tensor* x, const sdb_tensor* out) {
    if (!product_shapes(w, x, out) || !q4_valid(gate)) return 0;
    return w->k == gate->k && w->n == gate->n && w->group == gate->group && w->minimum == gate->minimum;
}

int sdb_mul_mat_q4_gated(const sdb_q4* w, const sdb_q4* gate, const sdb_tensor* x, const sdb_tensor* out,
                         int32_t act, const sdb_chain* chain, void* stream) {
    if (!sdb_mul_mat_q4_gated_supported(w, gate, x, out))
        return fail(SDB_NOT_SUPPORTED, "sdb_mul_mat_q4_gated: shapes not supported");
    if (act != SDB_GATE_GELU && act != SDB_GATE_SILU)
        return fail(SDB_INVALID, "sdb_mul_mat_q4_gated: act is SDB_GATE_GELU or SDB_GATE_SILU");
    if (!chain_ok(chain, out, true)) return fail(SDB_INVALID, "sdb_mul_mat_q4_gated: invalid chain");
    return run(w, gate, x, out, act, chain, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
