// Linear layers of a few rows with 4-bit weights (q4.cuh), plain and gated:
//   y[m][n] = sum_k x[m][k] W[n][k], then the chain;
//   gated: out[m][j] = a[m][j] act(b[m][j]) of two such products.
//
// The kernel and its forms are in q4_rows.cuh; here are the checks and the plan.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/sdb.h"
#include "chain.cuh"
#include "q4.cuh"
#include "q4_rows.cuh"
#include "runtime.cuh"

namespace sdb {

namespace {

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
    // A grid's second dimension counts runs of rows; each extent on its own first, so that no product overflows.
    const int64_t limit = 1LL << 20;
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

// Cuts the product: the rows of x a CTA takes (a form), the warps and CTAs that share a tile's k-blocks.
//
// With up to four rows x is cheap and the weights are all: eight warps share a tile, so that a round is a long
// run of memory (8192 -> 28672, one row: 33.0 us; four warps 35.0, sixteen 34.9).  Up to eight rows likewise (five
// rows 72; four CTAs and one warp 130), but where a CTA walks one or two tiles' groups the splitting of FP32 rows is
// what it does: the CTAs of a cluster split them between them (8 rows of 4096 -> 4096: four CTAs 11.3, one 12.1; of
// FP16 8.9 and 8.0).  So do those of more rows, with one warp a tile (16 rows of 4096 -> 4096: four CTAs 14.9, one
// 21.9).  Short rows are no cluster's (1280 -> 20160, 16 rows: one CTA and one warp a tile 24.6, two warps 26.4, two
// CTAs 28.4; 8 rows: four warps 17.1, eight 17.5), and two matrices, whose sums take the registers, share less
// (1280 -> 5120, 5 rows: two warps 11.7, one 12.3, eight 12.9; 16 rows at a time: 16 rows with two warps, 32 with one
// 29.8, with two 36.8).  FP32 rows, three columns each, are taken 16 at a time, FP16 rows 32 (4096 -> 4096: 32 FP32
// rows 22.1 us, taken at once 43.5, 77 rows 64.6 and 92.9; 77 FP16 rows 41.5); but 9 to 16 FP32 rows of two long
// matrices in two runs of eight, whose CTAs hold more of x (4096 -> 11008: 16 rows 62 us, at once 77).  And where the tiles leave most SMs
// idle, more warps share one (320 -> 1280, two rows: sixteen 4.3 us, eight 4.7).
Q4Plan plan(const Q4Args& a) {
    Q4Plan p{};
    const bool gated = a.gate != nullptr;
    p.form = a.rows == 1 ? 1 : a.rows <= 4 && !a.x_half ? (a.rows + 1) / 2 * 2 : a.rows <= 8 ? 8 : a.rows <= 16 || !a.x_half ? 16 : 32;
    if (p.form == 16 && gated && !a.x_half && a.rows <= 16 && a.kblocks >= 16) p.form = 8;
    p.shared = kQ4MaxShared;
    const int warps = p.form <= 16 && !gated ? 16 : 8, runs = (a.rows + p.form - 1) / p.form;
    if (p.form <= 4) {
        p.wk_log = 3;
    } else if (p.form == 8) {
        if (a.kblocks < 16) p.wk_log = gated ? 1 : 2;
        else if (a.x_half || gated || a.tiles > 2 * current_sm_count()) p.wk_log = runs > 1 ? 2 : 3;
        else p.cluster_log = 2;
    } else if (a.kblocks >= 16) {
        p.cluster_log = gated ? 1 : 2;
    } else {
        p.wk_log = gated && p.form == 16 && runs == 1 ? 1 : 0;
    }
    while ((warps >> p.wk_log) > 1 &&
           (static_cast<long long>(a.tiles / (warps >> p.wk_log)) << p.cluster_log) * runs < current_sm_count() / 2)
        ++p.wk_log;
    return p;
}

int run(const sdb_q4* w, const sdb_q4* gate, const sdb_tensor* x, const sdb_tensor* dst, int act,
        const sdb_chain* chain, cudaStream_t st) {
    const Q4View v = q4_view(w);
    Q4Args a{};
    a.w = v.data;
    a.gate = gate ? static_cast<const uint8_t*>(gate->data) : nullptr;
    a.tiles = v.tiles;
    a.kblocks = v.kblocks;
    a.k = static_cast<int>(v.k);
    a.n = static_cast<int>(v.n);
    a.x = x->data;
    a.y = chain && chain->redirect ? chain->redirect : dst->data;
    a.x_half = x->type == SDB_TYPE_F16;
    const int es = a.x_half ? 2 : 4;
    a.y_half = dst->type == SDB_TYPE_F16;
    a.x_vec = reinterpret_cast<uintptr_t>(x->data) % (4 * es) == 0;
    for (int d = 0; d < 3; ++d) {
        a.xnb[d] = x->nb[d + 1] / es;
        a.ynb[d] = dst->nb[d + 1] / (a.y_half ? 2 : 4);
        if (x->ne[d + 1] > 1 && a.xnb[d] % 4 != 0) a.x_vec = 0;
    }
    a.ne1 = static_cast<int>(x->ne[1]);
    a.ne2 = static_cast<int>(x->ne[2]);
    a.flat = x->ne[2] == 1 && x->ne[3] == 1;
    a.rows = static_cast<int>(x->ne[1] * x->ne[2] * x->ne[3]);
    a.act = act;
    a.err = device_error_word();
    a.chain = make_chain(chain);
    if (a.rows == 0) return SDB_OK;
    const Q4Plan p = plan(a);
    if (w->minimum) {
        if (w->group == 32) return q4_launch<32, true>(a, p, st);
        return w->group == 64 ? q4_launch<64, true>(a, p, st) : q4_launch<128, true>(a, p, st);
    }
    if (w->group == 32) return q4_launch<32, false>(a, p, st);
    return w->group == 64 ? q4_launch<64, false>(a, p, st) : q4_launch<128, false>(a, p, st);
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
