// The launches of q4_rows.cuh's kernel for one group size, with minima or without (a translation unit each: q4_rows_*.cu).
#pragma once

#include <algorithm>
#include <atomic>

#include "q4_rows.cuh"
#include "runtime.cuh"

namespace sdb {

template <class F, int G, bool MINIMA>
int q4_launch_form(const Q4Args& args, const Q4Plan& p, cudaStream_t st) {
    auto kern = q4_rows_kernel<F, G, MINIMA>;
    // The kernel's shared-memory limit is raised once on each device (it costs about as much as a launch).
    static std::atomic<uint64_t> raised{0};
    int dev = 0;
    SDB_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !(raised.load(std::memory_order_relaxed) >> dev & 1)) {
        SDB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kQ4MaxShared));
        if (dev < 64) raised.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    Q4Args a = args;
    const int fixed = q4_fixed_bytes<F>(1024 + 4096 / G * (MINIMA ? 2 : 1));
    const int block = F::block_bytes(std::min(a.rows, F::kTokens), MINIMA ? 128 / G : 0);
    const int fit = (p.shared - fixed) / block;  // k-blocks of x that fit
    // All of a CTA's k-blocks of x are held where a cluster of up to eight brings them down to what fits: else x is
    // split again for every tile (28672 -> 8192, one row: two CTAs 33 us, one 66).  The CTAs then stand for warps that
    // share a tile, but for two (four rows: two 96 us, one 112).
    int wk_log = p.wk_log, cluster_log = p.cluster_log;
    while (cluster_log < 3 && ((a.kblocks - 1) >> cluster_log) + 1 > fit) {
        ++cluster_log;
        if (wk_log > 1) --wk_log;
    }
    const int cluster = 1 << cluster_log;
    a.cluster_log = static_cast<uint8_t>(cluster_log);
    a.range = (a.kblocks + cluster - 1) / cluster;
    while ((1 << wk_log) > F::kWarps || (wk_log > 0 && (1 << wk_log) > fit)) --wk_log;
    const int wk = 1 << wk_log, wr = F::kWarps / wk;
    if (fit < wk) return fail(SDB_CUDA_ERROR, "mul_mat_q4: shared memory");
    a.wk_log = static_cast<uint8_t>(wk_log);
    a.wr_log = 0;
    while ((1 << a.wr_log) < wr) ++a.wr_log;
    // The k-blocks of x held at a time: all of the CTA's, or the multiple of WK that fits.
    a.chunk = std::min(a.range, a.range <= fit ? a.range : fit / wk * wk);
    a.groups = (a.tiles + wr - 1) / wr;
    const int blocks = std::min(a.groups, std::max(1, current_sm_count() / cluster)) * cluster;
    const int runs = (a.rows + F::kTokens - 1) / F::kTokens;  // of x's rows
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(runs));
    cfg.blockDim = dim3(q4_threads<F>());
    cfg.dynamicSmemBytes = static_cast<size_t>(fixed + a.chunk * block);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    SDB_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
    count_launch();
    return SDB_OK;
}

template <bool GATED, int G, bool MINIMA>
int q4_launch_rows(const Q4Args& a, const Q4Plan& p, cudaStream_t st) {
    if (p.form == 1) return q4_launch_form<Q4Digits<GATED>, G, MINIMA>(a, p, st);
    if (p.form == 2) return q4_launch_form<Q4Pairs<1, GATED>, G, MINIMA>(a, p, st);
    if (p.form == 4) return q4_launch_form<Q4Pairs<2, GATED>, G, MINIMA>(a, p, st);
    if (p.form == 8)
        return a.x_half ? q4_launch_form<Q4Floats<1, true, GATED>, G, MINIMA>(a, p, st)
                        : q4_launch_form<Q4Floats<1, false, GATED>, G, MINIMA>(a, p, st);
    if (!a.x_half) return q4_launch_form<Q4Floats<2, false, GATED>, G, MINIMA>(a, p, st);
    if (p.form == 16) return q4_launch_form<Q4Floats<2, true, GATED>, G, MINIMA>(a, p, st);
    return q4_launch_form<Q4Floats<4, true, GATED>, G, MINIMA>(a, p, st);
}

template <int G, bool MINIMA>
int q4_launch(const Q4Args& a, const Q4Plan& p, cudaStream_t st) {
    return a.gate ? q4_launch_rows<true, G, MINIMA>(a, p, st) : q4_launch_rows<false, G, MINIMA>(a, p, st);
}

}  // namespace sdb
