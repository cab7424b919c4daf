// The launches of q4_rows.cuh's kernel for one group size (a translation unit each: q4_rows_*.cu).
#pragma once

#include <atomic>

#include "q4_rows.cuh"
#include "runtime.cuh"

namespace sdb {

template <int T, bool PAIRED, bool HALF, bool GATED, int G>
int q4_launch_form(const Q4Args& a, const Q4Plan& p, cudaStream_t st) {
    using S = Q4Shape<T, PAIRED, HALF, GATED>;
    auto kern = q4_rows_kernel<T, PAIRED, HALF, GATED, G>;
    const int bytes = S::fixed_bytes() + a.chunk * S::block_bytes(a.rows < S::kTokens ? a.rows : S::kTokens, 128 / G);
    // The kernel's shared-memory limit is raised once on each device (it costs about as much as a launch).
    static std::atomic<uint64_t> raised{0};
    int dev = 0;
    SDB_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !(raised.load(std::memory_order_relaxed) >> dev & 1)) {
        SDB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kQ4MaxShared));
        if (dev < 64) raised.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.blocks), static_cast<unsigned>(p.chunks));
    cfg.blockDim = dim3(kQ4Threads);
    cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(a.cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = a.cluster > 1 ? 1 : 0;
    SDB_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
    count_launch();
    return SDB_OK;
}

template <bool HALF, bool GATED, int G>
int q4_launch_rows(const Q4Args& a, const Q4Plan& p, cudaStream_t st) {
    if constexpr (!HALF)
        if (p.form == 0) return q4_launch_form<1, true, HALF, GATED, G>(a, p, st);
    if (p.form <= 1) return q4_launch_form<1, false, HALF, GATED, G>(a, p, st);
    if (p.form == 2) return q4_launch_form<2, false, HALF, GATED, G>(a, p, st);
    return q4_launch_form<4, false, HALF, GATED, G>(a, p, st);
}

template <int G>
int q4_launch(const Q4Args& a, const Q4Plan& p, bool half, cudaStream_t st) {
    const bool gated = a.gate.codes != nullptr;
    if (half) return gated ? q4_launch_rows<true, true, G>(a, p, st) : q4_launch_rows<true, false, G>(a, p, st);
    return gated ? q4_launch_rows<false, true, G>(a, p, st) : q4_launch_rows<false, false, G>(a, p, st);
}

}  // namespace sdb
