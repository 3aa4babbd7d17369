// What the translation units of the row kernels share: the launch itself, and the launchers of the instantiations
// (norm_quant_inst.cu, compiled once per element types and alignment so that the library builds in parallel).
#pragma once
#include <algorithm>
#include <cstring>

#include "norm_quant.cuh"

namespace mmeb200 {

template <typename P>
inline cudaError_t launch_rows(const RowLaunch& env, void (*kern)(P), const P& p, dim3 grid, unsigned threads, size_t smem, unsigned cluster = 1) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = env.stream;
    cudaLaunchAttribute attrs[2];
    cfg.attrs = attrs;
    if (env.dependent_launch) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[cfg.numAttrs].val.clusterDim.x = cluster;
        attrs[cfg.numAttrs].val.clusterDim.y = attrs[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, kern, p);   // (not the thread's last error, which may be an older one of the caller's)
}

// The gradient's form and shape: a function of the columns, so that its workspace can be asked for. A thread takes at most 32
// columns, a block 256 threads; up to eight blocks share a row.
struct GradShape {
    int form;
    uint32_t threads, rows_per_block, blocks_per_sm, ranks;
};
inline GradShape grad_shape(uint32_t row_cols) {
    const uint32_t cols = row_cols % 8 ? row_cols + 7 : row_cols;   // with room for a phase
    if (cols <= 1024) return {GRAD_WARP, 128, 4, 4, 1};
    const uint32_t ranks = (cols + 8191) / 8192, threads = 32 * (((cols + ranks - 1) / ranks + 1023) / 1024);
    if (ranks <= 8) return {ranks == 1 ? GRAD_BLOCK : GRAD_CLUSTER, threads, 1, std::max(1u, 512u / threads), ranks};
    return {GRAD_REREAD, 512, 1, 2, 1};
}

template <int XT, int RT, int VEC>
cudaError_t norm_of(const RowLaunch& env, const NormParams& p);
template <int XT, bool DSUM, int VEC>
cudaError_t norm_grad_of(const RowLaunch& env, const NormGradParams& p, uint32_t blocks);
bool norm_grad_clusters(uint32_t ranks, uint32_t threads, int* n);   // of so many blocks of so many threads that the current device holds at once
template <int XT, int VEC>
cudaError_t quant_trans_of(const RowLaunch& env, const QuantTransParams& p, int* launches);

}  // namespace mmeb200
