// Instantiations of the row kernels and their launchers. The Makefile compiles this file once per variant with -DINST_XT=<1|2>
// -DINST_VEC=<8|0|1> (element type of x, how rows lie: 0 is kPhased) and one of -DINST_NORM=<0|1|2> (element type of the residual),
// -DINST_GRAD=<0|1> (with a gradient of the sum) and -DINST_TRANS.
#include <algorithm>
#include <atomic>

#include "norm_quant.cuh"
#include "norm_quant_launch.h"

namespace mmeb200 {

#if defined(INST_NORM)

// Short rows take one warp each. At most 32 elements of a row per thread, 64 of the longest: few enough for registers, enough for
// the loads in flight to cover the latency of HBM and for the row's reduction to be a small part of the work.
template <int XT, int RT, int VEC>
cudaError_t norm_of(const RowLaunch& env, const NormParams& p) {
    const uint32_t cols = p.cols + (VEC == kPhased ? 7 : 0);   // as far as a row may reach
    const dim3 warps((p.rows + 3) / 4), blocks(p.rows);
    if (cols <= 256) return launch_rows(env, norm_kernel<XT, RT, VEC, 1, false, 128>, p, warps, 128, 0);
    if (cols <= 1024) return launch_rows(env, norm_kernel<XT, RT, VEC, 4, false, 128>, p, warps, 128, 0);
    if (cols <= 16384) return launch_rows(env, norm_kernel<XT, RT, VEC, 4, true, 512>, p, blocks, 32 * ((cols + 1023) / 1024), 0);
    if (cols <= 32768) return launch_rows(env, norm_kernel<XT, RT, VEC, 8, true, 512>, p, blocks, 32 * ((cols + 2047) / 2048), 0);
    return launch_rows(env, norm_long_kernel<XT, RT, VEC>, p, blocks, 1024, 0);
}
template cudaError_t norm_of<INST_XT, INST_NORM, INST_VEC>(const RowLaunch&, const NormParams&);

#elif defined(INST_GRAD)

template <int XT, bool DSUM, int VEC, int NV>
size_t grad_smem_bytes(const GradShape& shape, uint32_t cols) {
    using Pieces = GradPieces<XT, DSUM, VEC, NV>;
    return (Pieces::kFetched ? size_t(2) * Pieces::kTensors * NV * 16 * shape.threads : 0) + (shape.form == GRAD_WARP ? size_t(cols) * sizeof(float) : 0);
}
template <int XT, bool DSUM, int VEC, int NV, int FORM, int THREADS>
cudaError_t launch_grad(const RowLaunch& env, const NormGradParams& p, uint32_t blocks, const GradShape& shape) {
    const auto kern = norm_grad_kernel<XT, DSUM, VEC, NV, FORM, THREADS>;
    const size_t smem = grad_smem_bytes<XT, DSUM, VEC, NV>(shape, p.cols);
    static std::atomic<bool> done[64] = {};   // (two contexts may meet here on two threads)
    if (smem > 40 * 1024 && !done[env.device & 63]) {   // (48 KB with the static shared memory need no leave)
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
        if (e != cudaSuccess) return e;
        done[env.device & 63] = true;
    }
    return launch_rows(env, kern, p, dim3(blocks * shape.ranks), shape.threads, smem, shape.ranks);
}
template <int XT, bool DSUM, int VEC>
cudaError_t norm_grad_of(const RowLaunch& env, const NormGradParams& given, uint32_t blocks) {
    NormGradParams p = given;
    const GradShape shape = grad_shape(p.cols);
    p.ranks = shape.ranks;
    if (shape.form == GRAD_WARP && p.cols + (p.cols % 8 ? 7 : 0) <= 256) return launch_grad<XT, DSUM, VEC, 1, GRAD_WARP, 128>(env, p, blocks, shape);
    if (shape.form == GRAD_WARP) return launch_grad<XT, DSUM, VEC, 4, GRAD_WARP, 128>(env, p, blocks, shape);
    if (shape.form == GRAD_BLOCK) return launch_grad<XT, DSUM, VEC, 4, GRAD_BLOCK, 256>(env, p, blocks, shape);
    if (shape.form == GRAD_CLUSTER) return launch_grad<XT, DSUM, VEC, 4, GRAD_CLUSTER, 256>(env, p, blocks, shape);
    return launch_rows(env, norm_grad_loop_kernel<XT, DSUM, VEC>, p, dim3(blocks), shape.threads, 0);
}
template cudaError_t norm_grad_of<INST_XT, INST_GRAD != 0, INST_VEC>(const RowLaunch&, const NormGradParams&, uint32_t);

#if INST_XT == 1 && INST_GRAD == 1 && INST_VEC == 8
// Of the form that needs most shared memory; all have the same registers.
bool norm_grad_clusters(uint32_t ranks, uint32_t threads, int* n) {
    const auto kern = norm_grad_kernel<ROW_BF16, true, 8, 4, GRAD_CLUSTER, 256>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024) != cudaSuccess) return false;
    GradShape shape{GRAD_CLUSTER, threads, 1, 1, ranks};
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ranks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(ranks * 64);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = grad_smem_bytes<ROW_BF16, true, 8, 4>(shape, 0);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaOccupancyMaxActiveClusters(n, kern, &cfg) == cudaSuccess;
}
#endif

#elif defined(INST_TRANS)

struct ColumnSteps { float* scale; uint32_t cols; float top; };
static __global__ void __launch_bounds__(256) column_steps_kernel(const __grid_constant__ ColumnSteps p) { column_steps(p.scale, p.cols, p.top); }

template <int XT, int VEC>
cudaError_t quant_trans_of(const RowLaunch& env, const QuantTransParams& p, int* launches) {
    cudaError_t e = cudaSuccess;
    if (!p.given) {
        e = cudaMemsetAsync(p.scale, 0, size_t(p.cols) * sizeof(float), env.stream);
        if (e != cudaSuccess) return e;
        // strips of 256 columns, cut along the rows into as many blocks as the SMs hold at once, of at least 32 rows
        const uint32_t strips = (p.cols + kTransCols<VEC> - 1) / kTransCols<VEC>, held = uint32_t(env.sm_count) * (XT == ROW_BF16 ? 6 : 4);
        const uint32_t cuts = std::max(1u, std::min((p.rows + 31) / 32, held / strips));
        e = launch_rows(env, column_max_kernel<XT, VEC>, p, dim3(strips, cuts), 256, 0);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    // columns in x, rows in y (at most 65535 blocks of tiles at a time)
    constexpr uint32_t kRows = kTransRows;
    void (*kern)(QuantTransParams) = p.out_type == ROW_I8 ? (p.given ? quant_trans_kernel<XT, VEC, true, true> : quant_trans_kernel<XT, VEC, true, false>)
                                                          : (p.given ? quant_trans_kernel<XT, VEC, false, true> : quant_trans_kernel<XT, VEC, false, false>);
    for (uint64_t r = 0; r < p.rows; r += uint64_t(65535) * kRows) {
        QuantTransParams q = p;
        q.row0 = uint32_t(r);
        q.rows = uint32_t(std::min<uint64_t>(p.rows - r, uint64_t(65535) * kRows));
        e = launch_rows(env, kern, q, dim3((p.cols + kTransCols<VEC> - 1) / kTransCols<VEC>, (q.rows + kRows - 1) / kRows), 256, 0);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    if (!p.given) {
        const ColumnSteps s{p.scale, p.cols, p.top};
        e = launch_rows(env, column_steps_kernel, s, dim3((p.cols + 255) / 256), 256, 0);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    return cudaSuccess;
}
template cudaError_t quant_trans_of<INST_XT, INST_VEC>(const RowLaunch&, const QuantTransParams&, int*);

#endif

}  // namespace mmeb200
