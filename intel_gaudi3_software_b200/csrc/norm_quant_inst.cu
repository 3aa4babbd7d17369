// Instantiations of the row kernels and their launchers. The Makefile compiles this file once per variant with -DINST_XT=<1|2>
// -DINST_SHIFT=<0|1> (element type of x, rows at any alignment) and one of -DINST_NORM=<0|1|2> (element type of the residual),
// -DINST_GRAD=<0|1> (with a gradient of the sum) and -DINST_TRANS.
#include <algorithm>

#include "norm_quant.cuh"
#include "norm_quant_launch.h"

namespace mmeb200 {

#if defined(INST_NORM)

// Short rows take one warp each. Aligned rows are kept in registers, at most four pieces of eight elements to a lane: few enough
// for registers, enough for the loads in flight to cover the latency of HBM and for the row's reduction to be a small part of
// the work. Longer rows, and rows at any alignment, are kept in shared memory.
template <int XT, int RT, bool SHIFT>
cudaError_t norm_of(const RowLaunch& env, const NormParams& p) {
    const dim3 warps((p.rows + 3) / 4), blocks(p.rows);
    if (p.cols <= 256) return launch_rows(env, norm_kernel<XT, RT, SHIFT, 1, false, 128>, p, warps, 128, 0);
    if constexpr (!SHIFT) {
        if (p.cols <= 1024) return launch_rows(env, norm_kernel<XT, RT, SHIFT, 4, false, 128>, p, warps, 128, 0);
        if (p.cols <= 16384) return launch_rows(env, norm_kernel<XT, RT, SHIFT, 4, true, 512>, p, blocks, 32 * ((p.cols + 1023) / 1024), 0);
    }
    // a warp for every 1024 columns, at most 16 of them
    const unsigned threads = std::min(512u, 32 * ((p.cols + 1023) / 1024));
    const size_t keep = size_t((p.cols + threads * 8 - 1) / (threads * 8)) * threads * 8 * RowElem<RowKept<XT, RT>::kType>::kBytes;
    if (keep <= 200 * 1024) {
        static bool done[64] = {};
        if (!done[env.device & 63]) {
            const cudaError_t e = cudaFuncSetAttribute(norm_loop_kernel<XT, RT, SHIFT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
            if (e != cudaSuccess) return e;
            done[env.device & 63] = true;
        }
        return launch_rows(env, norm_loop_kernel<XT, RT, SHIFT>, p, blocks, threads, keep);
    }
    return launch_rows(env, norm_long_kernel<XT, RT, SHIFT>, p, blocks, 1024, 0);
}
template cudaError_t norm_of<INST_XT, INST_NORM, INST_SHIFT != 0>(const RowLaunch&, const NormParams&);

#elif defined(INST_GRAD)

template <int XT, bool DSUM, bool SHIFT>
cudaError_t norm_grad_of(const RowLaunch& env, const NormGradParams& p, uint32_t blocks) {
    const dim3 g(blocks);
    const unsigned threads = grad_threads(p.cols);
    const size_t sums = p.cols <= 1024 ? p.cols * sizeof(float) : 0;
    if (p.cols <= 256) return launch_rows(env, norm_grad_kernel<XT, DSUM, SHIFT, 1, false, 128>, p, g, threads, sums);
    if (p.cols <= 1024) return launch_rows(env, norm_grad_kernel<XT, DSUM, SHIFT, 4, false, 128>, p, g, threads, sums);
    if (p.cols <= 8192) return launch_rows(env, norm_grad_kernel<XT, DSUM, SHIFT, 4, true, 256>, p, g, threads, 0);
    return launch_rows(env, norm_grad_long_kernel<XT, DSUM, SHIFT>, p, g, threads, 0);
}
template cudaError_t norm_grad_of<INST_XT, INST_GRAD != 0, INST_SHIFT != 0>(const RowLaunch&, const NormGradParams&, uint32_t);

#elif defined(INST_TRANS)

struct ColumnSteps { float* scale; uint32_t cols; float top; };
static __global__ void __launch_bounds__(256) column_steps_kernel(const __grid_constant__ ColumnSteps p) { column_steps(p.scale, p.cols, p.top); }

template <int XT, bool SHIFT>
cudaError_t quant_trans_of(const RowLaunch& env, const QuantTransParams& p, int* launches) {
    cudaError_t e = cudaSuccess;
    if (!p.given) {
        e = cudaMemsetAsync(p.scale, 0, size_t(p.cols) * sizeof(float), env.stream);
        if (e != cudaSuccess) return e;
        // strips of 256 columns, cut along the rows into about eight blocks per SM, of at least 32 rows
        const uint32_t strips = (p.cols + 255) / 256, want = (uint32_t(env.sm_count) * 8 + strips - 1) / strips;
        const uint32_t cuts = std::max(1u, std::min((p.rows + 31) / 32, std::min(want, 65535u)));
        e = launch_rows(env, column_max_kernel<XT, SHIFT>, p, dim3(strips, cuts), 256, 0);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    // columns in x, rows in y (at most 65535 blocks of tiles at a time)
    constexpr uint32_t kRows = kTransTiles * 128;
    void (*kern)(QuantTransParams) = p.out_type == ROW_I8 ? (p.given ? quant_trans_kernel<XT, SHIFT, true, true> : quant_trans_kernel<XT, SHIFT, true, false>)
                                                          : (p.given ? quant_trans_kernel<XT, SHIFT, false, true> : quant_trans_kernel<XT, SHIFT, false, false>);
    for (uint64_t r = 0; r < p.rows; r += uint64_t(65535) * kRows) {
        QuantTransParams q = p;
        q.row0 = uint32_t(r);
        q.rows = uint32_t(std::min<uint64_t>(p.rows - r, uint64_t(65535) * kRows));
        e = launch_rows(env, kern, q, dim3((p.cols + 63) / 64, (q.rows + kRows - 1) / kRows), 256, 0);
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
template cudaError_t quant_trans_of<INST_XT, INST_SHIFT != 0>(const RowLaunch&, const QuantTransParams&, int*);

#endif

}  // namespace mmeb200
