// What the translation units of the row kernels share: the launch itself, and the launchers of the instantiations
// (norm_quant_inst.cu, compiled once per element types and alignment so that the library builds in parallel).
#pragma once
#include <algorithm>
#include <cstring>

#include "norm_quant.h"

namespace mmeb200 {

template <typename P>
inline cudaError_t launch_rows(const RowLaunch& env, void (*kern)(P), const P& p, dim3 grid, unsigned threads, size_t smem) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = env.stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = env.dependent_launch ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// The gradient's form and shape: a function of the columns and the type, so that its workspace can be asked for.
enum : int { GRAD_WARP, GRAD_BLOCK, GRAD_LOOP, GRAD_REREAD };
struct GradShape {
    int form;
    uint32_t threads, steps, rows_per_block, blocks_per_sm;   // steps: of 256 columns per warp
    size_t smem;
};
constexpr int kGradSmem = 220 * 1024;
inline GradShape grad_shape(uint32_t row_cols, bool fp32) {
    const uint32_t cols = row_cols % 8 ? row_cols + 7 : row_cols;   // with room for a phase
    if (cols <= 1024) return {GRAD_WARP, 128, cols <= 256 ? 1u : 4u, 4, 4, row_cols * sizeof(float)};
    if (cols <= 8192) {
        const uint32_t threads = 32 * ((cols + 1023) / 1024);
        return {GRAD_BLOCK, threads, 4, 1, std::max(1u, 512u / threads), 0};
    }
    const uint32_t steps = (cols + 16 * 256 - 1) / (16 * 256);
    const uint64_t smem = uint64_t(512) * steps * 8 * ((fp32 ? 8 : 4) + 4);   // x and dy, the sums of dgamma
    if (smem <= kGradSmem) return {GRAD_LOOP, 512, steps, 1, smem <= kGradSmem / 2 ? 2u : 1u, size_t(smem)};
    return {GRAD_REREAD, 512, steps, 1, 2, 0};
}

template <int XT, int RT, int VEC>
cudaError_t norm_of(const RowLaunch& env, const NormParams& p);
template <int XT, bool DSUM, int VEC>
cudaError_t norm_grad_of(const RowLaunch& env, const NormGradParams& p, uint32_t blocks);
template <int XT, int VEC>
cudaError_t quant_trans_of(const RowLaunch& env, const QuantTransParams& p, int* launches);

}  // namespace mmeb200
