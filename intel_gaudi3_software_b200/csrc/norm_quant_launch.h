// What the translation units of the row kernels share: the launch itself, and the launchers of the instantiations
// (norm_quant_inst.cu, compiled once per element types and alignment so that the library builds in parallel).
#pragma once
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

// Threads of a gradient block that works on one row at a time; rows of up to 1024 columns take a warp each, four to a block.
inline uint32_t grad_threads(uint32_t cols) { return cols <= 1024 ? 128 : cols <= 8192 ? 32 * ((cols + 1023) / 1024) : 1024; }

template <int XT, int RT, bool SHIFT>
cudaError_t norm_of(const RowLaunch& env, const NormParams& p);
template <int XT, bool DSUM, bool SHIFT>
cudaError_t norm_grad_of(const RowLaunch& env, const NormGradParams& p, uint32_t blocks);
template <int XT, bool SHIFT>
cudaError_t quant_trans_of(const RowLaunch& env, const QuantTransParams& p, int* launches);

}  // namespace mmeb200
