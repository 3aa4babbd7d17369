// Launchers of the row kernels (norm_quant.cuh): the instantiation for a row's length, types and alignment.
#include "norm_quant.cuh"

#include <algorithm>
#include <cstring>

namespace mmeb200 {

template <typename P>
static cudaError_t launch_rows(const RowLaunch& env, void (*kern)(P), const P& p, dim3 grid, unsigned threads, size_t smem) {
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

// A row's elements are spread over T threads with at most 32 of them per thread: few enough for registers, enough for
// the loads in flight to cover the latency of HBM. Short rows take one warp each.
template <int XT, int RT>
static cudaError_t norm_of(const RowLaunch& env, const NormParams& p, bool vec) {
    const dim3 warps((p.rows + 3) / 4), blocks(p.rows);
    if (vec) {
        if (p.cols <= 256) return launch_rows(env, norm_kernel<XT, RT, 8, 1, 32>, p, warps, 128, 0);
        if (p.cols <= 1024) return launch_rows(env, norm_kernel<XT, RT, 8, 4, 32>, p, warps, 128, 0);
        if (p.cols <= 2048) return launch_rows(env, norm_kernel<XT, RT, 8, 2, 128>, p, blocks, 128, 0);
        if (p.cols <= 4096) return launch_rows(env, norm_kernel<XT, RT, 8, 2, 256>, p, blocks, 256, 0);
        if (p.cols <= 8192) return launch_rows(env, norm_kernel<XT, RT, 8, 2, 512>, p, blocks, 512, 0);
        if (p.cols <= 16384) return launch_rows(env, norm_kernel<XT, RT, 8, 4, 512>, p, blocks, 512, 0);
        if (p.cols <= 32768) return launch_rows(env, norm_kernel<XT, RT, 8, 4, 1024>, p, blocks, 1024, 0);
        return launch_rows(env, norm_long_kernel<XT, RT, 8>, p, blocks, 1024, 0);
    }
    if (p.cols <= 256) return launch_rows(env, norm_kernel<XT, RT, 1, 8, 32>, p, warps, 128, 0);
    if (p.cols <= 1024) return launch_rows(env, norm_kernel<XT, RT, 1, 32, 32>, p, warps, 128, 0);
    if (p.cols <= 2048) return launch_rows(env, norm_kernel<XT, RT, 1, 16, 128>, p, blocks, 128, 0);
    if (p.cols <= 4096) return launch_rows(env, norm_kernel<XT, RT, 1, 16, 256>, p, blocks, 256, 0);
    if (p.cols <= 8192) return launch_rows(env, norm_kernel<XT, RT, 1, 16, 512>, p, blocks, 512, 0);
    if (p.cols <= 16384) return launch_rows(env, norm_kernel<XT, RT, 1, 32, 512>, p, blocks, 512, 0);
    return launch_rows(env, norm_long_kernel<XT, RT, 1>, p, blocks, 1024, 0);
}

cudaError_t launch_norm(const RowLaunch& env, const NormParams& p, bool vec) {
    const int rt = p.residual.ptr ? p.residual.type : ROW_NONE;
    if (p.x.type == ROW_BF16)
        return rt == ROW_NONE ? norm_of<ROW_BF16, ROW_NONE>(env, p, vec) : rt == ROW_BF16 ? norm_of<ROW_BF16, ROW_BF16>(env, p, vec) : norm_of<ROW_BF16, ROW_F32>(env, p, vec);
    return rt == ROW_NONE ? norm_of<ROW_F32, ROW_NONE>(env, p, vec) : rt == ROW_BF16 ? norm_of<ROW_F32, ROW_BF16>(env, p, vec) : norm_of<ROW_F32, ROW_F32>(env, p, vec);
}

uint32_t norm_grad_blocks(int sm_count, uint32_t rows, uint32_t cols) {
    const uint32_t per_block = cols <= 1024 ? 4 : 1;
    const uint32_t resident = cols <= 1024 ? 4 : cols <= 2048 ? 6 : cols <= 4096 ? 4 : cols <= 8192 ? 2 : 1;   // blocks an SM holds
    return std::min<uint32_t>((rows + per_block - 1) / per_block, uint32_t(sm_count) * resident);
}

template <int XT, int DT_>
static cudaError_t norm_grad_of(const RowLaunch& env, const NormGradParams& p, bool vec, uint32_t blocks) {
    const dim3 g(blocks);
    const size_t sums = p.cols <= 1024 ? p.cols * sizeof(float) : 0;
    if (vec) {
        if (p.cols <= 256) return launch_rows(env, norm_grad_kernel<XT, DT_, 8, 1, 32>, p, g, 128, sums);
        if (p.cols <= 1024) return launch_rows(env, norm_grad_kernel<XT, DT_, 8, 4, 32>, p, g, 128, sums);
        if (p.cols <= 2048) return launch_rows(env, norm_grad_kernel<XT, DT_, 8, 2, 128>, p, g, 128, 0);
        if (p.cols <= 4096) return launch_rows(env, norm_grad_kernel<XT, DT_, 8, 2, 256>, p, g, 256, 0);
        if (p.cols <= 8192) return launch_rows(env, norm_grad_kernel<XT, DT_, 8, 2, 512>, p, g, 512, 0);
        return launch_rows(env, norm_grad_long_kernel<XT, DT_, 8>, p, g, 1024, 0);
    }
    if (p.cols <= 256) return launch_rows(env, norm_grad_kernel<XT, DT_, 1, 8, 32>, p, g, 128, sums);
    if (p.cols <= 1024) return launch_rows(env, norm_grad_kernel<XT, DT_, 1, 32, 32>, p, g, 128, sums);
    if (p.cols <= 2048) return launch_rows(env, norm_grad_kernel<XT, DT_, 1, 16, 128>, p, g, 128, 0);
    if (p.cols <= 4096) return launch_rows(env, norm_grad_kernel<XT, DT_, 1, 16, 256>, p, g, 256, 0);
    if (p.cols <= 8192) return launch_rows(env, norm_grad_kernel<XT, DT_, 1, 16, 512>, p, g, 512, 0);
    return launch_rows(env, norm_grad_long_kernel<XT, DT_, 1>, p, g, 1024, 0);
}

cudaError_t launch_norm_grad(const RowLaunch& env, const NormGradParams& p, bool vec, uint32_t blocks) {
    if (p.x.type == ROW_BF16) return p.dsum.ptr ? norm_grad_of<ROW_BF16, ROW_BF16>(env, p, vec, blocks) : norm_grad_of<ROW_BF16, ROW_NONE>(env, p, vec, blocks);
    return p.dsum.ptr ? norm_grad_of<ROW_F32, ROW_F32>(env, p, vec, blocks) : norm_grad_of<ROW_F32, ROW_NONE>(env, p, vec, blocks);
}

struct ColumnSums { const float* partial; float* out; uint32_t blocks, cols; };
static __global__ void __launch_bounds__(256) column_sums_kernel(const __grid_constant__ ColumnSums p) { column_sums(p.partial, p.out, p.blocks, p.cols); }
cudaError_t launch_column_sums(const RowLaunch& env, const float* partial, float* out, uint32_t blocks, uint32_t cols) {
    const ColumnSums p{partial, out, blocks, cols};
    return launch_rows(env, column_sums_kernel, p, dim3((cols + 31) / 32), 256, 0);
}

struct ColumnSteps { float* scale; uint32_t cols; float top; };
static __global__ void __launch_bounds__(256) column_steps_kernel(const __grid_constant__ ColumnSteps p) { column_steps(p.scale, p.cols, p.top); }

cudaError_t launch_quant_trans(const RowLaunch& env, const QuantTransParams& p, int* launches) {
    *launches = 0;
    const bool bf16 = p.x_type == ROW_BF16;
    cudaError_t e = cudaSuccess;
    if (!p.given) {
        e = cudaMemsetAsync(p.scale, 0, size_t(p.cols) * sizeof(float), env.stream);
        if (e != cudaSuccess) return e;
        const uint32_t strips = (p.cols + 31) / 32;
        const uint32_t cuts = std::max(1u, std::min((p.rows + 63) / 64, uint32_t(env.sm_count) * 8 / std::max(1u, std::min(strips, uint32_t(env.sm_count) * 8))));
        e = launch_rows(env, bf16 ? column_max_kernel<ROW_BF16> : column_max_kernel<ROW_F32>, p, dim3(strips, cuts), 256, 0);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    e = launch_rows(env, bf16 ? quant_trans_kernel<ROW_BF16> : quant_trans_kernel<ROW_F32>, p, dim3((p.cols + 63) / 64, (p.rows + 63) / 64), 256, 0);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (!p.given) {
        const ColumnSteps s{p.scale, p.cols, p.top};
        e = launch_rows(env, column_steps_kernel, s, dim3((p.cols + 255) / 256), 256, 0);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    return cudaSuccess;
}

// A product's operand whose rows do not start on 16 bytes, copied to rows that do. A thread makes 16 bytes of the copy from
// the four or five aligned words that hold them; the words at a row's ends, which reach past it, are read byte by byte.
struct PadRows { const uint8_t* src; uint8_t* dst; uint64_t rows, cols, src_ld, dst_ld; };
static __global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadRows p) {
    griddep_wait();
    griddep_launch_dependents();
    const uint64_t pieces = (p.cols + 15) / 16, total = p.rows * pieces;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += uint64_t(gridDim.x) * 256) {
        const uint64_t r = i / pieces, c = (i % pieces) * 16;
        const uint8_t* s = p.src + r * p.src_ld + c;
        const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(s) & 3);
        uint32_t w[4];
        if (c >= 4 && c + 20 <= p.cols) {   // the aligned words around these 16 bytes lie inside the row
            const uint32_t* q = reinterpret_cast<const uint32_t*>(s - shift);
            uint32_t prev = q[0];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t next = (k < 3 || shift) ? q[k + 1] : 0u;
                w[k] = __funnelshift_r(prev, next, shift * 8);
                prev = next;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w[k] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (c + 4 * k + b < p.cols) w[k] |= uint32_t(s[4 * k + b]) << (8 * b);
            }
        }
        *reinterpret_cast<uint4*>(p.dst + r * p.dst_ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
cudaError_t launch_pad_rows(const RowLaunch& env, const void* src, void* dst, uint64_t rows, uint64_t cols, uint64_t src_ld, uint64_t dst_ld) {
    const PadRows p{static_cast<const uint8_t*>(src), static_cast<uint8_t*>(dst), rows, cols, src_ld, dst_ld};
    const uint64_t blocks = (rows * ((cols + 15) / 16) + 255) / 256;
    return launch_rows(env, pad_rows_kernel, p, dim3(unsigned(std::min<uint64_t>(blocks, uint64_t(env.sm_count) * 16))), 256, 0);
}

}  // namespace mmeb200
