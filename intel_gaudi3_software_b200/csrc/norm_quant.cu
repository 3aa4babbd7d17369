// Launchers of the row kernels: the instantiation for a call's element types and alignment, and the small kernels beside them.
#include <algorithm>
#include <atomic>

#include "layer_host.h"
#include "norm_quant.cuh"
#include "norm_quant_launch.h"

namespace mmeb200 {

template <int XT, int RT>
static cudaError_t norm_with(const RowLaunch& env, const NormParams& p, int vec) {
    return vec == 8 ? norm_of<XT, RT, 8>(env, p) : vec == kPhased ? norm_of<XT, RT, kPhased>(env, p) : norm_of<XT, RT, 1>(env, p);
}
cudaError_t launch_norm(const RowLaunch& env, const NormParams& p, int vec) {
    const int rt = p.residual.ptr ? p.residual.type : ROW_NONE;
    if (p.x.type == ROW_BF16)
        return rt == ROW_NONE ? norm_with<ROW_BF16, ROW_NONE>(env, p, vec) : rt == ROW_BF16 ? norm_with<ROW_BF16, ROW_BF16>(env, p, vec) : norm_with<ROW_BF16, ROW_F32>(env, p, vec);
    return rt == ROW_NONE ? norm_with<ROW_F32, ROW_NONE>(env, p, vec) : rt == ROW_BF16 ? norm_with<ROW_F32, ROW_BF16>(env, p, vec) : norm_with<ROW_F32, ROW_F32>(env, p, vec);
}

// As many blocks as the SMs hold at once: a block walks its rows to the end.
uint32_t norm_grad_blocks(int device, int sm_count, uint32_t rows, uint32_t cols) {
    const GradShape g = grad_shape(cols);
    uint64_t held = uint64_t(sm_count) * g.blocks_per_sm;
    if (g.form == GRAD_CLUSTER) {
        static std::atomic<int> known[64][9][9] = {};   // by device, ranks and warps
        // (any number is right; it is kept, so that the workspace asked for is the one the call wants)
        held = uint64_t(device_holds(known[device & 63][g.ranks][g.threads / 32], [&](int* n) { return norm_grad_clusters(g.ranks, g.threads, n); }, [] { cudaGetLastError(); },
                                     std::max(1, sm_count / int(g.ranks))));
    }
    return uint32_t(std::min<uint64_t>((uint64_t(rows) + g.rows_per_block - 1) / g.rows_per_block, held));
}
template <int XT, bool DSUM>
static cudaError_t norm_grad_with(const RowLaunch& env, const NormGradParams& p, int vec, uint32_t blocks) {
    return vec == 8 ? norm_grad_of<XT, DSUM, 8>(env, p, blocks) : vec == kPhased ? norm_grad_of<XT, DSUM, kPhased>(env, p, blocks) : norm_grad_of<XT, DSUM, 1>(env, p, blocks);
}
// A block walks rows that are `blocks` blocks apart and keeps the sums of its columns: phased rows need a multiple of eight blocks,
// so that a block's rows have one phase.
uint32_t norm_grad_phased_blocks(uint32_t blocks, uint32_t rows, uint32_t cols) {
    return uint64_t(blocks) * grad_shape(cols).rows_per_block >= rows ? blocks : blocks & ~7u;
}
cudaError_t launch_norm_grad(const RowLaunch& env, const NormGradParams& p, int vec, uint32_t blocks) {
    if (p.x.type == ROW_BF16) return p.dsum.ptr ? norm_grad_with<ROW_BF16, true>(env, p, vec, blocks) : norm_grad_with<ROW_BF16, false>(env, p, vec, blocks);
    return p.dsum.ptr ? norm_grad_with<ROW_F32, true>(env, p, vec, blocks) : norm_grad_with<ROW_F32, false>(env, p, vec, blocks);
}

struct ColumnSums { const float* partial; float* out; uint32_t blocks, cols; };
static __global__ void __launch_bounds__(1024) column_sums_kernel(const __grid_constant__ ColumnSums p) { column_sums(p.partial, p.out, p.blocks, p.cols); }
cudaError_t launch_column_sums(const RowLaunch& env, const float* partial, float* out, uint32_t blocks, uint32_t cols) {
    const ColumnSums p{partial, out, blocks, cols};
    return launch_rows(env, column_sums_kernel, p, dim3((cols + 31) / 32), 1024, 0);
}

template <int XT>
static cudaError_t quant_trans_with(const RowLaunch& env, const QuantTransParams& p, int vec, int* launches) {
    return vec == 8 ? quant_trans_of<XT, 8>(env, p, launches) : vec == kPhased ? quant_trans_of<XT, kPhased>(env, p, launches) : quant_trans_of<XT, 1>(env, p, launches);
}
cudaError_t launch_quant_trans(const RowLaunch& env, const QuantTransParams& p, int vec, int* launches) {
    *launches = 0;
    return p.x.type == ROW_BF16 ? quant_trans_with<ROW_BF16>(env, p, vec, launches) : quant_trans_with<ROW_F32>(env, p, vec, launches);
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
