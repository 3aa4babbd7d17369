// Host-side launchers of the row kernels (norm_quant.cu): RMS norm with the residual's addition and an optional 8-bit
// output, its gradient, and row-wise quantisation to 8 bits. This is what api.cu sees of them.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "numerics.cuh"

namespace mmeb200 {

enum : int { ROW_NONE = 0, ROW_BF16 = 1, ROW_F32 = 2, ROW_I8 = 3, ROW_F8 = 4 };   // element types of the row kernels

// What a norm writes: floats, codes whose step the row decides, codes under a given scale.
enum : int { NORM_BF16 = 0, NORM_F32 = 1, NORM_I8 = 2, NORM_F8 = 3, NORM_I8_GIVEN = 4, NORM_F8_GIVEN = 5 };

// Rows of a tensor: row r is the index of dims 1..4 with dim 1 fastest; element c of it sits at base + off(r) + c.
struct RowTensor {
    void* ptr;
    int type;              // ROW_*
    uint32_t stride[4];    // elements, dims 1..4
};

struct NormParams {
    RowTensor x, residual, sum, out;
    RowTensor gamma;       // one row; ptr nullptr: ones
    float* scale;          // 8-bit outputs: the step of every row (written)
    const float* given;    // 8-bit outputs with a given scale: read instead; given_stride 0 = one for all rows
    uint32_t given_stride;
    uint32_t rows, cols;
    uint32_t dims[4];      // sizes of dims 1..4
    uint32_t flat;         // 1: rows are dims[0] alone (no division per row)
    uint32_t norm;         // 0: quantise x as it is
    int mode;              // NORM_*
    float eps, per_col;    // per_col: 1 / cols
    float top;             // largest code of the 8-bit output
    Fp8HwCast hw;          // ROW_F8
    uint32_t fp8_direct;   // no quotient of a row's own step passes the hardware conversion's limit
};

struct NormGradParams {
    RowTensor dx, dy, x, dsum;
    RowTensor gamma;
    float* partial;        // [blocks][cols]; nullptr: no gradient of gamma wanted
    uint32_t rows, cols;
    uint32_t dims[4];
    uint32_t flat;
    uint32_t ranks;        // blocks of a row's cluster; set by the launcher
    float eps, per_col;
};

// Quantisation of columns with a transposed result: x is rows x cols (cols fastest), out cols x rows (rows fastest).
struct QuantTransParams {
    RowTensor x;
    uint64_t x_ld, out_ld;   // elements between rows of x / of out
    void* out;
    int out_type;
    float* scale;            // [cols]
    const float* given;
    uint32_t given_stride;
    uint32_t rows, cols;
    uint32_t row0;           // first of the rows this launch quantises (the maxima are of all)
    float top;
    Fp8HwCast hw;
    uint32_t fp8_direct;
};

struct RowLaunch {
    int device, sm_count;
    cudaStream_t stream;
    bool dependent_launch;
};

// How the rows of a call's tensors lie (`vec`): 8, every row of every tensor, and its end, on eight elements; kPhased, a row of
// every tensor equally far past eight elements (gamma on 16 bytes); 1, anything.
constexpr int kPhased = 0;
cudaError_t launch_norm(const RowLaunch& env, const NormParams& p, int vec);
// Blocks (or clusters of blocks) the gradient kernel runs with, i.e. rows of `partial`.
uint32_t norm_grad_blocks(int device, int sm_count, uint32_t rows, uint32_t cols);
// Of those, the blocks that phased rows can use (0: none).
uint32_t norm_grad_phased_blocks(uint32_t blocks, uint32_t rows, uint32_t cols);
cudaError_t launch_norm_grad(const RowLaunch& env, const NormGradParams& p, int vec, uint32_t blocks);
cudaError_t launch_column_sums(const RowLaunch& env, const float* partial, float* out, uint32_t blocks, uint32_t cols);
// Number of kernels launched is returned in *launches.
cudaError_t launch_quant_trans(const RowLaunch& env, const QuantTransParams& p, int vec, int* launches);

// Rows of `cols` bytes, src_ld bytes apart at any alignment, copied to rows dst_ld bytes apart (dst and dst_ld multiples of 16).
cudaError_t launch_pad_rows(const RowLaunch& env, const void* src, void* dst, uint64_t rows, uint64_t cols, uint64_t src_ld, uint64_t dst_ld);

}  // namespace mmeb200
