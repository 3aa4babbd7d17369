// Host-side launcher of the few-token product kernel (gemm_tokens.cuh).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_launch.h"

namespace mmeb200 {

struct TokenGemmParams {
    CUtensorMap tm_w, tm_x;     // (K, channels) and (K, tokens); boxes 128 B x 128 rows and 128 B x tok rows
    uint32_t M, N;              // tokens, output channels
    uint32_t num_k_blocks;      // 128-byte blocks of K
    uint32_t tok;               // tokens of a tile (a multiple of 16, at most 256)
    uint32_t splits;            // CTAs of a cluster, each with its share of the k blocks
    uint32_t ctas;              // CTAs that share an SM (1 or 2): sets how much shared memory each has for its ring
    uint32_t m_tile0;           // first token tile of this launch: a grid has at most kTokenTilesY of them
    uint32_t stages, stage_bytes;
    uint32_t tmem_cols;
    uint32_t idesc;
    float scale;                // power of two of the operands' exponent biases
    ScaledOut scaled;
    void* out;
    uint32_t out_bf16;
    uint64_t out_ld;
    uint32_t* status;
};

constexpr uint32_t kTokenTilesY = 65535;
// Fills stages, stage_bytes and tmem_cols for p.tok and launches on a grid of splits x channel tiles x token tiles (from m_tile0 on,
// kTokenTilesY at most).
LaunchResult launch_gemm_tokens(const LaunchEnv& env, uint32_t kind, TokenGemmParams p);
// out = bias (or zero) for operands without a common dimension.
LaunchResult launch_gemm_empty_sum(const LaunchEnv& env, const TokenGemmParams& p);
// Most CTAs the device runs at once in clusters of `splits` with tiles of `tok` tokens; false where the question fails.
bool gemm_tokens_capacity(const LaunchEnv& env, uint32_t kind, uint32_t tok, uint32_t splits, uint32_t ctas, int* n);
// Stages of the ring of a CTA, one of `ctas` on its SM; fewer than three do not keep the tensor cores fed.
uint32_t gemm_tokens_stages(uint32_t tok, uint32_t ctas);

}  // namespace mmeb200
