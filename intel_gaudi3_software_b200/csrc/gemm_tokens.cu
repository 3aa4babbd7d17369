// Launcher of the few-token product kernel; see gemm_tokens.h.
#include "gemm_tokens.cuh"

#include <atomic>
#include <cstring>

namespace mmeb200 {

constexpr int kTokenSmem = 227 * 1024;   // of a CTA alone on an SM

uint32_t gemm_tokens_stages(uint32_t tok, uint32_t ctas) {
    const uint32_t smem = ctas == 1 ? kTokenSmem : 228 * 1024 / ctas - 1024;   // 1 KB of every CTA is the system's
    const uint32_t n = (smem - kTokenBarrierBytes) / (kTokenWBytes + tok * kRowBytes);
    return n < kTokenMaxStages ? n : kTokenMaxStages;
}

template <int KIND>
static cudaError_t configure(const LaunchEnv& env, uint32_t tok, uint32_t splits, uint32_t ctas, cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attrs) {
    static std::atomic<bool> done[64] = {};   // (two contexts may meet here on two threads)
    if (!done[env.device & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(gemm_tokens_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTokenSmem);
        if (e != cudaSuccess) return e;
        done[env.device & 63] = true;
    }
    memset(cfg, 0, sizeof *cfg);
    cfg->blockDim = dim3(kTokenThreads);
    cfg->dynamicSmemBytes = gemm_tokens_stages(tok, ctas) * (kTokenWBytes + tok * kRowBytes) + kTokenBarrierBytes;
    cfg->stream = env.stream;
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = splits; attrs[0].val.clusterDim.y = 1; attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg->attrs = attrs;
    cfg->numAttrs = env.dependent_launch ? 2 : 1;
    return cudaSuccess;
}

template <int KIND>
static LaunchResult launch(const LaunchEnv& env, TokenGemmParams& p) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attrs[2];
    cudaError_t e = configure<KIND>(env, p.tok, p.splits, p.ctas, &cfg, attrs);
    if (e != cudaSuccess) return {e, LAUNCH_OK, "cudaFuncSetAttribute(few-token kernel)"};
    p.stage_bytes = kTokenWBytes + p.tok * kRowBytes;
    p.stages = gemm_tokens_stages(p.tok, p.ctas);
    p.tmem_cols = 32;
    while (p.tmem_cols < p.tok) p.tmem_cols *= 2;
    const uint32_t m_tiles = (p.M + p.tok - 1) / p.tok - p.m_tile0;
    cfg.gridDim = dim3(p.splits * ((p.N + kBlockM - 1) / kBlockM), m_tiles < kTokenTilesY ? m_tiles : kTokenTilesY);
    e = cudaLaunchKernelEx(&cfg, gemm_tokens_kernel<KIND>, p);
    return {e, LAUNCH_OK, "few-token kernel launch"};   // (not the thread's last error, which may be an older one of the caller's)
}

LaunchResult launch_gemm_tokens(const LaunchEnv& env, uint32_t kind, TokenGemmParams p) {
    return kind == KIND_I8 ? launch<KIND_I8>(env, p) : launch<KIND_F8>(env, p);
}

template <int KIND>
static bool capacity(const LaunchEnv& env, uint32_t tok, uint32_t splits, uint32_t ctas, int* n) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attrs[2];
    if (configure<KIND>(env, tok, splits, ctas, &cfg, attrs) != cudaSuccess) return false;
    cfg.gridDim = dim3(splits * unsigned(env.sm_count));
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(n, gemm_tokens_kernel<KIND>, &cfg) != cudaSuccess) return false;
    *n *= int(splits);
    return true;
}

LaunchResult launch_gemm_empty_sum(const LaunchEnv& env, const TokenGemmParams& p) {
    const uint64_t blocks = (uint64_t(p.M) * p.N + 255) / 256, most = uint64_t(env.sm_count) * 8;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3(unsigned(blocks < most ? blocks : most));
    cfg.blockDim = dim3(256);
    cfg.stream = env.stream;
    return {cudaLaunchKernelEx(&cfg, gemm_empty_sum_kernel, p), LAUNCH_OK, "empty-sum kernel launch"};
}

bool gemm_tokens_capacity(const LaunchEnv& env, uint32_t kind, uint32_t tok, uint32_t splits, uint32_t ctas, int* n) {
    return kind == KIND_I8 ? capacity<KIND_I8>(env, tok, splits, ctas, n) : capacity<KIND_F8>(env, tok, splits, ctas, n);
}

}  // namespace mmeb200
