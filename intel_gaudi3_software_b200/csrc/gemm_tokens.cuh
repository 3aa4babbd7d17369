// Scaled 8-bit product for few tokens (or few output tiles): out[m][n] = acc * row_scale[m] * col_scale[n] + bias[n].
//
// With few tokens the weights are what has to be read, once, and everything else is small, so the weights take the MMA's
// 128-row side and the tokens its N side: a CTA accumulates (128 output channels) x (tok tokens), tok a multiple of 16 that
// just holds the tokens, and the padding costs neither bandwidth nor shared memory. Tensor cores at this shape consume
// 64 bytes of weights per clock and SM, above what HBM delivers, so the kernel is bound by the weights' stream; a ring of
// 128-byte-wide stages that fills the SM's shared memory keeps it fed.
//
// One column of channel tiles rarely fills 148 SMs, so the k blocks are split over the CTAs of a cluster. Their partial
// accumulators meet in distributed shared memory: every CTA owns a share of the tile's tokens, receives the others' partial
// sums for them, adds them in rank order (integer sums are exact anyway; fp32 sums have a fixed order) and writes them
// out. No workspace in global memory, no second launch, no atomics.
//
// Where there are more CTAs than SMs, two of them share an SM (with half the ring each): one's set-up and epilogue run under
// the other's stream, and a number of CTAs that is not a multiple of the SMs' still keeps HBM busy to the end.
//
// Measured (GPU events, int8): 1 x 8192 x 8192 13.7 us and 37 x 28672 x 8192 41 us, 75 % and 88 % of the time in which HBM's copy
// rate delivers the weights (the rest is the launch, the first stage's latency and the exchange); 256 x 8192 x 8192 20 us.
//
// CTA layout (320 threads): warp 0 feeds the ring by TMA, warp 1 allocates tensor memory and issues the MMAs, warps 2-9 are
// the epilogue (lane = channel; two warps per 32 channels share the tokens: one alone is bound by its instructions' latency). Every mbarrier wait is bounded as in the other GEMM kernels.
#pragma once
#include "gemm_tokens.h"

namespace mmeb200 {

constexpr int kTokenThreads = 320;
constexpr uint32_t kTokenBarrierBytes = 256;
constexpr uint32_t kTokenWBytes = kBlockM * kRowBytes;
constexpr uint32_t kTokenMaxStages = 12;

// One output: 32 lanes write 32 consecutive channels of a token.
template <bool BF16>
__device__ __forceinline__ void token_put(const TokenGemmParams& p, uint32_t m, uint32_t n, float y) {
    if constexpr (BF16) {
        uint32_t w;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(0.0f), "f"(y));
        static_cast<uint16_t*>(p.out)[uint64_t(m) * p.out_ld + n] = uint16_t(w);
    } else {
        static_cast<float*>(p.out)[uint64_t(m) * p.out_ld + n] = y;
    }
}
// COUNT consecutive tokens of this lane's channel: acc * (the token's scale, held by lane `place` + j), rounded, then * ws + bias in
// one operation, as in the CTA-pair kernel (epilogue_scaled). `exist` of them exist. All values first, then all stores: nothing waits
// between two of them.
template <int KIND, bool BF16, int COUNT>
__device__ __forceinline__ void token_put_all(const TokenGemmParams& p, const uint32_t* v, uint32_t m, uint32_t exist, uint32_t n, float scales, uint32_t place, float ws,
                                              float bias) {
    float y[COUNT];
#pragma unroll
    for (int j = 0; j < COUNT; ++j) y[j] = fmaf(scaled_acc<KIND>(v[j]) * __shfl_sync(0xffffffffu, scales, place + j), ws, bias);
    if (n < p.N) {
#pragma unroll
        for (int j = 0; j < COUNT; ++j)
            if (uint32_t(j) < exist) token_put<BF16>(p, m + j, n, y[j]);
    }
}
template <int KIND, int COUNT>
__device__ __forceinline__ void token_store(const TokenGemmParams& p, const uint32_t* v, uint32_t m, uint32_t exist, uint32_t n, float scales, uint32_t place, float ws,
                                            float bias) {
    if (p.out_bf16) token_put_all<KIND, true, COUNT>(p, v, m, exist, n, scales, place, ws, bias);
    else token_put_all<KIND, false, COUNT>(p, v, m, exist, n, scales, place, ws, bias);
}
template <int KIND>
__device__ __forceinline__ uint32_t token_add(uint32_t a, uint32_t b) {
    if constexpr (KIND == KIND_I8) return a + b;
    else return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
template <int KIND>
__global__ void __launch_bounds__(kTokenThreads, 2) gemm_tokens_kernel(const __grid_constant__ TokenGemmParams p) {
    griddep_launch_dependents();
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {   // uniform over the cluster
        if (threadIdx.x == 0) atomicCAS(p.status, 0u, SMEM_MISALIGNED);
        return;
    }
    const uint32_t stages = p.stages, stage_bytes = p.stage_bytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
    uint64_t* empty_bar = full_bar + kTokenMaxStages;
    uint64_t* done_bar = empty_bar + kTokenMaxStages;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done_bar + 1);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % p.splits, n0 = (blockIdx.x / p.splits) * kBlockM, m0 = (p.m_tile0 + blockIdx.y) * p.tok;
    const uint32_t per = (p.num_k_blocks + p.splits - 1) / p.splits;
    const uint32_t kb0 = rank * per, kb1 = min(p.num_k_blocks, kb0 + per);   // the planner leaves no share empty

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(done_bar, 1);
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_w);
        tma_prefetch_desc(&p.tm_x);
    }
    if (warp == 1) {
        tmem_alloc(tmem_holder, p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_holder;
    griddep_wait();

    const uint32_t sub = warp & 3, grp = (warp - 2) >> 2, n = n0 + sub * 32 + lane;   // epilogue: this lane's channel
    float ws = 0.0f, bias = -0.0f;   // (no bias: minus zero, which leaves every sum as it is)
    bool ready = true;
    if (warp == 0) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, kWaitLimitNs)) {
                    atomicCAS(p.status, 0u, WAIT_PRODUCER_EMPTY);
                    break;
                }
                uint8_t* dst = smem + stage * stage_bytes;
                mbar_arrive_expect_tx(&full_bar[stage], stage_bytes);
                tma_load_5d(dst, &p.tm_w, &full_bar[stage], int(kb * kRowBytes), int(n0), 0, 0, 0);
                tma_load_5d(dst + kTokenWBytes, &p.tm_x, &full_bar[stage], int(kb * kRowBytes), int(m0), 0, 0, 0);
                if (++stage == stages) { stage = 0; phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, accumulate = 0;
            const uint64_t w_desc0 = make_smem_desc(smem_u32(smem), 16, 1024);
            bool ok = true;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(&full_bar[stage], phase, kWaitLimitNs)) {
                    atomicCAS(p.status, 0u, WAIT_MMA_FULL);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint64_t w_desc = w_desc0 + ((stage * stage_bytes) >> 4);
                const uint64_t x_desc = w_desc + (kTokenWBytes >> 4);
#pragma unroll
                for (uint32_t k = 0; k < kRowBytes / kUmmaKBytes; ++k) {
                    umma_ss<KIND>(tmem_base, w_desc + k * (kUmmaKBytes >> 4), x_desc + k * (kUmmaKBytes >> 4), p.idesc, accumulate);
                    accumulate = 1;
                }
                umma_commit(&empty_bar[stage]);
                if (++stage == stages) { stage = 0; phase ^= 1; }
            }
            if (ok) umma_commit(done_bar);
        }
        __syncwarp();
    } else {
        if (n < p.N) {
            ws = p.scaled.col_scale[uint64_t(n) * p.scaled.col_stride];
            if (p.scaled.col_bias) bias = scaled_bias(p.scaled, n);
        }
        ready = mbar_wait_bounded(done_bar, 0, kWaitLimitNs);
        ready = __all_sync(0xffffffffu, ready);
        if (!ready) atomicCAS(p.status, 0u, WAIT_EPILOGUE_TMEM_FULL);
        tc_fence_after_sync();
    }

    const uint32_t tokens = min(p.tok, p.M - m0);
    // the scale of a token, held by the lane of its place among 32 tokens
    auto token_scale = [&](uint32_t first) {
        const uint32_t t = first + lane;
        return t < tokens ? p.scaled.row_scale[uint64_t(m0 + t) * p.scaled.row_stride] * p.scale : 0.0f;
    };
    if (p.splits == 1) {
        if (warp >= 2 && ready) {
            for (uint32_t c0 = grp * 16; c0 < tokens; c0 += 32) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(tmem_base + c0 + ((sub * 32) << 16), v);
                const float xs = token_scale(c0);
                tmem_ld_wait();
                token_store<KIND, 16>(p, v, m0 + c0, tokens - c0, n, xs, 0, ws, bias);
            }
        }
    } else {
        // Every CTA's stages are idle (its MMAs have completed) before anyone writes into them.
        cluster_sync_all();
        const uint32_t share = ((tokens + p.splits - 1) / p.splits + 3) & ~3u;   // tokens a rank owns, in fours
        const uint32_t channel = sub * 32 + lane;
        uint4* inbox = reinterpret_cast<uint4*>(smem) + channel;                  // [source rank][four tokens][channel]
        if (warp >= 2 && ready) {
            const uint32_t mine = smem_u32(inbox + rank * (share / 4) * kBlockM);   // the slot of this rank
            // each rank begins with its own share and goes round, so that no two ranks write to the same CTA at once
            for (uint32_t i = grp; i < p.splits; i += 2) {
                const uint32_t owner = rank + i < p.splits ? rank + i : rank + i - p.splits, first = owner * share;
                const uint32_t to = mapa_shared(mine, owner);
                for (uint32_t t = 0; t < share && first + t < tokens; t += 16) {
                    uint32_t v[16];
#pragma unroll
                    for (uint32_t j = 0; j < 16; j += 4)
                        if (t + j < share && first + t + j < tokens) tmem_ld_32x32b_x4(tmem_base + first + t + j + ((sub * 32) << 16), v + j);
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t j = 0; j < 16; j += 4)
                        if (t + j < share && first + t + j < tokens) st_shared_cluster_v4(to + (t + j) * (kBlockM * 4), v[j], v[j + 1], v[j + 2], v[j + 3]);
                }
            }
        }
        cluster_sync_all();
        if (warp >= 2) {
            const uint32_t first = rank * share, count = first < tokens ? min(share, tokens - first) : 0;
            float xs = 0.0f;
            for (uint32_t t = 4 * grp; t < count; t += 8) {
                if ((t & 31) == 4 * grp) xs = token_scale(first + t - 4 * grp);
                uint4 sum = inbox[(t / 4) * kBlockM];
#pragma unroll 7
                for (uint32_t r = 1; r < p.splits; ++r) {
                    const uint4 v = inbox[(r * share + t) / 4 * kBlockM];
                    sum.x = token_add<KIND>(sum.x, v.x);
                    sum.y = token_add<KIND>(sum.y, v.y);
                    sum.z = token_add<KIND>(sum.z, v.z);
                    sum.w = token_add<KIND>(sum.w, v.w);
                }
                const uint32_t four[4] = {sum.x, sum.y, sum.z, sum.w};
                token_store<KIND, 4>(p, four, m0 + first + t, count - t, n, xs, t & 31, ws, bias);
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }
}

// No common dimension: the sums are empty and the bias, or zero, is the result.
static __global__ void __launch_bounds__(256) gemm_empty_sum_kernel(const __grid_constant__ TokenGemmParams p) {
    griddep_wait();
    const uint64_t total = uint64_t(p.M) * p.N;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += uint64_t(gridDim.x) * 256) {
        const uint32_t m = uint32_t(i / p.N), n = uint32_t(i % p.N);
        const float y = p.scaled.col_bias ? scaled_bias(p.scaled, n) : 0.0f;
        if (p.out_bf16) token_put<true>(p, m, n, y);
        else token_put<false>(p, m, n, y);
    }
}

}  // namespace mmeb200
