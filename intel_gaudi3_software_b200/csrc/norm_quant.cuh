// Row kernels around the 8-bit products: RMS norm with the residual's addition and an optional 8-bit output, its gradient,
// and row-wise quantisation. All of them are bound by HBM: a row is read once, kept in registers while its sums are taken,
// and written once.
//
// Norm of one row, in 32 bits (h: the row as the residual stream keeps it, after its rounding to the stream's type):
//     inv = 1 / sqrt(mean(h^2) + eps),  v = h * gamma,  y = v * inv.
// 8-bit output: with a = max |v|, step = a / top, every code is the nearest representable value to the 32-bit quotient
// v / step (ties to even), and the row's scale is step * inv. inv does not enter the codes, so sum and maximum are taken in
// one pass, and the codes do not depend on the order of any sum: they are fixed by the definition, bit for bit.
#pragma once
#include "norm_quant.h"
#include "ptx_sm100.cuh"

namespace mmeb200 {

// ------------------------------------------------------------------------------------------ elements
template <int TYPE>
struct RowElem;
template <> struct RowElem<ROW_BF16> { using T = uint16_t; static constexpr int kBytes = 2; };
template <> struct RowElem<ROW_F32> { using T = float; static constexpr int kBytes = 4; };

// VEC elements as they lie in memory. Loading and decoding are separate so that all loads of a row are in flight before
// the first value is needed.
template <int TYPE, int VEC>
struct RowPiece {
    static constexpr int kWords = VEC == 8 ? RowElem<TYPE>::kBytes * 2 : 1;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const void* base, uint64_t at) {
        if constexpr (VEC == 8) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const typename RowElem<TYPE>::T*>(base) + at);
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 q = p[i];
                w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
            }
        } else if constexpr (TYPE == ROW_BF16) {
            w[0] = static_cast<const uint16_t*>(base)[at];
        } else {
            w[0] = static_cast<const uint32_t*>(base)[at];
        }
    }
    __device__ __forceinline__ float value(int e) const {
        if constexpr (TYPE == ROW_F32) return __uint_as_float(w[e]);
        else return __uint_as_float(VEC == 8 ? ((e & 1) ? (w[e >> 1] & 0xFFFF0000u) : (w[e >> 1] << 16)) : (w[0] << 16));
    }
};
template <int VEC>
struct RowPiece<ROW_NONE, VEC> {
    __device__ __forceinline__ void load(const void*, uint64_t) {}
    __device__ __forceinline__ float value(int) const { return 0.0f; }
};

// gamma is read by every row and sits in the caches; its type is a runtime value.
template <int VEC>
__device__ __forceinline__ void load_gamma(float (&g)[VEC], const void* base, int type, uint32_t at) {
    if (type == ROW_BF16) {
        RowPiece<ROW_BF16, VEC> p;
        p.load(base, at);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] = p.value(e);
    } else if (type == ROW_F32) {
        RowPiece<ROW_F32, VEC> p;
        p.load(base, at);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] = p.value(e);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] = 1.0f;
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
template <int VEC>
__device__ __forceinline__ void store_bf16(void* base, uint64_t at, const float (&f)[VEC]) {
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    if constexpr (VEC == 8) *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    else *p = uint16_t(pack_bf16(f[0], 0.0f));
}
template <int VEC>
__device__ __forceinline__ void store_f32(void* base, uint64_t at, const float (&f)[VEC]) {
    float* p = static_cast<float*>(base) + at;
    if constexpr (VEC == 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *p = f[0];
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ uint64_t row_offset(const RowTensor& t, uint32_t row, const uint32_t (&dims)[4], uint32_t flat) {
    if (flat) return uint64_t(row) * t.stride[0];
    uint64_t off = 0;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        off += uint64_t(row % dims[d]) * t.stride[d];
        row /= dims[d];
    }
    return off;
}

// ------------------------------------------------------------------------------------------ 8-bit codes
// How a row's values become codes. `ok` is false for rows whose step is zero or no number: their codes are zero.
struct RowStep {
    float step, recip;
    bool ok, fast;
};
__device__ __forceinline__ RowStep make_row_step(float step) {
    RowStep s;
    s.step = step;
    s.recip = __frcp_rn(step);
    s.ok = step > 0.0f && step < __uint_as_float(0x7F800000u);
    s.fast = step >= 0x1p-126f && step <= 0x1p126f;   // the reciprocal is a normal number
    return s;
}
constexpr float kRoundMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to the nearest whole number, ties to even

// The int8 code of v / step in the low byte. v * recip is within 2^-23 of the quotient, relatively, i.e. within 2^-16 for
// |quotient| <= 127: unless it lies closer than 2^-15 to the middle between two whole numbers, it rounds as the correctly
// rounded quotient does. The few that do lie there are divided.
__device__ __forceinline__ uint32_t int8_code(float v, const RowStep& s) {
    float t = v * s.recip;
    t = fminf(fmaxf(t, -127.0f), 127.0f);
    float m = t + kRoundMagic;
    const float f = fabsf(t - (m - kRoundMagic));
    if (f > 0.5f - 0x1p-15f || !s.fast) {
        t = fminf(fmaxf(__fdiv_rn(v, s.step), -127.0f), 127.0f);
        m = t + kRoundMagic;
    }
    return __float_as_uint(m);
}

// VEC codes of the values v: stored at element `at` of a row of codes.
template <int VEC>
__device__ __forceinline__ void store_codes(void* base, uint64_t at, const float (&v)[VEC], int type, const RowStep& s, const Fp8HwCast& hw) {
    uint8_t* p = static_cast<uint8_t*>(base) + at;
    uint32_t w[VEC == 8 ? 2 : 1];
    if (!s.ok) {
#pragma unroll
        for (int i = 0; i < (VEC == 8 ? 2 : 1); ++i) w[i] = 0;
    } else if (type == ROW_I8) {
        uint32_t q[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) q[e] = int8_code(v[e] == v[e] ? v[e] : 0.0f, s);   // a NaN (given scales only) has no code
        if constexpr (VEC == 8) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lo = __byte_perm(q[4 * i], q[4 * i + 1], 0x0040), hi = __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040);
                w[i] = __byte_perm(lo, hi, 0x5410);
            }
        } else {
            w[0] = q[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < (VEC == 8 ? 2 : 1); ++i) {
            float t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = (VEC == 8 || e == 0) ? __fdiv_rn(v[VEC == 8 ? 4 * i + e : 0], s.step) : 0.0f;
            w[i] = f32x4_to_fp8_hw(t, hw);
        }
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *p = uint8_t(w[0]);
}

// ------------------------------------------------------------------------------------------ reductions
// Sum of `a` and NaN-keeping maximum of `b` over the T threads of a row (a warp, or the whole block). The order is fixed.
struct RowSums { float sum, top; };
template <int T>
__device__ __forceinline__ RowSums reduce_row(float a, float b, float2* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
    if constexpr (T > 32) {
        constexpr int W = T / 32;
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        const float2 v = (threadIdx.x & 31) < W ? scratch[threadIdx.x & 31] : make_float2(0.0f, 0.0f);
        a = v.x;
        b = v.y;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
        }
        a = __shfl_sync(0xffffffffu, a, 0);
        b = __shfl_sync(0xffffffffu, b, 0);
    }
    return {a, b};
}
template <int T>
__device__ __forceinline__ float2 reduce_row2(float a, float b, float2* scratch) {   // two sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (T > 32) {
        constexpr int W = T / 32;
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        const float2 v = (threadIdx.x & 31) < W ? scratch[threadIdx.x & 31] : make_float2(0.0f, 0.0f);
        a = v.x;
        b = v.y;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        a = __shfl_sync(0xffffffffu, a, 0);
        b = __shfl_sync(0xffffffffu, b, 0);
    }
    return make_float2(a, b);
}
__device__ __forceinline__ float inverse_rms(float sum_of_squares, uint32_t cols, float eps) {
    return __frcp_rn(__fsqrt_rn(__fdiv_rn(sum_of_squares, float(cols)) + eps));
}

// What a row's sums decide: the factor of float outputs, the step of codes, the scale that is written.
struct RowFactors { float inv; RowStep step; float scale; };
__device__ __forceinline__ RowFactors row_factors(const NormParams& p, const RowSums& s, uint32_t row) {
    RowFactors f;
    f.inv = p.norm ? inverse_rms(s.sum, p.cols, p.eps) : 1.0f;
    f.scale = 0.0f;
    if (p.given) {
        f.step = make_row_step(p.given[uint64_t(row) * p.given_stride]);
    } else {
        f.step = make_row_step(__fdiv_rn(s.top, p.top));
        const bool finite = f.step.step < __uint_as_float(0x7F800000u);   // false for NaN
        f.scale = !finite ? __uint_as_float(0x7FC00000u) : f.step.ok ? f.step.step * f.inv : 0.0f;
    }
    return f;
}
template <int VEC>
__device__ __forceinline__ void store_row_piece(const NormParams& p, uint64_t at, float (&v)[VEC], const RowFactors& f) {
    if (p.out.type >= ROW_I8) {
        if (p.given) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] *= f.inv;
        }
        store_codes<VEC>(p.out.ptr, at, v, p.out.type, f.step, p.hw);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= f.inv;
        if (p.out.type == ROW_BF16) store_bf16<VEC>(p.out.ptr, at, v);
        else store_f32<VEC>(p.out.ptr, at, v);
    }
}
// h of one piece: the residual's addition, rounded to the stream's type, which is what the norm sees.
template <int XT, int RT, int VEC>
__device__ __forceinline__ void stream_values(const RowPiece<XT, VEC>& x, const RowPiece<RT, VEC>& r, float (&h)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        h[e] = x.value(e);
        if constexpr (RT != ROW_NONE) h[e] += r.value(e);
        if constexpr (RT == ROW_BF16) h[e] = __uint_as_float(pack_bf16(h[e], 0.0f) << 16);
    }
}

// One row per T threads (a warp: several rows per block; else the block), NV pieces of VEC elements per thread, all in
// registers between the row's one read and its one write.
template <int XT, int RT, int VEC, int NV, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T) norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 scratch[32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tid = T == 32 ? (threadIdx.x & 31) : threadIdx.x;
    const uint32_t row = T == 32 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= p.rows) return;   // whole warps (T == 32), never part of a block that synchronises
    const uint64_t xo = row_offset(p.x, row, p.dims, p.flat), ro = RT != ROW_NONE ? row_offset(p.residual, row, p.dims, p.flat) : 0;
    RowPiece<XT, VEC> xs[NV];
    RowPiece<RT, VEC> rs[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = (i * T + tid) * VEC;
        if (c < p.cols) {
            xs[i].load(p.x.ptr, xo + c);
            rs[i].load(p.residual.ptr, ro + c);
        }
    }
    const bool eight = p.out.type >= ROW_I8;
    const uint64_t so = RT != ROW_NONE ? row_offset(p.sum, row, p.dims, p.flat) : 0;
    float v[NV][VEC];
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = (i * T + tid) * VEC;
        if (c < p.cols) {
            float g[VEC];
            load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
            stream_values<XT, RT, VEC>(xs[i], rs[i], v[i]);
            if constexpr (RT != ROW_NONE) {
                if (p.sum.ptr) {
                    if constexpr (RT == ROW_BF16) store_bf16<VEC>(p.sum.ptr, so + c, v[i]);
                    else store_f32<VEC>(p.sum.ptr, so + c, v[i]);
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sum = fmaf(v[i][e], v[i][e], sum);
                v[i][e] *= g[e];
                if (eight) top = max_nan(top, fabsf(v[i][e]));
            }
        }
    }
    const RowSums s = reduce_row<T>(sum, top, scratch);
    const RowFactors f = row_factors(p, s, row);
    if (p.scale && tid == 0) p.scale[row] = f.scale;
    const uint64_t oo = row_offset(p.out, row, p.dims, p.flat);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = (i * T + tid) * VEC;
        if (c < p.cols) store_row_piece<VEC>(p, oo + c, v[i], f);
    }
}

// Rows too long for registers: the row is read a second time (from L2, mostly) once its sums are known. The second read
// takes the stream from `sum` where it was written (in place, x and the residual may be gone by then). A thread reads and
// writes the same elements in both passes.
template <int XT, int RT, int VEC>
__global__ void __launch_bounds__(1024) norm_long_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 scratch[32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = blockIdx.x;
    const uint64_t xo = row_offset(p.x, row, p.dims, p.flat), ro = RT != ROW_NONE ? row_offset(p.residual, row, p.dims, p.flat) : 0;
    const uint64_t so = RT != ROW_NONE ? row_offset(p.sum, row, p.dims, p.flat) : 0, oo = row_offset(p.out, row, p.dims, p.flat);
    const bool eight = p.out.type >= ROW_I8;
    float sum = 0.0f, top = 0.0f;
#pragma unroll 1
    for (uint32_t c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
        RowPiece<XT, VEC> x;
        RowPiece<RT, VEC> r;
        float g[VEC], h[VEC];
        x.load(p.x.ptr, xo + c);
        r.load(p.residual.ptr, ro + c);
        load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
        stream_values<XT, RT, VEC>(x, r, h);
        if constexpr (RT != ROW_NONE) {
            if (p.sum.ptr) {
                if constexpr (RT == ROW_BF16) store_bf16<VEC>(p.sum.ptr, so + c, h);
                else store_f32<VEC>(p.sum.ptr, so + c, h);
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sum = fmaf(h[e], h[e], sum);
            if (eight) top = max_nan(top, fabsf(h[e] * g[e]));
        }
    }
    const RowSums s = reduce_row<1024>(sum, top, scratch);
    const RowFactors f = row_factors(p, s, row);
    if (p.scale && threadIdx.x == 0) p.scale[row] = f.scale;
#pragma unroll 1
    for (uint32_t c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
        float g[VEC], h[VEC];
        load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
        bool kept = false;
        if constexpr (RT != ROW_NONE) {
            if (p.sum.ptr) {
                RowPiece<RT, VEC> r;
                r.load(p.sum.ptr, so + c);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[e] = r.value(e);
                kept = true;
            }
        }
        if (!kept) {
            RowPiece<XT, VEC> x;
            RowPiece<RT, VEC> r;
            x.load(p.x.ptr, xo + c);
            r.load(p.residual.ptr, ro + c);
            stream_values<XT, RT, VEC>(x, r, h);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[e] *= g[e];
        store_row_piece<VEC>(p, oo + c, h, f);
    }
}

// ------------------------------------------------------------------------------------------ gradient
// With a = dy * gamma, u = x * inv:  dx = inv * (a - u * mean(a * u)) + dsum,  dgamma = sum over rows of dy * u.
// mean(a * u) = inv * mean(a * x), so both sums of a row (x^2 and a * x) are taken in one pass. A block walks rows b, b +
// blocks, ...; every thread keeps the sums of its own columns of dgamma, and the block's partial sums (one row of `partial`)
// are added in a fixed order by column_sums: results do not depend on timing.
template <int XT, int DT_, int VEC, int NV, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T) norm_grad_kernel(const __grid_constant__ NormGradParams p) {
    constexpr int kRowsPerBlock = T == 32 ? 4 : 1;
    __shared__ float2 scratch[2][32];
    extern __shared__ float block_sums[];   // T == 32: [cols], the four warps' sums of dgamma
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tid = T == 32 ? (threadIdx.x & 31) : threadIdx.x;
    const uint32_t sub = T == 32 ? (threadIdx.x >> 5) : 0;
    float acc[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[i][e] = 0.0f;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x * kRowsPerBlock + sub; row < p.rows; row += gridDim.x * kRowsPerBlock, turn ^= 1) {
        const uint64_t xo = row_offset(p.x, row, p.dims, p.flat), yo = row_offset(p.dy, row, p.dims, p.flat);
        const uint64_t so = DT_ != ROW_NONE ? row_offset(p.dsum, row, p.dims, p.flat) : 0;
        RowPiece<XT, VEC> xs[NV], ys[NV];
        RowPiece<DT_, VEC> ds[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = (i * T + tid) * VEC;
            if (c < p.cols) {
                xs[i].load(p.x.ptr, xo + c);
                ys[i].load(p.dy.ptr, yo + c);
                ds[i].load(p.dsum.ptr, so + c);
            }
        }
        float squares = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = (i * T + tid) * VEC;
            if (c < p.cols) {
                float g[VEC];
                load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float x = xs[i].value(e);
                    squares = fmaf(x, x, squares);
                    dot = fmaf(ys[i].value(e) * g[e], x, dot);
                }
            }
        }
        const float2 s = reduce_row2<T>(squares, dot, scratch[turn]);   // two buffers: the next row's sums may start before all have read
        const float inv = inverse_rms(s.x, p.cols, p.eps);
        const float mean_au = __fdiv_rn(s.y, float(p.cols)) * inv;
        const uint64_t oo = row_offset(p.dx, row, p.dims, p.flat);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = (i * T + tid) * VEC;
            if (c < p.cols) {
                float g[VEC], d[VEC];
                load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float u = xs[i].value(e) * inv, y = ys[i].value(e);
                    d[e] = (y * g[e] - u * mean_au) * inv;
                    if constexpr (DT_ != ROW_NONE) d[e] += ds[i].value(e);
                    acc[i][e] = fmaf(y, u, acc[i][e]);
                }
                if (p.dx.type == ROW_BF16) store_bf16<VEC>(p.dx.ptr, oo + c, d);
                else store_f32<VEC>(p.dx.ptr, oo + c, d);
            }
        }
    }
    if (!p.partial) return;
    float* mine = p.partial + uint64_t(blockIdx.x) * p.cols;
    if constexpr (T == 32) {
        for (uint32_t w = 0; w < 4; ++w) {   // the warps add their sums in turn: the order is fixed
            if (sub == w) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const uint32_t c = (i * T + tid) * VEC;
                    if (c < p.cols) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) block_sums[c + e] = w ? block_sums[c + e] + acc[i][e] : acc[i][e];
                    }
                }
            }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < p.cols; c += blockDim.x) mine[c] = block_sums[c];
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = (i * T + tid) * VEC;
            if (c < p.cols) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) mine[c + e] = acc[i][e];
            }
        }
    }
}
// Rows too long for registers: both passes read from memory, the sums of dgamma are kept in the block's row of `partial`
// (every thread its own columns, so no two threads touch a word).
template <int XT, int DT_, int VEC>
__global__ void __launch_bounds__(1024) norm_grad_long_kernel(const __grid_constant__ NormGradParams p) {
    __shared__ float2 scratch[2][32];
    griddep_wait();
    griddep_launch_dependents();
    float* mine = p.partial ? p.partial + uint64_t(blockIdx.x) * p.cols : nullptr;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const uint64_t xo = row_offset(p.x, row, p.dims, p.flat), yo = row_offset(p.dy, row, p.dims, p.flat);
        const uint64_t so = DT_ != ROW_NONE ? row_offset(p.dsum, row, p.dims, p.flat) : 0, oo = row_offset(p.dx, row, p.dims, p.flat);
        float squares = 0.0f, dot = 0.0f;
#pragma unroll 1
        for (uint32_t c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
            RowPiece<XT, VEC> xs, ys;
            float g[VEC];
            xs.load(p.x.ptr, xo + c);
            ys.load(p.dy.ptr, yo + c);
            load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = xs.value(e);
                squares = fmaf(x, x, squares);
                dot = fmaf(ys.value(e) * g[e], x, dot);
            }
        }
        const float2 s = reduce_row2<1024>(squares, dot, scratch[turn]);
        const float inv = inverse_rms(s.x, p.cols, p.eps);
        const float mean_au = __fdiv_rn(s.y, float(p.cols)) * inv;
        const bool first = row == blockIdx.x;
#pragma unroll 1
        for (uint32_t c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
            RowPiece<XT, VEC> xs, ys;
            RowPiece<DT_, VEC> ds;
            float g[VEC], d[VEC];
            xs.load(p.x.ptr, xo + c);
            ys.load(p.dy.ptr, yo + c);
            ds.load(p.dsum.ptr, so + c);
            load_gamma<VEC>(g, p.gamma, p.gamma_type, c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float u = xs.value(e) * inv, y = ys.value(e);
                d[e] = (y * g[e] - u * mean_au) * inv;
                if constexpr (DT_ != ROW_NONE) d[e] += ds.value(e);
                if (mine) mine[c + e] = first ? y * u : fmaf(y, u, mine[c + e]);
            }
            if (p.dx.type == ROW_BF16) store_bf16<VEC>(p.dx.ptr, oo + c, d);
            else store_f32<VEC>(p.dx.ptr, oo + c, d);
        }
    }
}
// out[c] = sum over blocks, in block order within each of eight interleaved shares, then share by share: a fixed order.
__device__ __forceinline__ void column_sums(const float* partial, float* out, uint32_t blocks, uint32_t cols) {
    __shared__ float part[8][33];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, share = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (uint32_t b = share; b < blocks; b += 8) s += partial[uint64_t(b) * cols + c];
    }
    part[share][lane] = s;
    __syncthreads();
    if (share == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += part[i][lane];
        out[c] = s;
    }
}

// ------------------------------------------------------------------------------------------ columns, transposed
// One step per column of x, result transposed. First the columns' maxima (as bit patterns, whose order is the values'; a NaN's
// is above infinity's, so it stays), then the codes through a tile in shared memory, then the steps in place of the maxima.
template <int XT>
__global__ void __launch_bounds__(256) column_max_kernel(const __grid_constant__ QuantTransParams p) {
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t c = blockIdx.x * 32 + (threadIdx.x & 31);
    const uint32_t rows_per = (p.rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * rows_per, r1 = min(p.rows, r0 + rows_per);
    __shared__ float part[8][33];
    float top = 0.0f;
    if (c < p.cols) {
#pragma unroll 4
        for (uint32_t r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
            RowPiece<XT, 1> x;
            x.load(p.x, uint64_t(r) * p.x_ld + c);
            top = max_nan(top, fabsf(x.value(0)));
        }
    }
    part[threadIdx.x >> 5][threadIdx.x & 31] = top;
    __syncthreads();
    if (threadIdx.x < 32 && c < p.cols) {
#pragma unroll
        for (int i = 1; i < 8; ++i) top = max_nan(top, part[i][threadIdx.x]);
        atomicMax(reinterpret_cast<uint32_t*>(p.scale) + c, __float_as_uint(top) & 0x7FFFFFFFu);
    }
}
template <int XT>
__global__ void __launch_bounds__(256) quant_trans_kernel(const __grid_constant__ QuantTransParams p) {
    __shared__ uint8_t tile[64][68];   // [column][row]
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
    const uint32_t cl = threadIdx.x & 63, c = c0 + cl;
    if (c < p.cols) {
        const RowStep s = make_row_step(p.given ? p.given[uint64_t(c) * p.given_stride] : __fdiv_rn(p.scale[c], p.top));
#pragma unroll 4
        for (uint32_t i = threadIdx.x >> 6; i < 64; i += 4) {
            if (r0 + i < p.rows) {
                RowPiece<XT, 1> x;
                x.load(p.x, uint64_t(r0 + i) * p.x_ld + c);
                const float v[1] = {x.value(0)};
                store_codes<1>(&tile[0][0], cl * 68 + i, v, p.out_type, s, p.hw);
            }
        }
    }
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = threadIdx.x >> 6; i < 64; i += 4) {
        const uint32_t r = threadIdx.x & 63;
        if (c0 + i < p.cols && r0 + r < p.rows) static_cast<uint8_t*>(p.out)[uint64_t(c0 + i) * p.out_ld + r0 + r] = tile[i][r];
    }
}
__device__ __forceinline__ void column_steps(float* scale, uint32_t cols, float top) {
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c < cols) {
        const float s = __fdiv_rn(scale[c], top);
        scale[c] = s < __uint_as_float(0x7F800000u) ? s : __uint_as_float(0x7FC00000u);
    }
}

}  // namespace mmeb200
