// Row kernels around the 8-bit products: RMS norm with the residual's addition and an optional 8-bit output, its gradient,
// and row-wise quantisation. All of them are bound by HBM: a row is read once, kept in registers while its sums are taken,
// and written once.
//
// Norm of one row, in 32 bits (h: the row as the residual stream keeps it, after its rounding to the stream's type):
//     inv = 1 / sqrt(mean(h^2) + eps),  v = h * gamma,  y = v * inv.
// 8-bit output: with a = max |v|, step = a / top, every code is the nearest representable value to the 32-bit quotient
// v / step (ties to even), and the row's scale is step * inv. inv does not enter the codes, so sum and maximum are taken in
// one pass, and the codes do not depend on the order of any sum: they are fixed by the definition, bit for bit.
//
// A row takes a warp (up to 1024 columns), a block (32 columns a thread, 64 past 16384), or a loop that reads it twice. Blocks are
// not kept over rows: the next row's loads come from the block beside it, two of 512 threads per SM. Measured against what has to
// be read and written at 6549 GB/s: 8192 x 8192 bf16 with residual to int8 71.8 us (100 %), 16384 x 4096 with an fp32 residual to
// bf16 121 us (102 %), quantisation of 2048 x 28672 bf16 33.5 us (80 %) and 8192 x 8192 fp32 52.8 us (97 %).
// Odd rows shift gamma's words for every row, and their block forms of a bf16 stream spill 28 to 108 bytes at 64 registers; beside
// even rows of about the same length: 8192 x 4999 bf16 with residual to int8 57 us (bf16 gamma) and 61 us (fp32 gamma), 46 us at
// 5000 columns; without a residual 41 and 31 us; 8192 x 8191 without a residual 72 us (43 %: seven columns of phase make a ninth
// warp, three blocks per SM in place of four), 48 us at 8192; 2048 x 20001 fp32 without a residual 94 us (33 %), 66 us at 20000.
// Short rows: 200000 of 128 columns take 54 us (22 %), of 129 columns 93 us (13 %): a block lives for four rows, and at 128 columns
// half of a warp's lanes have no element. Codes under given scales are divided for, out of line: 8192 x 8192 bf16 with residual to
// int8 101 us and to fp8 106 us.
#pragma once
#include <type_traits>

#include "norm_quant.h"
#include "ptx_sm100.cuh"

namespace mmeb200 {

// ------------------------------------------------------------------------------------------ elements
// A warp works on steps of 256 consecutive columns, a lane on eight of them. VEC says how rows allow elements to be moved.
// 8: every row starts and ends on eight elements, one or two 16-byte accesses per tensor and step. kPhased: rows start anywhere,
// but the same distance (the phase) past eight elements in every tensor, as rows of an odd length that lie one behind the other do:
// columns are counted from the boundary before the row, and all but the pieces at a row's two ends move as with 8. 1: element by
// element, a lane's elements 32 columns apart so that a warp's accesses stay contiguous. (bf16 rows of 4999 columns to int8 with a
// residual and an fp32 gamma, 8192 of them: 61 us phased, 83 us one by one; 5000 columns take 46 us.)
template <int TYPE>
struct RowElem;
template <> struct RowElem<ROW_BF16> { static constexpr int kBytes = 2; };
template <> struct RowElem<ROW_F32> { static constexpr int kBytes = 4; };
template <> struct RowElem<ROW_I8> { static constexpr int kBytes = 1; };   // codes of either kind

// The columns of a row as its lanes count them: [phase, end).
template <int VEC>
struct RowSpan {
    static constexpr uint32_t phase = 0;
    uint32_t end;
    __device__ __forceinline__ RowSpan(const void*, int, uint32_t cols) : end(cols) {}
    __device__ __forceinline__ bool touches(uint32_t, uint32_t) const { return true; }
};
template <>
struct RowSpan<kPhased> {
    uint32_t phase, end;
    __device__ __forceinline__ RowSpan(const void* row, int bytes, uint32_t cols) : phase(uint32_t(reinterpret_cast<uintptr_t>(row) / bytes) & 7u), end(cols + phase) {}
    __device__ __forceinline__ bool whole(uint32_t c) const { return c >= phase && c + 8 <= end; }
    __device__ __forceinline__ bool has(uint32_t c) const { return c >= phase && c < end; }
    __device__ __forceinline__ bool touches(uint32_t c, uint32_t n) const { return c + n > phase && c < end; }
};

// Column of element e of this lane within a step.
template <int VEC>
__device__ __forceinline__ uint32_t lane_column(int e) { return VEC == 1 ? uint32_t(e) * 32 + (threadIdx.x & 31) : (threadIdx.x & 31) * 8 + uint32_t(e); }

// Whether a lane has anything to do in the step at c0. With VEC = 1 it is the same for all lanes and the elements are looked at one
// by one.
template <int VEC>
__device__ __forceinline__ bool in_row(uint32_t c0, const RowSpan<VEC>& span) { return c0 + (VEC == 1 ? 0 : (threadIdx.x & 31) * 8) < span.end; }

template <int TYPE>
__device__ __forceinline__ uint32_t load_element(const uint8_t* a) {
    if constexpr (TYPE == ROW_BF16) return *reinterpret_cast<const uint16_t*>(a);
    else return *reinterpret_cast<const uint32_t*>(a);
}
template <int TYPE, int W>
__device__ __forceinline__ void store_element(uint8_t* a, const uint32_t (&w)[W], int e) {
    if constexpr (TYPE == ROW_F32) *reinterpret_cast<uint32_t*>(a) = w[e];
    else if constexpr (TYPE == ROW_BF16) *reinterpret_cast<uint16_t*>(a) = uint16_t(w[e >> 1] >> (16 * (e & 1)));
    else *a = uint8_t(w[e >> 2] >> (8 * (e & 3)));
}
// The eight elements of a lane, packed. Columns from `c0` on (in_row); those outside the span read as zeros, of a phased row once
// trim_piece has cleared them: there the aligned 16 bytes around a row's ends are read whole (none without a byte of the row), so
// that no lane goes another way while loads are issued (a branch for the ends: 79 us where this took 71, 8192 x 4999 bf16 with a
// residual to int8 and an fp32 gamma, before gamma was fetched ahead: 61 us since). Such a word lies in the page of the byte it shares with the row. `row` is where column 0 would be.
template <int TYPE, int VEC, int W>
__device__ __forceinline__ void load_piece(const void* row, uint32_t c0, const RowSpan<VEC>& span, uint32_t (&w)[W]) {
    constexpr int kBytes = RowElem<TYPE>::kBytes;
    static_assert(W == 2 * kBytes, "packed words");
    const uint32_t c = c0 + lane_column<VEC>(0);
    const uint8_t* a = static_cast<const uint8_t*>(row) + uint64_t(c) * kBytes;
    if constexpr (VEC != 1) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (VEC == 8 || span.touches(c + i * (16 / kBytes), 16 / kBytes)) q = reinterpret_cast<const uint4*>(a)[i];
            w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
        }
    } else {
        uint32_t t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = c + e * 32 < span.end ? load_element<TYPE>(a + e * 32 * kBytes) : 0u;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = TYPE == ROW_BF16 ? __byte_perm(t[2 * i % 8], t[(2 * i + 1) % 8], 0x5410) : t[i % 8];
    }
}
template <int TYPE, int VEC, int W>
__device__ __forceinline__ void trim_piece(uint32_t c0, const RowSpan<VEC>& span, uint32_t (&w)[W]) {
    if constexpr (VEC == kPhased) {
        const uint32_t c = c0 + lane_column<VEC>(0);
        if (!span.whole(c)) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if constexpr (TYPE == ROW_BF16) w[i] &= (span.has(c + 2 * i) ? 0xFFFFu : 0u) | (span.has(c + 2 * i + 1) ? 0xFFFF0000u : 0u);
                else w[i] = span.has(c + i) ? w[i] : 0u;
            }
        }
    }
}
template <int TYPE, int VEC, int W>
__device__ __forceinline__ void store_piece(void* row, uint32_t c0, const RowSpan<VEC>& span, const uint32_t (&w)[W]) {
    constexpr int kBytes = RowElem<TYPE>::kBytes;
    static_assert(W == 2 * kBytes, "packed words");
    const uint32_t c = c0 + lane_column<VEC>(0);
    uint8_t* a = static_cast<uint8_t*>(row) + uint64_t(c) * kBytes;
    bool whole = VEC == 8;
    if constexpr (VEC == kPhased) whole = span.whole(c);
    if (whole) {
        if constexpr (W == 2) *reinterpret_cast<uint2*>(a) = make_uint2(w[0], w[1]);
        else {
#pragma unroll
            for (int i = 0; i < W / 4; ++i) reinterpret_cast<uint4*>(a)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t d = lane_column<VEC>(e) - lane_column<VEC>(0);
            bool there = c + d < span.end;
            if constexpr (VEC == kPhased) there = span.has(c + d);
            if (there) store_element<TYPE>(a + d * kBytes, w, e);
        }
    }
}
// The same to rows that keep no phase (fp32 partial sums, counted from the row's first column).
template <int VEC>
__device__ __forceinline__ void store_floats(float* row, uint32_t c0, const RowSpan<VEC>& span, const uint32_t (&w)[8]) {
    if constexpr (VEC != kPhased) store_piece<ROW_F32, VEC>(row, c0, span, w);
    else {
        const uint32_t c = c0 + lane_column<VEC>(0);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (span.has(c + e)) reinterpret_cast<uint32_t*>(row)[c + e - span.phase] = w[e];
    }
}
template <int VEC>
__device__ __forceinline__ void load_floats(const float* row, uint32_t c0, const RowSpan<VEC>& span, uint32_t (&w)[8]) {
    if constexpr (VEC != kPhased) load_piece<ROW_F32, VEC>(row, c0, span, w);
    else {
        const uint32_t c = c0 + lane_column<VEC>(0);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = span.has(c + e) ? reinterpret_cast<const uint32_t*>(row)[c + e - span.phase] : 0u;
    }
}

// The eight elements are worked on as four pairs: sm_100a adds and multiplies two floats per instruction, and the row kernels
// are as near the issue rate as they are to HBM's.
template <int TYPE, int W>
__device__ __forceinline__ void unpack(const uint32_t (&w)[W], float2 (&f)[4]) {
    static_assert(W == 2 * RowElem<TYPE>::kBytes, "packed words");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == ROW_F32) f[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ uint32_t pack_bf16(float2 v) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(v.y), "f"(v.x));
    return w;
}
template <int TYPE, int W>
__device__ __forceinline__ void pack(const float2 (&f)[4], uint32_t (&w)[W]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == ROW_F32) { w[2 * i] = __float_as_uint(f[i].x); w[2 * i + 1] = __float_as_uint(f[i].y); }
        else w[i] = pack_bf16(f[i]);
    }
}
// gamma is read by every row and sits in the caches; its type is a runtime value. It has no phase: a phased row's eight elements
// are cut out of the aligned words around them. Its words are fetched a step ahead of their use, before anything of the step
// before is stored: past a store that might be to gamma the compiler moves no load.
template <int VEC>
struct GammaWords { uint32_t t[VEC == kPhased ? 12 : 8]; };
template <int TYPE, int VEC>
__device__ __forceinline__ void fetch_gamma_of(const void* gamma, uint32_t c0, const RowSpan<VEC>& span, GammaWords<VEC>& g) {
    constexpr int kBytes = RowElem<TYPE>::kBytes, kWord = 16 / kBytes;   // elements per 16-byte access
    const uint8_t* base = static_cast<const uint8_t*>(gamma);
    const uint32_t c = c0 + lane_column<VEC>(0);
    if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g.t[e] = c + e * 32 < span.end ? load_element<TYPE>(base + uint64_t(c + e * 32) * kBytes) : 0u;
    } else {
        constexpr int kWords = (TYPE == ROW_BF16 ? 1 : 2) + (VEC == kPhased ? 1 : 0);
        // phased: words outside the row are never used; the nearest inside stands for them
        const int first = int(c) - int((span.phase + kWord - 1) & ~(kWord - 1u)), last = int((span.end - span.phase - 1) & ~(kWord - 1u));
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint4* at = reinterpret_cast<const uint4*>(base + uint64_t(c) * kBytes) + i;
            if constexpr (VEC == kPhased) at = reinterpret_cast<const uint4*>(base + uint64_t(uint32_t(min(max(first + i * kWord, 0), last))) * kBytes);
            const uint4 q = *at;
            g.t[4 * i] = q.x; g.t[4 * i + 1] = q.y; g.t[4 * i + 2] = q.z; g.t[4 * i + 3] = q.w;
        }
    }
}
template <int TYPE, int VEC>
__device__ __forceinline__ void gamma_values_of(uint32_t c0, const RowSpan<VEC>& span, const GammaWords<VEC>& g, float2 (&v)[4]) {
    constexpr int W = 2 * RowElem<TYPE>::kBytes;
    uint32_t w[W];
    if constexpr (VEC == 1) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = TYPE == ROW_BF16 ? __byte_perm(g.t[2 * i % 8], g.t[(2 * i + 1) % 8], 0x5410) : g.t[i % 8];
    } else if constexpr (VEC == 8) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = g.t[i];
    } else {
        constexpr uint32_t kWord = TYPE == ROW_BF16 ? 8 : 4, kUnit = TYPE == ROW_BF16 ? 2 : 1;   // elements of 16 and of 4 bytes
        constexpr int kHave = TYPE == ROW_BF16 ? 8 : 12;
        const uint32_t cut = (0u - span.phase) & (kWord - 1);
        uint32_t t[kHave];
#pragma unroll
        for (int i = 0; i < kHave; ++i) t[i] = g.t[i];
#pragma unroll
        for (int step = 2; step > 0; step /= 2) {
            const bool move = cut & (step * kUnit);
#pragma unroll
            for (int i = 0; i + step < kHave; ++i) t[i] = move ? t[i + step] : t[i];
        }
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = TYPE == ROW_BF16 ? __funnelshift_r(t[i], t[i + 1], (cut & 1) * 16) : t[i];
        trim_piece<TYPE, VEC>(c0, span, w);   // (a NaN there would pass into the row's maximum)
    }
    unpack<TYPE>(w, v);
}
template <int VEC>
__device__ __forceinline__ void fetch_gamma(const RowTensor& gamma, uint32_t c0, const RowSpan<VEC>& span, GammaWords<VEC>& g) {
    if (!in_row<VEC>(c0, span)) return;
    if (gamma.type == ROW_BF16) fetch_gamma_of<ROW_BF16, VEC>(gamma.ptr, c0, span, g);
    else fetch_gamma_of<ROW_F32, VEC>(gamma.ptr, c0, span, g);
}
template <int VEC>
__device__ __forceinline__ void gamma_values(const RowTensor& gamma, uint32_t c0, const RowSpan<VEC>& span, const GammaWords<VEC>& g, float2 (&v)[4]) {
    if (gamma.type == ROW_BF16) gamma_values_of<ROW_BF16, VEC>(c0, span, g, v);
    else gamma_values_of<ROW_F32, VEC>(c0, span, g, v);
}
// Both at once.
template <int TYPE, int VEC>
__device__ __forceinline__ void load_gamma_of(const void* gamma, uint32_t c0, const RowSpan<VEC>& span, float2 (&v)[4]) {
    GammaWords<VEC> g;
    fetch_gamma_of<TYPE, VEC>(gamma, c0, span, g);
    gamma_values_of<TYPE, VEC>(c0, span, g, v);
}
template <int VEC>
__device__ __forceinline__ void load_gamma(const RowTensor& gamma, uint32_t c0, const RowSpan<VEC>& span, float2 (&v)[4]) {
    if (gamma.type == ROW_BF16) load_gamma_of<ROW_BF16, VEC>(gamma.ptr, c0, span, v);
    else load_gamma_of<ROW_F32, VEC>(gamma.ptr, c0, span, v);
}
// A walk over a row's steps that takes gamma from the words fetched AHEAD, or (rows that need all registers) as it goes.
template <int VEC, bool GAMMA, bool AHEAD>
struct GammaWalk {
    GammaWords<VEC> words;
    __device__ __forceinline__ GammaWalk(const RowTensor& gamma, uint32_t c, const RowSpan<VEC>& span) {
        if constexpr (GAMMA && AHEAD) fetch_gamma<VEC>(gamma, c, span, words);
    }
    // h *= gamma of the step at c, where `of` is what the walk held before it went on to the next
    static __device__ __forceinline__ void multiply(const GammaWalk& of, const RowTensor& gamma, uint32_t c, const RowSpan<VEC>& span, float2 (&h)[4]) {
        if constexpr (GAMMA) {
            float2 g[4];
            if constexpr (AHEAD) gamma_values<VEC>(gamma, c, span, of.words, g);
            else load_gamma<VEC>(gamma, c, span, g);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __fmul2_rn(h[i], g[i]);
        }
    }
};

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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

template <int TYPE>
__device__ __forceinline__ uint8_t* row_of(const RowTensor& t, uint32_t row, const uint32_t (&dims)[4], uint32_t flat) {
    return static_cast<uint8_t*>(t.ptr) + row_offset(t, row, dims, flat) * RowElem<TYPE>::kBytes;
}

// ------------------------------------------------------------------------------------------ 8-bit codes
// How values become codes: `step`, and minus its reciprocal. 0: no codes (a step that is zero, negative or no finite number);
// NaN: so large or small a step that the quotient has to be divided for.
struct CodeStep {
    float step, nrecip;
};
__device__ __forceinline__ CodeStep make_code_step(float step) {
    CodeStep s;
    s.step = step;
    if (!(step > 0.0f && step < __uint_as_float(0x7F800000u))) s.nrecip = 0.0f;
    else s.nrecip = (step >= 0x1p-60f && step <= 0x1p60f) ? -__frcp_rn(step) : __uint_as_float(0x7FC00000u);
    return s;
}
constexpr float kRoundMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to the nearest whole number, ties to even

__device__ __forceinline__ uint32_t pack_low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
// Minus the correctly rounded quotients v / step, in two operations more than a multiplication: with y the correctly rounded
// reciprocal and q = v * y, the remainder r = v - q * step is exact in one fused multiply-add, and q + r * y rounds to the
// quotient (P. W. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, IBM J. Res. Dev. 34,
// 1990). Steps between 2^-60 and 2^60 keep every remainder that can decide a code a normal number. Worked with the sign
// turned, zeros keep theirs.
__device__ __forceinline__ float2 minus_quotient(float2 v, const CodeStep& s) {
    const float2 q = __fmul2_rn(v, both(s.nrecip)), r = __ffma2_rn(q, both(s.step), v);
    return __ffma2_rn(r, both(s.nrecip), q);
}
__device__ __forceinline__ uint32_t int8_codes(float2 nq0, float2 nq1) {   // |quotient| <= 127
    const float2 a = __ffma2_rn(nq0, both(-1.0f), both(kRoundMagic)), b = __ffma2_rn(nq1, both(-1.0f), both(kRoundMagic));
    return pack_low_bytes(a.x, a.y, b.x, b.y);
}
// Four fp8 codes of quotients that stay below the hardware conversion's own limit (hw.scale: the exponent bias).
__device__ __forceinline__ uint32_t fp8_codes(float2 nq0, float2 nq1, const Fp8HwCast& hw) {
    const float2 a = __fmul2_rn(nq0, both(hw.scale)), b = __fmul2_rn(nq1, both(hw.scale));
    uint16_t lo, hi;
    if (hw.e5m2) {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
    } else {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
    }
    return (uint32_t(lo) | uint32_t(hi) << 16) ^ 0x80808080u;
}
// Four codes under any step and of any value: given steps, steps of extreme size, conventions whose codes pass the hardware's.
template <bool I8>
static __device__ __noinline__ uint32_t codes_by_division(float v0, float v1, float v2, float v3, float step, const Fp8HwCast& hw) {
    float t[4] = {__fdiv_rn(v0, step), __fdiv_rn(v1, step), __fdiv_rn(v2, step), __fdiv_rn(v3, step)};
    if constexpr (I8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = t[e] == t[e] ? fminf(fmaxf(t[e], -127.0f), 127.0f) + kRoundMagic : kRoundMagic;   // a NaN has no code
        return pack_low_bytes(t[0], t[1], t[2], t[3]);
    } else {
        return f32x4_to_fp8_hw(t, hw);
    }
}
// SURE: the step is the values' own (no quotient beyond the largest code) and has a reciprocal (fast_step).
template <bool I8, bool SURE>
__device__ __forceinline__ uint32_t make_codes(float2 v0, float2 v1, const CodeStep& s, const Fp8HwCast& hw) {
    if constexpr (SURE) {
        if constexpr (I8) return int8_codes(minus_quotient(v0, s), minus_quotient(v1, s));
        else return fp8_codes(minus_quotient(v0, s), minus_quotient(v1, s), hw);
    } else {
        return s.nrecip == 0.0f ? 0u : codes_by_division<I8>(v0.x, v0.y, v1.x, v1.y, s.step, hw);
    }
}
// (int8: direct = true; fp8: no quotient of a row's own step passes the hardware conversion's limit)
__device__ __forceinline__ bool fast_step(const CodeStep& s, bool direct) { return direct && s.nrecip < 0.0f; }

// ------------------------------------------------------------------------------------------ reductions
// Sums over the threads of a row: a warp, or the `warps` warps of the block (BLOCK). The order is fixed. MAX: the second is a
// maximum that keeps NaN.
template <bool BLOCK, bool MAX>
__device__ __forceinline__ float2 reduce_row(float a, float b, uint32_t warps, float2* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        const float t = __shfl_xor_sync(0xffffffffu, b, o);
        b = MAX ? max_nan(b, t) : b + t;
    }
    if constexpr (BLOCK) {
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = scratch[0].x;
        b = scratch[0].y;
#pragma unroll 4
        for (uint32_t w = 1; w < warps; ++w) {
            const float2 t = scratch[w];
            a += t.x;
            b = MAX ? max_nan(b, t.y) : b + t.y;
        }
    }
    return make_float2(a, b);
}
__device__ __forceinline__ float inverse_rms(float sum_of_squares, float per_col, float eps) {
    return __frsqrt_rn(fmaf(sum_of_squares, per_col, eps));   // per_col: 1 / cols
}

// What a row's sums decide: the factor of float outputs, the step of codes, the scale that is written.
struct RowFactors { float inv; CodeStep step; float scale; };
__device__ __forceinline__ RowFactors row_factors(const NormParams& p, float sum, float top, uint32_t row) {
    RowFactors f;
    f.inv = p.norm ? inverse_rms(sum, p.per_col, p.eps) : 1.0f;
    f.scale = 0.0f;
    if (p.mode == NORM_I8_GIVEN || p.mode == NORM_F8_GIVEN) {
        f.step = make_code_step(p.given[uint64_t(row) * p.given_stride]);
    } else if (p.mode == NORM_I8 || p.mode == NORM_F8) {
        f.step = make_code_step(__fdiv_rn(top, p.top));
        const bool finite = f.step.step < __uint_as_float(0x7F800000u);   // false for NaN
        f.scale = !finite ? __uint_as_float(0x7FC00000u) : f.step.step > 0.0f ? f.step.step * f.inv : 0.0f;
    }
    return f;
}
// The type a row is kept in while its sums are taken: the stream's, or x's where nothing is added. bf16 rows take four
// registers per piece, and their values are exact.
template <int XT, int RT>
struct RowKept {
    static constexpr int kType = RT != ROW_NONE ? RT : XT, kWords = 2 * RowElem<kType>::kBytes;
    uint32_t w[kWords];
    __device__ __forceinline__ void values(float2 (&h)[4]) const { unpack<kType>(w, h); }
};
// Or, for codes of rows that leave registers enough, the finished products h * gamma: gamma is then read once per row.
struct RowProducts {
    float2 v[4];
};
// x + residual, rounded to the stream's type, which is what the norm sees.
template <int XT, int RT>
__device__ __forceinline__ void stream_values(const uint32_t (&x)[2 * RowElem<XT>::kBytes], const uint32_t (&r)[2 * RowElem<RT>::kBytes], RowKept<XT, RT>& h) {
    float2 f[4], g[4];
    unpack<XT>(x, f);
    unpack<RT>(r, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __fadd2_rn(f[i], g[i]);
    pack<RT>(f, h.w);
}
// The rows of a norm's tensors, each from where column 0 would be.
template <int XT, int RT, int VEC>
struct NormRows {
    const uint8_t *x, *residual;
    uint8_t* sum;
    RowSpan<VEC> span;
    __device__ __forceinline__ NormRows(const NormParams& p, uint32_t row) : x(row_of<XT>(p.x, row, p.dims, p.flat)), span(x, RowElem<XT>::kBytes, p.cols) {
        x -= span.phase * RowElem<XT>::kBytes;
        if constexpr (RT != ROW_NONE) {
            residual = row_of<RT>(p.residual, row, p.dims, p.flat) - span.phase * RowElem<RT>::kBytes;
            sum = p.sum.ptr ? row_of<RT>(p.sum, row, p.dims, p.flat) - span.phase * RowElem<RT>::kBytes : nullptr;
        }
    }
};
// COUNT steps of the first pass from column c0 on: all loads first, then the stream's values (kept, and written), then the sums.
// TOPS: the largest |h * gamma| too. Kept: RowKept or RowProducts.
template <int XT, int RT, int VEC, int COUNT, bool TOPS, bool GAMMA, bool AHEAD, typename Kept>
__device__ __forceinline__ void read_steps(const NormParams& p, const NormRows<XT, RT, VEC>& rows, uint32_t c0, Kept* kept, float2& sum, float& top) {
    constexpr int WX = 2 * RowElem<XT>::kBytes, WR = RT != ROW_NONE ? 2 * RowElem<RT != ROW_NONE ? RT : XT>::kBytes : 1;
    uint32_t x[COUNT][WX], r[COUNT][WR];
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        if (in_row<VEC>(c0 + j * 256, rows.span)) {
            load_piece<XT, VEC>(rows.x, c0 + j * 256, rows.span, x[j]);
            if constexpr (RT != ROW_NONE) load_piece<RT, VEC>(rows.residual, c0 + j * 256, rows.span, r[j]);
        }
    }
    using Walk = GammaWalk<VEC, TOPS && GAMMA, AHEAD>;
    Walk gamma(p.gamma, c0, rows.span);
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        const uint32_t c = c0 + j * 256;
        const Walk now = gamma;
        if (j + 1 < COUNT) gamma = Walk(p.gamma, c + 256, rows.span);
        if (in_row<VEC>(c, rows.span)) {
            RowKept<XT, RT> stream;
            trim_piece<XT, VEC>(c, rows.span, x[j]);
            if constexpr (RT != ROW_NONE) {
                trim_piece<RT, VEC>(c, rows.span, r[j]);
                stream_values<XT, RT>(x[j], r[j], stream);
                if (rows.sum) store_piece<RT, VEC>(rows.sum, c, rows.span, stream.w);
            } else {
#pragma unroll
                for (int i = 0; i < WX; ++i) stream.w[i] = x[j][i];
            }
            float2 h[4];
            stream.values(h);
            if (p.norm) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum = __ffma2_rn(h[i], h[i], sum);
            }
            if constexpr (TOPS) {
                Walk::multiply(now, p.gamma, c, rows.span, h);
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max_nan(top, fabsf(h[i].x), fabsf(h[i].y));
            }
            if constexpr (std::is_same_v<Kept, RowProducts>) {
#pragma unroll
                for (int i = 0; i < 4; ++i) kept[j].v[i] = h[i];
            } else {
                kept[j] = stream;
            }
        }
    }
}
// One step of the second pass: the finished values v (h * gamma), as floats or codes.
template <int MODE, bool FAST, int VEC>
__device__ __forceinline__ void write_values(const NormParams& p, uint8_t* out, uint32_t c, const RowSpan<VEC>& span, float2 (&v)[4], const RowFactors& f) {
    constexpr int kType = MODE == NORM_BF16 ? ROW_BF16 : MODE == NORM_F32 ? ROW_F32 : ROW_I8;
    uint32_t w[2 * RowElem<kType>::kBytes];
    if constexpr (MODE != NORM_I8 && MODE != NORM_F8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __fmul2_rn(v[k], both(f.inv));
    }
    if constexpr (MODE == NORM_BF16 || MODE == NORM_F32) pack<kType>(v, w);
    else {
#pragma unroll
        for (int k = 0; k < 2; ++k) w[k] = make_codes<MODE == NORM_I8 || MODE == NORM_I8_GIVEN, FAST>(v[2 * k], v[2 * k + 1], f.step, p.hw);
    }
    store_piece<kType, VEC>(out, c, span, w);
}
template <int MODE, bool FAST, int VEC, int COUNT, bool GAMMA, bool AHEAD, typename Kept>
__device__ __forceinline__ void write_steps(const NormParams& p, uint8_t* out, uint32_t c0, const RowSpan<VEC>& span, const Kept* kept, const RowFactors& f) {
    constexpr bool kProducts = std::is_same_v<Kept, RowProducts>;
    using Walk = GammaWalk<VEC, !kProducts && GAMMA, AHEAD>;
    Walk gamma(p.gamma, c0, span);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const uint32_t c = c0 + i * 256;
        const Walk now = gamma;
        if (i + 1 < COUNT) gamma = Walk(p.gamma, c + 256, span);
        if (in_row<VEC>(c, span)) {
            float2 v[4];
            if constexpr (kProducts) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = kept[i].v[k];
            } else {
                kept[i].values(v);
                Walk::multiply(now, p.gamma, c, span, v);
            }
            write_values<MODE, FAST, VEC>(p, out, c, span, v, f);
        }
    }
}
// What differs between the kinds of output is decided once per row: `write(mode, fast)` is called with the kind as a constant,
// and whether the row's codes can do without a test of the step.
template <bool CODES, typename F>   // CODES: of the row's own step
__device__ __forceinline__ void for_mode(const NormParams& p, const RowFactors& f, F&& write) {
    if constexpr (CODES) {
        if (p.mode == NORM_I8) {
            if (fast_step(f.step, true)) write(std::integral_constant<int, NORM_I8>(), std::true_type());
            else write(std::integral_constant<int, NORM_I8>(), std::false_type());
        } else {
            if (fast_step(f.step, p.fp8_direct)) write(std::integral_constant<int, NORM_F8>(), std::true_type());
            else write(std::integral_constant<int, NORM_F8>(), std::false_type());
        }
    } else {
        switch (p.mode) {
            case NORM_BF16: write(std::integral_constant<int, NORM_BF16>(), std::false_type()); break;
            case NORM_F32: write(std::integral_constant<int, NORM_F32>(), std::false_type()); break;
            case NORM_I8_GIVEN: write(std::integral_constant<int, NORM_I8_GIVEN>(), std::false_type()); break;
            default: write(std::integral_constant<int, NORM_F8_GIVEN>(), std::false_type()); break;
        }
    }
}
__device__ __forceinline__ uint8_t* out_row(const NormParams& p, uint32_t row, uint32_t phase) {
    return static_cast<uint8_t*>(p.out.ptr) + (row_offset(p.out, row, p.dims, p.flat) - phase) * (p.mode == NORM_BF16 ? 2 : p.mode == NORM_F32 ? 4 : 1);
}

// A row per warp (BLOCK = false: four rows per block) or per block, NV steps per warp, kept in registers between the row's one
// read and its one write. Two blocks of 512 threads fit an SM where rows are kept in bf16.
template <int XT, int RT, int VEC, int NV, bool BLOCK, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 && RowKept<XT, RT>::kType == ROW_BF16 ? 2 : 1) norm_kernel(const __grid_constant__ NormParams p) {
    constexpr int G = NV < 2 ? 1 : (VEC != 1 && RT == ROW_NONE) ? NV : (VEC != 1 && XT != ROW_F32 && RT != ROW_F32) ? 4 : 2;   // steps loaded at a time
    __shared__ float2 scratch[32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = BLOCK ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= p.rows) return;   // whole warps, never part of a block that synchronises
    const uint32_t c0 = BLOCK ? (threadIdx.x >> 5) * 256 * NV : 0;
    const NormRows<XT, RT, VEC> rows(p, row);
    auto whole_row = [&](auto codes, auto gamma) {
        constexpr bool kCodes = decltype(codes)::value, kGamma = decltype(gamma)::value, kAhead = NV <= 4;
        std::conditional_t<kCodes && NV <= 4, RowProducts, RowKept<XT, RT>> kept[NV];
        float2 sum = both(0.0f);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i += G) read_steps<XT, RT, VEC, G, kCodes, kGamma, kAhead>(p, rows, c0 + i * 256, kept + i, sum, top);
        const float2 s = reduce_row<BLOCK, true>(sum.x + sum.y, top, blockDim.x >> 5, scratch);
        const RowFactors f = row_factors(p, s.x, s.y, row);
        if (p.scale && (BLOCK ? threadIdx.x : threadIdx.x & 31) == 0) p.scale[row] = f.scale;
        uint8_t* out = out_row(p, row, rows.span.phase);
        for_mode<kCodes>(p, f, [&](auto mode, auto fast) { write_steps<decltype(mode)::value, decltype(fast)::value, VEC, NV, kGamma, kAhead>(p, out, c0, rows.span, kept, f); });
    };
    if (p.mode == NORM_I8 || p.mode == NORM_F8) {
        if (p.gamma.ptr) whole_row(std::true_type(), std::true_type());
        else whole_row(std::true_type(), std::false_type());
    } else {
        if (p.gamma.ptr) whole_row(std::false_type(), std::true_type());
        else whole_row(std::false_type(), std::false_type());
    }
}

// Rows too long for registers: the row is read a second time (from L2, mostly) once its sums are known. The second read
// takes the stream from `sum` where it was written (in place, x and the residual may be gone by then). A thread reads and
// writes the same elements in both passes.
template <int XT, int RT, int VEC>
__global__ void __launch_bounds__(1024) norm_long_kernel(const __grid_constant__ NormParams p) {
    constexpr int KT = RowKept<XT, RT>::kType;
    __shared__ float2 scratch[32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = blockIdx.x, first = (threadIdx.x >> 5) * 256;
    const NormRows<XT, RT, VEC> rows(p, row);
    auto whole_row = [&](auto codes, auto gamma) {
        constexpr bool kCodes = decltype(codes)::value, kGamma = decltype(gamma)::value;
        float2 sum = both(0.0f);
        float top = 0.0f;
#pragma unroll 1
        for (uint32_t c = first; in_row<VEC>(c, rows.span); c += 32 * 256) {
            RowKept<XT, RT> kept;
            read_steps<XT, RT, VEC, 1, kCodes, kGamma, true>(p, rows, c, &kept, sum, top);
        }
        const float2 s = reduce_row<true, true>(sum.x + sum.y, top, 32, scratch);
        const RowFactors f = row_factors(p, s.x, s.y, row);
        if (p.scale && threadIdx.x == 0) p.scale[row] = f.scale;
        uint8_t* out = out_row(p, row, rows.span.phase);
        for_mode<kCodes>(p, f, [&](auto mode, auto fast) {
#pragma unroll 1
            for (uint32_t c = first; in_row<VEC>(c, rows.span); c += 32 * 256) {
                RowKept<XT, RT> kept;
                if constexpr (RT == ROW_NONE) {
                    load_piece<XT, VEC>(rows.x, c, rows.span, kept.w);
                } else if (rows.sum) {
                    load_piece<KT, VEC>(rows.sum, c, rows.span, kept.w);
                } else {
                    uint32_t x[2 * RowElem<XT>::kBytes], r[2 * RowElem<RT != ROW_NONE ? RT : XT>::kBytes];
                    load_piece<XT, VEC>(rows.x, c, rows.span, x);
                    load_piece<RT, VEC>(rows.residual, c, rows.span, r);
                    stream_values<XT, RT>(x, r, kept);
                }
                write_steps<decltype(mode)::value, decltype(fast)::value, VEC, 1, kGamma, true>(p, out, c, rows.span, &kept, f);
            }
        });
    };
    if (p.mode == NORM_I8 || p.mode == NORM_F8) {
        if (p.gamma.ptr) whole_row(std::true_type(), std::true_type());
        else whole_row(std::true_type(), std::false_type());
    } else {
        if (p.gamma.ptr) whole_row(std::false_type(), std::true_type());
        else whole_row(std::false_type(), std::false_type());
    }
}

// ------------------------------------------------------------------------------------------ gradient
// With a = dy * gamma, u = x * inv:  dx = inv * (a - u * mean(a * u)) + dsum,  dgamma = sum over rows of dy * u.
// mean(a * u) = inv * mean(a * x), so both sums of a row (x^2 and a * x) are taken in one pass. A block walks rows b, b +
// blocks, ...; every thread keeps the sums of its own columns of dgamma, and the block's partial sums (one row of `partial`)
// are added in a fixed order by column_sums: results do not depend on timing. HBM bounds it: 16384 x 4096 bf16 67.6 us (91 % of the
// copy rate), 91 us with the sum's gradient (90 %), 2048 x 16384 54 us (76 %, two blocks of a cluster per row); 8000 rows of 1000
// columns 20 us (37 %), where the block's first row and the second launch weigh most. Odd rows: 8192 x 4999 64 us (59 %; 5000 columns
// 49 us), 2048 x 16383 with the sum's 93 us (44 %). fp32 forms keep their pieces in registers and, with the sum's gradient, spill 112
// to 440 bytes: 4096 x 8192 121 us (68 %), 86 us without it (71 %).
//
// a (dy * gamma) becomes dx; acc += dy * u.
template <bool DSUM>
__device__ __forceinline__ void grad_piece(const float2 (&x)[4], const float2 (&y)[4], float2 (&a)[4], const float2 (&add)[4], float inv, float mean_au, float2 (&acc)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 u = __fmul2_rn(x[k], both(inv)), t = __ffma2_rn(u, both(-mean_au), a[k]);
        if constexpr (DSUM) a[k] = __ffma2_rn(t, both(inv), add[k]);
        else a[k] = __fmul2_rn(t, both(inv));
        acc[k] = __ffma2_rn(y[k], u, acc[k]);
    }
}
template <int VEC>
__device__ __forceinline__ void grad_scale(const NormGradParams& p, const float2 (&y)[4], uint32_t c, const RowSpan<VEC>& span, float2 (&a)[4]) {
    if (p.gamma.ptr) {
        load_gamma<VEC>(p.gamma, c, span, a);
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = __fmul2_rn(a[k], y[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = y[k];
    }
}
__device__ __forceinline__ void sum_grad(const float2 (&x)[4], const float2 (&a)[4], float2& squares, float2& dot) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        squares = __ffma2_rn(x[k], x[k], squares);
        dot = __ffma2_rn(a[k], x[k], dot);
    }
}
// A lane's eight sums of dgamma to the block's row of `partial`.
template <int VEC>
__device__ __forceinline__ void store_sums(float* mine, uint32_t c, const RowSpan<VEC>& span, const float2 (&acc)[4]) {
    uint32_t w[8];
    pack<ROW_F32>(acc, w);
    store_floats<VEC>(mine, c, span, w);
}
// The span of a block's (or warp's) rows: all of them have the first one's phase (launch_norm_grad).
template <int XT, int VEC>
__device__ __forceinline__ RowSpan<VEC> grad_span(const NormGradParams& p, uint32_t row) { return RowSpan<VEC>(row_of<XT>(p.x, row, p.dims, p.flat), RowElem<XT>::kBytes, p.cols); }
// How a row is shared: by a warp (four rows per block), a block, or the blocks of a cluster (`ranks` of them, which add their sums
// through each other's shared memory).
enum : int { GRAD_WARP, GRAD_BLOCK, GRAD_CLUSTER, GRAD_REREAD };

// The pieces of a row's tensors (x, dy, dsum), which every thread keeps for itself. FETCHED (bf16 rows that move by 16 bytes): in
// shared memory, copied there a row ahead. Else in registers, loaded when the row begins.
// (16384 x 4096 bf16 with gamma in registers: 67 us, and 91 us with dsum; pieces in registers and gamma read twice per row: 90 and
// 101 us. fp32 pieces would leave an SM half its threads.)
template <int XT, bool DSUM, int VEC, int NV>
struct GradPieces {
    static constexpr bool kFetched = XT == ROW_BF16 && VEC != 1;
    static constexpr int W = 2 * RowElem<XT>::kBytes, kTensors = DSUM ? 3 : 2;
    uint32_t w[kFetched ? 1 : kTensors * NV][W];
    uint4* mine;         // [stage][tensor][step][thread]
    uint32_t stage = 0;
    __device__ __forceinline__ explicit GradPieces(uint4* smem) : mine(smem + threadIdx.x) {}
    __device__ __forceinline__ uint4* slot(uint32_t at, int tensor, int i) const { return mine + ((at * kTensors + tensor) * NV + i) * blockDim.x; }
    // Row `row` into the stage that is not in use; done counts with wait().
    __device__ __forceinline__ void fetch(const NormGradParams& p, uint32_t row, uint32_t c0, const RowSpan<VEC>& span) const {
        if constexpr (kFetched) {
            if (row < p.rows) {
                const RowTensor* t[3] = {&p.x, &p.dy, &p.dsum};
#pragma unroll
                for (int k = 0; k < kTensors; ++k) {
                    const uint8_t* a = row_of<XT>(*t[k], row, p.dims, p.flat) + (int64_t(c0 + lane_column<VEC>(0)) - span.phase) * RowElem<XT>::kBytes;
#pragma unroll
                    for (int i = 0; i < NV; ++i)
                        if (in_row<VEC>(c0 + i * 256, span)) cp_async16(slot(stage ^ 1, k, i), a + i * 256 * RowElem<XT>::kBytes);
                }
            }
            cp_async_commit();
        }
    }
    // The row that is to be worked on.
    __device__ __forceinline__ void begin(const NormGradParams& p, uint32_t row, uint32_t next, uint32_t c0, const RowSpan<VEC>& span) {
        if constexpr (kFetched) {
            stage ^= 1;
            fetch(p, next, c0, span);   // into the stage that the row before left: its values were used up by what was stored
            cp_async_wait<1>();
        } else {
            const RowTensor* t[3] = {&p.x, &p.dy, &p.dsum};
#pragma unroll
            for (int k = 0; k < kTensors; ++k) {
                const uint8_t* a = row_of<XT>(*t[k], row, p.dims, p.flat) - span.phase * RowElem<XT>::kBytes;
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (in_row<VEC>(c0 + i * 256, span)) load_piece<XT, VEC>(a, c0 + i * 256, span, w[k * NV + i]);
            }
        }
    }
    __device__ __forceinline__ void values(int tensor, int i, uint32_t c, const RowSpan<VEC>& span, float2 (&v)[4]) const {
        uint32_t q[W];
        if constexpr (kFetched) {
            const uint4 u = *slot(stage, tensor, i);
            q[0] = u.x; q[1] = u.y; q[2] = u.z; q[3] = u.w;
        } else {
#pragma unroll
            for (int k = 0; k < W; ++k) q[k] = w[tensor * NV + i][k];
        }
        trim_piece<XT, VEC>(c, span, q);
        unpack<XT>(q, v);
    }
};
// XT: type of x, dy, dsum and dx; DSUM: whether there is a gradient of the sum.
template <int XT, bool DSUM, int VEC, int NV, int FORM, int THREADS>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) norm_grad_kernel(const __grid_constant__ NormGradParams p) {
    constexpr bool BLOCK = FORM != GRAD_WARP;
    constexpr int kRowsPerBlock = BLOCK ? 1 : 4, W = 2 * RowElem<XT>::kBytes;
    __shared__ float2 scratch[2][32];
    __shared__ float2 shares[2][8];        // GRAD_CLUSTER: the sums of every block of the cluster
    extern __shared__ uint4 grad_smem[];   // the pieces; GRAD_WARP: then [cols] floats, the four warps' sums of dgamma
    griddep_wait();
    griddep_launch_dependents();
    uint32_t rank = 0, unit = blockIdx.x, units = gridDim.x;
    if constexpr (FORM == GRAD_CLUSTER) {
        rank = cluster_ctarank();
        unit /= p.ranks;
        units /= p.ranks;
        cluster_sync_all();   // all blocks run before the first writes to another's memory
    }
    const uint32_t warp = threadIdx.x >> 5, sub = BLOCK ? 0 : warp, c0 = BLOCK ? (rank * (blockDim.x >> 5) + warp) * 256 * NV : 0;
    float2 acc[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][k] = both(0.0f);
    // a thread's columns are the same in all rows: where its registers do not hold the pieces too, they hold gamma
    constexpr bool kHold = GradPieces<XT, DSUM, VEC, NV>::kFetched;
    float2 gamma[kHold ? NV : 1][4];
    const uint32_t first = unit * kRowsPerBlock + sub, stride = units * kRowsPerBlock;
    const RowSpan<VEC> span = grad_span<XT, VEC>(p, first);
    GradPieces<XT, DSUM, VEC, NV> pieces(grad_smem);
    pieces.fetch(p, first, c0, span);
#pragma unroll
    for (int i = 0; i < (kHold ? NV : 0); ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) gamma[i][k] = both(1.0f);
        if (p.gamma.ptr && in_row<VEC>(c0 + i * 256, span)) load_gamma<VEC>(p.gamma, c0 + i * 256, span, gamma[i]);
    }
    const auto scale = [&](const float2(&y)[4], int i, float2(&a)[4]) {
        if constexpr (kHold) {
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = __fmul2_rn(y[k], gamma[i][k]);
        } else {
            grad_scale<VEC>(p, y, c0 + i * 256, span, a);
        }
    };
    uint32_t turn = 0;
    for (uint32_t row = first; row < p.rows; row += stride, turn ^= 1) {
        pieces.begin(p, row, row + stride, c0, span);
        float2 squares = both(0.0f), dot = both(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = c0 + i * 256;
            if (in_row<VEC>(c, span)) {
                float2 x[4], y[4], a[4];
                pieces.values(0, i, c, span, x);
                pieces.values(1, i, c, span, y);
                scale(y, i, a);
                sum_grad(x, a, squares, dot);
            }
        }
        // two buffers: the next row's sums may start before all have read
        float2 s = reduce_row<BLOCK, false>(squares.x + squares.y, dot.x + dot.y, blockDim.x >> 5, scratch[turn]);
        if constexpr (FORM == GRAD_CLUSTER) {
            if (threadIdx.x < p.ranks) st_shared_cluster_f2(mapa_shared(smem_u32(&shares[turn][rank]), threadIdx.x), s);
            __syncwarp();
            cluster_sync_all();
            s = shares[turn][0];
            for (uint32_t r = 1; r < p.ranks; ++r) s = __fadd2_rn(s, shares[turn][r]);
        }
        const float inv = inverse_rms(s.x, p.per_col, p.eps);
        const float mean_au = s.y * p.per_col * inv;
        uint8_t* out = row_of<XT>(p.dx, row, p.dims, p.flat) - span.phase * RowElem<XT>::kBytes;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = c0 + i * 256;
            if (in_row<VEC>(c, span)) {
                float2 x[4], y[4], a[4], add[4];
                pieces.values(0, i, c, span, x);
                pieces.values(1, i, c, span, y);
                if constexpr (DSUM) pieces.values(2, i, c, span, add);
                scale(y, i, a);
                grad_piece<DSUM>(x, y, a, add, inv, mean_au, acc[i]);
                uint32_t w[W];
                pack<XT>(a, w);
                store_piece<XT, VEC>(out, c, span, w);
            }
        }
    }
    if (!p.partial) return;
    float* mine = p.partial + uint64_t(unit) * p.cols;
    if constexpr (!BLOCK) {
        float* block_sums = reinterpret_cast<float*>(grad_smem + (GradPieces<XT, DSUM, VEC, NV>::kFetched ? 2 * GradPieces<XT, DSUM, VEC, NV>::kTensors * NV * THREADS : 0));
        for (uint32_t w = 0; w < 4; ++w) {   // the warps add their sums in turn: the order is fixed
            if (sub == w) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t c = i * 256 + lane_column<VEC>(e) - span.phase;   // (below the phase: past any column)
                        const float v = (e & 1) ? acc[i][e >> 1].y : acc[i][e >> 1].x;
                        if (c < p.cols) block_sums[c] = w ? block_sums[c] + v : v;
                    }
            }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < p.cols; c += blockDim.x) mine[c] = block_sums[c];
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (in_row<VEC>(c0 + i * 256, span)) store_sums<VEC>(mine, c0 + i * 256, span, acc[i]);
    }
}
// Rows too long even for a cluster: both passes read from memory and the sums of dgamma live in the block's row of `partial`.
template <int XT, bool DSUM, int VEC>
__global__ void __launch_bounds__(512, 2) norm_grad_loop_kernel(const __grid_constant__ NormGradParams p) {
    constexpr int W = 2 * RowElem<XT>::kBytes;
    __shared__ float2 scratch[2][32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t first = (threadIdx.x >> 5) * 256, stride = (blockDim.x >> 5) * 256;
    float* mine = p.partial ? p.partial + uint64_t(blockIdx.x) * p.cols : nullptr;
    const RowSpan<VEC> span = grad_span<XT, VEC>(p, blockIdx.x);
    const uint32_t shift = span.phase * RowElem<XT>::kBytes;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const uint8_t *xr = row_of<XT>(p.x, row, p.dims, p.flat) - shift, *yr = row_of<XT>(p.dy, row, p.dims, p.flat) - shift;
        const uint8_t* sr = DSUM ? row_of<XT>(p.dsum, row, p.dims, p.flat) - shift : nullptr;
        float2 squares = both(0.0f), dot = both(0.0f);
#pragma unroll 2
        for (uint32_t c = first; in_row<VEC>(c, span); c += stride) {
            uint32_t xw[W], yw[W];
            float2 x[4], y[4], a[4];
            load_piece<XT, VEC>(xr, c, span, xw);
            load_piece<XT, VEC>(yr, c, span, yw);
            trim_piece<XT, VEC>(c, span, xw);
            trim_piece<XT, VEC>(c, span, yw);
            unpack<XT>(xw, x);
            unpack<XT>(yw, y);
            grad_scale<VEC>(p, y, c, span, a);
            sum_grad(x, a, squares, dot);
        }
        const float2 s = reduce_row<true, false>(squares.x + squares.y, dot.x + dot.y, blockDim.x >> 5, scratch[turn]);
        const float inv = inverse_rms(s.x, p.per_col, p.eps);
        const float mean_au = s.y * p.per_col * inv;
        const bool begin = row == blockIdx.x;
        uint8_t* out = row_of<XT>(p.dx, row, p.dims, p.flat) - shift;
#pragma unroll 1
        for (uint32_t c = first; in_row<VEC>(c, span); c += stride) {
            uint32_t xw[W], yw[W], w[W];
            float2 x[4], y[4], a[4], add[4], acc[4];
            load_piece<XT, VEC>(xr, c, span, xw);
            load_piece<XT, VEC>(yr, c, span, yw);
            if constexpr (DSUM) {
                load_piece<XT, VEC>(sr, c, span, w);
                unpack<XT>(w, add);
            }
            unpack<XT>(xw, x);
            unpack<XT>(yw, y);
            grad_scale<VEC>(p, y, c, span, a);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] = both(0.0f);
            if (mine && !begin) {
                uint32_t t[8];
                load_floats<VEC>(mine, c, span, t);
                unpack<ROW_F32>(t, acc);
            }
            grad_piece<DSUM>(x, y, a, add, inv, mean_au, acc);
            if (mine) store_sums<VEC>(mine, c, span, acc);
            pack<XT>(a, w);
            store_piece<XT, VEC>(out, c, span, w);
        }
    }
}
// out[c] = sum over blocks: 32 interleaved shares, each in block order, then share by share: a fixed order.
__device__ __forceinline__ void column_sums(const float* partial, float* out, uint32_t blocks, uint32_t cols) {
    __shared__ float part[32][33];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, share = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (uint32_t b = share; b < blocks; b += 32) s += partial[uint64_t(b) * cols + c];
    }
    part[share][lane] = s;
    __syncthreads();
    if (share == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 32; ++i) s += part[i][lane];
        out[c] = s;
    }
}

// ------------------------------------------------------------------------------------------ columns, transposed
// One step per column of x, result transposed. First the columns' maxima (as bit patterns, whose order is the values'; a NaN's
// is above infinity's, so it stays), then the codes through a tile in shared memory, then the steps in place of the maxima.
// x is read twice; the second pass walks the rows from the end, so that it begins with what the first left in L2. In both a
// warp reads 256 consecutive columns of a row; slot e * 32 + lane stands for the column of that lane's element e. Phased rows: every
// eighth row has the same phase, so a warp takes rows that are a multiple of eight apart, and of its 256 columns it can be sure of
// 248 whatever its phase.
template <int VEC>
__device__ __forceinline__ uint32_t slot_column(uint32_t slot) {
    const uint32_t e = slot >> 5, lane = slot & 31;
    return VEC == 1 ? e * 32 + lane : lane * 8 + e;
}
template <int VEC>
constexpr uint32_t kTransCols = VEC == kPhased ? 248 : 256;   // columns of a tile
// Offset of a lane's element e from the tile's first column (negative below it) in rows of this phase.
template <int VEC>
__device__ __forceinline__ int element_column(int e, uint32_t phase) { return int(lane_column<VEC>(e)) - int(phase); }
template <int VEC>
__device__ __forceinline__ uint32_t element_slot(int e, uint32_t phase) {
    const uint32_t lane = threadIdx.x & 31;
    if constexpr (VEC != kPhased) return e * 32 + lane;
    return ((uint32_t(e) - phase) & 7) * 32 + lane - (uint32_t(e) < phase);
}
template <int XT>
__device__ __forceinline__ const uint8_t* trans_row(const QuantTransParams& p, uint32_t row) {
    return static_cast<const uint8_t*>(p.x.ptr) + uint64_t(row) * p.x_ld * RowElem<XT>::kBytes;
}
template <int XT, int VEC>
__global__ void __launch_bounds__(256) column_max_kernel(const __grid_constant__ QuantTransParams p) {
    constexpr int W = 2 * RowElem<XT>::kBytes;
    constexpr uint32_t kCols = kTransCols<VEC>;
    __shared__ float part[8][257];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, c0 = blockIdx.x * kCols;
    const uint32_t rows_per = ((p.rows + gridDim.y - 1) / gridDim.y + 7) & ~7u, r0 = min(p.rows, blockIdx.y * rows_per), r1 = min(p.rows, r0 + rows_per);
    float2 top[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) top[k] = both(0.0f);
    const RowSpan<VEC> span(trans_row<XT>(p, r0 + warp), RowElem<XT>::kBytes, p.cols);
    const uint32_t shift = span.phase * RowElem<XT>::kBytes;
    const bool there = in_row<VEC>(c0, span);
#pragma unroll 1
    for (uint32_t r = r0 + warp; r < r1; r += 32) {
        uint32_t x[4][W];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (there && r + 8 * j < r1) load_piece<XT, VEC>(trans_row<XT>(p, r + 8 * j) - shift, c0, span, x[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (there && r + 8 * j < r1) {
                float2 v[4];
                unpack<XT>(x[j], v);
#pragma unroll
                for (int k = 0; k < 4; ++k) top[k] = make_float2(max_nan(top[k].x, fabsf(v[k].x)), max_nan(top[k].y, fabsf(v[k].y)));
            }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (VEC != kPhased || element_column<VEC>(e, span.phase) >= 0) part[warp][element_slot<VEC>(e, span.phase)] = (e & 1) ? top[e >> 1].y : top[e >> 1].x;
    __syncthreads();
    const uint32_t column = slot_column<VEC>(threadIdx.x), mine = c0 + column;
    if (column >= kCols || mine >= p.cols) return;
    float t = part[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 8; ++i) t = max_nan(t, part[i][threadIdx.x]);
    atomicMax(reinterpret_cast<uint32_t*>(p.scale) + mine, __float_as_uint(t) & 0x7FFFFFFFu);
}
// Both passes together: 8192 x 8192 bf16 64 us, where reading x twice and writing once is 51 us: the first pass covers the whole
// matrix, so the second reads most of it from HBM again; 4096 x 4096 fp32 30 us; 8191 x 8193 bf16 112 us (the ends of the result's
// rows are written byte by byte; in a pass of their own that was 121 us).
// Tiles of 128 rows x 256 columns (248 phased): a warp takes four rows at a time, a lane eight of their columns, whose codes make one
// word per column. The tile's columns leave as aligned 16-byte words (byte by byte at their ends). Four blocks per SM hide one's
// loads behind another's stores: 8192 x 8192 bf16 64 us, with three and rows read a step ahead 68 us.
constexpr uint32_t kTransRows = 128;
template <int XT, int VEC, bool I8, bool GIVEN>
__global__ void __launch_bounds__(256, XT == ROW_BF16 ? 4 : 3) quant_trans_kernel(const __grid_constant__ QuantTransParams p) {
    constexpr int W = 2 * RowElem<XT>::kBytes;
    constexpr uint32_t kPitch = 33;               // words: 128 rows and one word that keeps the banks apart
    __shared__ uint32_t tile[256 * kPitch + 4];   // by slot: neighbouring lanes, neighbouring banks
    __shared__ CodeStep steps[256];               // by slot
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, c0 = blockIdx.x * kTransCols<VEC>, r0 = (gridDim.y - 1 - blockIdx.y) * kTransRows;
    {
        const uint32_t c = c0 + slot_column<VEC>(threadIdx.x);
        float s = 1.0f;
        if (c < p.cols) s = GIVEN ? p.given[uint64_t(c) * p.given_stride] : __fdiv_rn(p.scale[c], p.top);
        steps[threadIdx.x] = make_code_step(s);
    }
    // a step is 32 rows, four of them a warp's: neighbours, or (phased) eight apart
    constexpr uint32_t kApart = VEC == kPhased ? 8 : 1;
    const uint32_t first = VEC == kPhased ? warp : warp * 4;
    const RowSpan<VEC> span(trans_row<XT>(p, p.row0 + r0 + first), RowElem<XT>::kBytes, p.cols);
    const uint32_t shift = span.phase * RowElem<XT>::kBytes;
    __syncthreads();
    CodeStep mine[8];   // of this lane's columns
    bool all_fast = !GIVEN;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        mine[e] = VEC != kPhased || element_column<VEC>(e, span.phase) >= 0 ? steps[element_slot<VEC>(e, span.phase)] : CodeStep{1.0f, -1.0f};
        all_fast = all_fast && fast_step(mine[e], I8 || p.fp8_direct);
    }
#pragma unroll 1
    for (uint32_t g = 0; g < kTransRows / 32; ++g) {
        const uint32_t r = r0 + g * 32 + first;
        uint32_t x[4][W];
        float2 v[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (in_row<VEC>(c0, span) && r + j * kApart < p.rows) load_piece<XT, VEC>(trans_row<XT>(p, p.row0 + r + j * kApart) - shift, c0, span, x[j]);
            else {
#pragma unroll
                for (int k = 0; k < W; ++k) x[j][k] = 0;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack<XT>(x[j], v[j]);
        const auto put = [&](int e, uint32_t word) {
            if (VEC != kPhased || element_column<VEC>(e, span.phase) >= 0) tile[element_slot<VEC>(e, span.phase) * kPitch + g * 8 + warp] = word;
        };
        const auto codes = [&](auto fast) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                put(2 * k, make_codes<I8, decltype(fast)::value>(make_float2(v[0][k].x, v[1][k].x), make_float2(v[2][k].x, v[3][k].x), mine[2 * k], p.hw));
                put(2 * k + 1, make_codes<I8, decltype(fast)::value>(make_float2(v[0][k].y, v[1][k].y), make_float2(v[2][k].y, v[3][k].y), mine[2 * k + 1], p.hw));
            }
        };
        if (all_fast) codes(std::true_type());
        else codes(std::false_type());
    }
    __syncthreads();
    if constexpr (VEC == kPhased) {
        // word w of a step holds rows w, w + 8, w + 16, w + 24: put the bytes in the rows' order
        for (uint32_t i = threadIdx.x; i < 256 * (kTransRows / 32); i += 256) {
            uint32_t* w = tile + (i & 255) * kPitch + (i >> 8) * 8;
            uint32_t o[8];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t a = w[4 * half], b = w[4 * half + 1], c = w[4 * half + 2], d = w[4 * half + 3];
                const uint32_t ab = __byte_perm(a, b, 0x5140), cd = __byte_perm(c, d, 0x5140), ab2 = __byte_perm(a, b, 0x7362), cd2 = __byte_perm(c, d, 0x7362);
                o[half] = __byte_perm(ab, cd, 0x5410); o[2 + half] = __byte_perm(ab, cd, 0x7632);
                o[4 + half] = __byte_perm(ab2, cd2, 0x5410); o[6 + half] = __byte_perm(ab2, cd2, 0x7632);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = o[k];
        }
        __syncthreads();
    }
    const uint32_t rows = min(kTransRows, p.rows - r0), cols = min(kTransCols<VEC>, p.cols - c0);
    // nine 16-byte words cover a column's 128 bytes at any alignment, eight where they are aligned; neighbouring lanes take
    // neighbouring slots, whose words lie in different banks
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.out) + p.row0 + r0) | p.out_ld) % 16 == 0;
    const uint32_t words = aligned ? 8 : 9;
    for (uint32_t i = threadIdx.x; i < 256 * words; i += 256) {
        const uint32_t slot = aligned ? i / 8 : i / 9, k = i - slot * words, col = slot_column<VEC>(slot);
        if (col >= cols) continue;
        if (aligned && 16 * k + 16 <= rows) {
            const uint32_t* w = tile + slot * kPitch + 4 * k;
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + uint64_t(c0 + col) * p.out_ld + p.row0 + r0 + 16 * k) = make_uint4(w[0], w[1], w[2], w[3]);
            continue;
        }
        uint8_t* a = static_cast<uint8_t*>(p.out) + uint64_t(c0 + col) * p.out_ld + p.row0 + r0;
        const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(a)) & 15u;
        const int begin = int(16 * k) - int(off);   // first row of the word
        if (begin >= int(rows)) continue;
        const uint32_t* column = tile + slot * kPitch;
        if (begin >= 0 && begin + 16 <= int(rows)) {
            const uint32_t w0 = uint32_t(begin) >> 2, sh = (uint32_t(begin) & 3u) * 8;
            uint32_t w[5], o[4];
#pragma unroll
            for (int j = 0; j < 5; ++j) w[j] = column[w0 + j];   // the fifth word (the padding, at the end) counts only when sh != 0
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __funnelshift_r(w[j], w[j + 1], sh);
            *reinterpret_cast<uint4*>(a + begin) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
            for (int r = max(begin, 0); r < min(begin + 16, int(rows)); ++r) a[r] = uint8_t(column[r >> 2] >> (8 * (r & 3)));
        }
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
