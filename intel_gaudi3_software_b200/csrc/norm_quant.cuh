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
// A lane works on pieces of eight consecutive elements, a warp on a run of consecutive pieces. Where every row of every tensor
// starts on a multiple of eight elements (SHIFT = false) a piece is one or two 16-byte accesses. Rows of any other length,
// pitch or start (SHIFT = true) are read as the aligned 16-byte words that contain the piece and shifted into place in
// registers, and written as aligned words put together from the lane's piece and its left neighbour's: odd rows move as many
// bytes per instruction as even ones do. How far a row is off is the same for all its pieces, so the shifts are branches that
// a whole warp takes. Reads stay inside the tensor (first byte to last), writes inside the row; the ends of a warp's run go
// element by element.
template <int TYPE>
struct RowElem;
template <> struct RowElem<ROW_BF16> { static constexpr int kBytes = 2; };
template <> struct RowElem<ROW_F32> { static constexpr int kBytes = 4; };
template <> struct RowElem<ROW_I8> { static constexpr int kBytes = 1; };   // codes of either kind

// out[i] = the four bytes from byte `off` + 4 i of `in`. off < 4 * (N - W) is the same in all lanes.
template <int N, int W>
__device__ __forceinline__ void shift_words(const uint32_t (&in)[N], uint32_t off, uint32_t (&out)[W]) {
    const uint32_t bits = (off & 3) * 8;
#pragma unroll
    for (int q = 0; q < N - W; ++q)
        if ((off >> 2) == uint32_t(q)) {
#pragma unroll
            for (int i = 0; i < W; ++i) out[i] = __funnelshift_r(in[q + i], in[q + i + 1], bits);
        }
}

__device__ __forceinline__ int piece_size(uint32_t c, uint32_t cols) { return c >= cols ? 0 : int(min(8u, cols - c)); }

// A row that is read: `raw` pieces are loaded first, all of them in flight, and turned into packed elements when needed.
template <int TYPE, bool SHIFT>
struct RowIn {
    static constexpr int kBytes = RowElem<TYPE>::kBytes, kWords = 2 * kBytes, kRaw = kWords + (SHIFT ? 4 : 0);
    struct Raw { uint32_t w[kRaw]; };
    const uint8_t* row;      // SHIFT: rounded down to 16 bytes
    const uint8_t* lo;       // SHIFT: the tensor's bytes, [lo, hi)
    const uint8_t* hi;
    uint32_t off;
    __device__ __forceinline__ RowIn(const RowTensor& t, uint64_t at) {
        lo = static_cast<const uint8_t*>(t.ptr);
        row = lo + at * kBytes;
        if constexpr (SHIFT) {
            hi = lo + t.bytes;
            off = uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u;
            row -= off;
        }
    }
    __device__ __forceinline__ void load(Raw& r, uint32_t c) const {
        const uint8_t* a = row + uint64_t(c) * kBytes;
        if (!SHIFT || (a >= lo && a + 4 * kRaw <= hi)) {
#pragma unroll
            for (int i = 0; i < kRaw / 4; ++i) {
                const uint4 q = reinterpret_cast<const uint4*>(a)[i];
                r.w[4 * i] = q.x; r.w[4 * i + 1] = q.y; r.w[4 * i + 2] = q.z; r.w[4 * i + 3] = q.w;
            }
        } else {   // the tensor's first and last pieces
            load_guarded(r, a);
        }
    }
    __device__ __forceinline__ void words(const Raw& r, uint32_t (&w)[kWords]) const {
        if constexpr (SHIFT) shift_words(r.w, off, w);
        else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = r.w[i];
        }
    }

private:
    __device__ __noinline__ void load_guarded(Raw& r, const uint8_t* a) const {
#pragma unroll 1
        for (int i = 0; i < kRaw; ++i) {
            uint32_t v = 0;
#pragma unroll 1
            for (int k = 0; k < 4; k += kBytes) {   // elements, which do not straddle the tensor's ends
                const uint8_t* e = a + 4 * i + k;
                if (e >= lo && e + kBytes <= hi) v |= (kBytes == 2 ? uint32_t(*reinterpret_cast<const uint16_t*>(e)) : *reinterpret_cast<const uint32_t*>(e)) << (8 * k);
            }
            r.w[i] = v;
        }
    }
};
template <bool SHIFT>
struct RowIn<ROW_NONE, SHIFT> {
    struct Raw {};
    __device__ __forceinline__ RowIn(const RowTensor&, uint64_t) {}
    __device__ __forceinline__ void load(Raw&, uint32_t) const {}
};
// The eight elements of a piece are worked on as four pairs: sm_100a adds and multiplies two floats per instruction, and the
// row kernels are as near the issue rate as they are to HBM's.
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

// Elements [from, to) of a packed piece, one by one. Out of line: only the ends of a warp's run come here, and inlined at every
// store the code would not stay in the instruction cache.
static __device__ __noinline__ void put_elements_16(uint16_t* a, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, int from, int to) {
    const uint32_t w[4] = {w0, w1, w2, w3};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e >= from && e < to) a[e] = uint16_t(w[e >> 1] >> (16 * (e & 1)));
}
static __device__ __noinline__ void put_elements_8(uint8_t* a, uint32_t w0, uint32_t w1, int from, int to) {
    const uint32_t w[2] = {w0, w1};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e >= from && e < to) a[e] = uint8_t(w[e >> 2] >> (8 * (e & 3)));
}
static __device__ __noinline__ void put_elements_32(uint32_t* a, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, int from, int to) {
    const uint32_t w[4] = {w0, w1, w2, w3};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e >= from && e < to) a[e] = w[e];
}
template <int TYPE, int W>
__device__ __forceinline__ void put_elements(uint8_t* a, const uint32_t (&v)[W], int from, int to) {
    if constexpr (W == 2) put_elements_8(a, v[0], v[1], from, to);
    else if constexpr (W == 4) put_elements_16(reinterpret_cast<uint16_t*>(a), v[0], v[1], v[2], v[3], from, to);
    else {
        put_elements_32(reinterpret_cast<uint32_t*>(a), v[0], v[1], v[2], v[3], from, to);
        put_elements_32(reinterpret_cast<uint32_t*>(a) + 4, v[4], v[5], v[6], v[7], from - 4, to - 4);
    }
}

// A row that is written. A warp writes its run step by step (32 pieces each), in order, all lanes together (SHIFT).
// `start`: its first step; `last`: no step follows whose first piece is full.
template <int TYPE, bool SHIFT>
struct RowOut {
    static constexpr int kBytes = RowElem<TYPE>::kBytes, kWords = 2 * kBytes;
    static constexpr uint32_t kUnit = kWords == 2 ? 8 : 16;   // bytes of an aligned store
    static constexpr int kTail = kUnit / 4;
    uint8_t* row;
    uint32_t off;
    uint32_t carry[SHIFT ? kTail : 1];   // the end of this lane's piece before
    __device__ __forceinline__ RowOut(const RowTensor& t, uint64_t at) {
        row = static_cast<uint8_t*>(t.ptr) + at * kBytes;
        if constexpr (SHIFT) {
            off = uint32_t(reinterpret_cast<uintptr_t>(row)) & (kUnit - 1);
#pragma unroll
            for (int i = 0; i < kTail; ++i) carry[i] = 0;
        }
    }
    __device__ __forceinline__ static void put(uint8_t* a, const uint32_t (&v)[kWords]) {
        if constexpr (kWords == 2) *reinterpret_cast<uint2*>(a) = make_uint2(v[0], v[1]);
        else {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(a)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
    }
    // n: elements of this lane's piece that exist; whole: the warp's 32 pieces are full
    __device__ __forceinline__ void store(uint32_t c, int n, const uint32_t (&v)[kWords], bool whole, bool start, bool last) {
        uint8_t* a = row + uint64_t(c) * kBytes;
        if constexpr (!SHIFT) {
            if (n) put(a, v);
        } else if (off == 0) {
            if (n == 8) put(a, v);
            else put_elements<TYPE>(a, v, 0, n);
        } else {
            const uint32_t lane = threadIdx.x & 31;
            uint32_t both[kTail + kWords], out[kWords];
#pragma unroll
            for (int i = 0; i < kTail; ++i) {
                // lane L takes lane L - 1's end, lane 0 what lane 31 had before
                const uint32_t mine = v[kWords - kTail + i], give = lane == 31 ? carry[i] : mine;
                both[i] = __shfl_sync(0xffffffffu, give, (lane + 31) & 31);
                carry[i] = mine;
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) both[kTail + i] = v[i];
            shift_words(both, kUnit - off, out);
            const bool head = start && lane == 0;   // nobody gave it the bytes before its piece
            if (n == 8 && !head) put(a - off, out);
            if (start || last || !whole) {
                // by elements: a head, and a piece that is not full; the last `off` bytes of a full piece without a successor,
                // and those of a left neighbour of a piece that is not full
                const int left = int(off) / kBytes;
                const bool next_full = __shfl_down_sync(0xffffffffu, n, 1) == 8 && lane != 31;
                const bool tail_mine = !(next_full || (lane == 31 && !last));
                int from = 8, to = n;
                if (head || n < 8) from = 0;
                else if (tail_mine) from = 8 - left;
                if (n == 8 && !tail_mine && from == 0) to = 8 - left;
                if (from < to) put_elements<TYPE>(a, v, from, to);
            }
        }
    }
};

// gamma is read by every row and sits in the caches; its type is a runtime value. SHIFT = false: it starts on 16 bytes.
template <bool SHIFT>
__device__ __forceinline__ void load_gamma(float2 (&g)[4], const void* base, int type, bool whole, uint32_t at, int n) {
    if (!SHIFT || (whole && n == 8)) {
        if (type == ROW_BF16) {
            const uint4 q = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
            unpack<ROW_BF16>(w, g);
        } else {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
            const float4 a = __ldg(q), b = __ldg(q + 1);
            g[0] = make_float2(a.x, a.y); g[1] = make_float2(a.z, a.w);
            g[2] = make_float2(b.x, b.y); g[3] = make_float2(b.z, b.w);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float t = 1.0f;
            if (e < n) t = type == ROW_BF16 ? __uint_as_float(uint32_t(static_cast<const uint16_t*>(base)[at + e]) << 16) : static_cast<const float*>(base)[at + e];
            if (e & 1) g[e >> 1].y = t;
            else g[e >> 1].x = t;
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float2 v) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(v.y), "f"(v.x));
    return w;
}
// Eight floats, packed as the type keeps them.
template <int TYPE, int W>
__device__ __forceinline__ void pack(const float2 (&f)[4], uint32_t (&w)[W]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == ROW_F32) { w[2 * i] = __float_as_uint(f[i].x); w[2 * i + 1] = __float_as_uint(f[i].y); }
        else w[i] = pack_bf16(f[i]);
    }
}

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

// ------------------------------------------------------------------------------------------ 8-bit codes
// How values become codes: `step`, and its reciprocal where that decides them. recip = 0: no codes (a step that is zero,
// negative or no finite number), NaN: the reciprocal is no normal number, every code is divided for.
struct CodeStep {
    float step, recip;
};
__device__ __forceinline__ CodeStep make_code_step(float step) {
    CodeStep s;
    s.step = step;
    if (!(step > 0.0f && step < __uint_as_float(0x7F800000u))) s.recip = 0.0f;
    else s.recip = (step >= 0x1p-126f && step <= 0x1p126f) ? __frcp_rn(step) : __uint_as_float(0x7FC00000u);
    return s;
}
constexpr float kRoundMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to the nearest whole number, ties to even

__device__ __forceinline__ uint32_t pack_low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
// Four codes by the definition: the correctly rounded quotient, then the code. Out of line: few values come here.
template <bool I8>
static __device__ __noinline__ uint32_t codes_by_division(float v0, float v1, float v2, float v3, float step, const Fp8HwCast& hw) {
    float t[4] = {__fdiv_rn(v0, step), __fdiv_rn(v1, step), __fdiv_rn(v2, step), __fdiv_rn(v3, step)};
    if constexpr (I8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fminf(fmaxf(t[e], -127.0f), 127.0f) + kRoundMagic;
        return pack_low_bytes(t[0], t[1], t[2], t[3]);
    } else {
        return f32x4_to_fp8_hw(t, hw);
    }
}
// The four codes of v / step, packed. v * recip is within 2^-23 of the quotient, relatively, and the 32-bit quotient within
// 2^-24 of the exact one, so
//   int8: for |quotient| <= 127 the product is off by at most 2^-15.4; unless it lies closer than 2^-15 to the middle between two
//         whole numbers it rounds as the quotient does (one multiplication and three additions per element);
//   fp8:  where product * (1 - 2^-22) and product * (1 + 2^-22) have the same code, it is the quotient's (the cast is monotone).
// The few quads with an element that fails its test are divided. GIVEN: the step is the caller's, quotients may be anything.
template <bool I8, bool GIVEN>
__device__ __forceinline__ uint32_t make_codes(float2 v0, float2 v1, const CodeStep& s, const Fp8HwCast& hw) {
    if (s.recip == 0.0f) return 0u;
    float2 x[2] = {v0, v1};
    uint32_t w;
    bool sure;
    if constexpr (I8) {
        float2 m[2];
        float worst = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (GIVEN) {   // a NaN has no code (rows with one have no step of their own)
                x[i].x = x[i].x == x[i].x ? x[i].x : 0.0f;
                x[i].y = x[i].y == x[i].y ? x[i].y : 0.0f;
            }
            float2 t = __fmul2_rn(x[i], both(s.recip));
            if constexpr (GIVEN) {
                t.x = fminf(fmaxf(t.x, -127.0f), 127.0f);
                t.y = fminf(fmaxf(t.y, -127.0f), 127.0f);
            }
            m[i] = __fadd2_rn(t, both(kRoundMagic));
            const float2 back = __fadd2_rn(m[i], both(-kRoundMagic)), off = __ffma2_rn(back, both(-1.0f), t);
            worst = fmaxf(worst, fmaxf(fabsf(off.x), fabsf(off.y)));
        }
        sure = worst <= 0.5f - 0x1p-15f && s.recip == s.recip;
        w = pack_low_bytes(m[0].x, m[0].y, m[1].x, m[1].y);
    } else {
        float lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 t = __fmul2_rn(x[i], both(s.recip)), l = __fmul2_rn(t, both(1.0f - 0x1p-22f)), h = __fmul2_rn(t, both(1.0f + 0x1p-22f));
            lo[2 * i] = l.x; lo[2 * i + 1] = l.y;
            hi[2 * i] = h.x; hi[2 * i + 1] = h.y;
        }
        w = f32x4_to_fp8_hw(lo, hw);
        sure = w == f32x4_to_fp8_hw(hi, hw) && s.recip == s.recip;
    }
    if (!sure) w = codes_by_division<I8>(x[0].x, x[0].y, x[1].x, x[1].y, s.step, hw);
    return w;
}

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
// x + residual, rounded to the stream's type, which is what the norm sees.
template <int XT, int RT, bool SHIFT>
__device__ __forceinline__ void stream_piece(const RowIn<XT, SHIFT>& xin, const typename RowIn<XT, SHIFT>::Raw& x, const RowIn<RT, SHIFT>& rin,
                                             const typename RowIn<RT, SHIFT>::Raw& r, RowKept<XT, RT>& h) {
    uint32_t xw[RowIn<XT, SHIFT>::kWords];
    xin.words(x, xw);
    if constexpr (RT == ROW_NONE) {
#pragma unroll
        for (int i = 0; i < RowIn<XT, SHIFT>::kWords; ++i) h.w[i] = xw[i];
    } else {
        uint32_t rw[RowIn<RT, SHIFT>::kWords];
        rin.words(r, rw);
        float2 f[4], g[4];
        unpack<XT>(xw, f);
        unpack<RT>(rw, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __fadd2_rn(f[i], g[i]);
        pack<RT>(f, h.w);
    }
}
// A row's last piece may be partial: its missing elements count as zeros.
template <int XT, int RT>
__device__ __forceinline__ void clear_missing(RowKept<XT, RT>& h, int n) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e >= n) {
            if constexpr (RowKept<XT, RT>::kType == ROW_F32) h.w[e] = 0;
            else h.w[e >> 1] &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
        }
}
// Adds a piece to its row's sums.
template <bool TOPS, bool SHIFT, int XT, int RT>
__device__ __forceinline__ void sum_piece(const NormParams& p, const RowKept<XT, RT>& kept, uint32_t c, int n, float2& sum, float& top) {
    float2 h[4];
    kept.values(h);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = __ffma2_rn(h[i], h[i], sum);
    if constexpr (TOPS) {
        if (p.gamma_type != ROW_NONE) {
            float2 g[4];
            load_gamma<SHIFT>(g, p.gamma, p.gamma_type, p.gamma_whole, c, n);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __fmul2_rn(h[i], g[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max_nan(top, fabsf(h[i].x), fabsf(h[i].y));
    }
}
// v = h * gamma of a piece.
template <bool SHIFT, int XT, int RT>
__device__ __forceinline__ void scaled_piece(const NormParams& p, const RowKept<XT, RT>& kept, uint32_t c, int n, float2 (&v)[4]) {
    kept.values(v);
    if (p.gamma_type != ROW_NONE && n) {
        float2 g[4];
        load_gamma<SHIFT>(g, p.gamma, p.gamma_type, p.gamma_whole, c, n);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fmul2_rn(v[i], g[i]);
    }
}

// The warp's run of pieces: piece i of a lane starts at column c0 + 256 i.
template <bool SHIFT>
struct WarpRun {
    uint32_t c0, cols;
    __device__ __forceinline__ uint32_t col(uint32_t i) const { return c0 + 256 * i + (threadIdx.x & 31) * 8; }
    __device__ __forceinline__ bool any(uint32_t i) const { return c0 + 256 * i < cols; }
    __device__ __forceinline__ bool whole(uint32_t i) const { return c0 + 256 * i + 256 <= cols; }
    __device__ __forceinline__ int size(uint32_t i) const { return SHIFT ? piece_size(col(i), cols) : col(i) < cols ? 8 : 0; }
    // step i is the last of `steps` that hands nothing on to a full piece
    __device__ __forceinline__ bool last(uint32_t i, uint32_t steps) const { return i + 1 == steps || c0 + 256 * (i + 1) + 8 > cols; }
};

// The second pass over a row: `piece(i, n, v)` gives the values h * gamma of piece i.
template <int MODE, bool SHIFT, int UNROLL, typename F>
__device__ __forceinline__ void write_row(const NormParams& p, uint64_t at, const WarpRun<SHIFT>& run, uint32_t pieces, const RowFactors& f, F&& piece) {
    constexpr int kType = MODE == NORM_BF16 ? ROW_BF16 : MODE == NORM_F32 ? ROW_F32 : ROW_I8;
    RowOut<kType, SHIFT> out(p.out, at);
#pragma unroll UNROLL
    for (uint32_t i = 0; i < pieces; ++i) {
        const int n = run.size(i);
        if (SHIFT ? run.any(i) : n != 0) {
            float2 v[4];
            uint32_t w[RowOut<kType, SHIFT>::kWords];
            piece(i, n, v);
            if constexpr (MODE == NORM_I8 || MODE == NORM_F8) {
#pragma unroll
                for (int q = 0; q < 2; ++q) w[q] = make_codes<MODE == NORM_I8, false>(v[2 * q], v[2 * q + 1], f.step, p.hw);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = __fmul2_rn(v[k], both(f.inv));
                if constexpr (MODE == NORM_BF16 || MODE == NORM_F32) pack<kType>(v, w);
                else {
#pragma unroll
                    for (int q = 0; q < 2; ++q) w[q] = make_codes<MODE == NORM_I8_GIVEN, true>(v[2 * q], v[2 * q + 1], f.step, p.hw);
                }
            }
            out.store(run.col(i), n, w, run.whole(i), i == 0, run.last(i, pieces));
        }
    }
}
// What differs between the kinds of output is decided once per row, not once per piece.
template <bool SHIFT, int UNROLL, typename F>
__device__ __forceinline__ void write_row_any(const NormParams& p, uint64_t at, const WarpRun<SHIFT>& run, uint32_t pieces, const RowFactors& f, F&& piece) {
    switch (p.mode) {
        case NORM_BF16: write_row<NORM_BF16, SHIFT, UNROLL>(p, at, run, pieces, f, piece); break;
        case NORM_F32: write_row<NORM_F32, SHIFT, UNROLL>(p, at, run, pieces, f, piece); break;
        case NORM_I8: write_row<NORM_I8, SHIFT, UNROLL>(p, at, run, pieces, f, piece); break;
        case NORM_F8: write_row<NORM_F8, SHIFT, UNROLL>(p, at, run, pieces, f, piece); break;
        case NORM_I8_GIVEN: write_row<NORM_I8_GIVEN, SHIFT, UNROLL>(p, at, run, pieces, f, piece); break;
        default: write_row<NORM_F8_GIVEN, SHIFT, UNROLL>(p, at, run, pieces, f, piece); break;
    }
}

// The first pass: reads x and the residual, writes the stream, takes the sums. NV pieces per lane, loads G pieces at a time.
template <bool TOPS, int XT, int RT, bool SHIFT, int NV>
__device__ __forceinline__ float2 read_row(const NormParams& p, uint32_t row, const WarpRun<SHIFT>& run, RowKept<XT, RT> (&kept)[NV]) {
    constexpr int G = NV < 2 ? 1 : (!SHIFT && XT != ROW_F32 && RT != ROW_F32) ? 4 : 2, KT = RowKept<XT, RT>::kType;
    const RowIn<XT, SHIFT> xin(p.x, row_offset(p.x, row, p.dims, p.flat));
    const RowIn<RT, SHIFT> rin(p.residual, RT != ROW_NONE ? row_offset(p.residual, row, p.dims, p.flat) : 0);
    RowOut<KT, SHIFT> sout(p.sum, RT != ROW_NONE ? row_offset(p.sum, row, p.dims, p.flat) : 0);
    float2 sum = both(0.0f);
    float top = 0.0f;
#pragma unroll
    for (int i0 = 0; i0 < NV; i0 += G) {
        typename RowIn<XT, SHIFT>::Raw x[G];
        typename RowIn<RT, SHIFT>::Raw r[G];
#pragma unroll
        for (int j = 0; j < G; ++j)
            if (run.size(i0 + j)) {
                xin.load(x[j], run.col(i0 + j));
                rin.load(r[j], run.col(i0 + j));
            }
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int i = i0 + j;
            const int n = run.size(i);
            if (n) {
                stream_piece<XT, RT, SHIFT>(xin, x[j], rin, r[j], kept[i]);
                if (SHIFT && n < 8) clear_missing(kept[i], n);
                sum_piece<TOPS, SHIFT>(p, kept[i], run.col(i), n, sum, top);
            }
            if constexpr (RT != ROW_NONE) {
                if (p.sum.ptr && (SHIFT ? run.any(i) : n != 0)) sout.store(run.col(i), n, kept[i].w, run.whole(i), i == 0, run.last(i, NV));
            }
        }
    }
    return make_float2(sum.x + sum.y, top);
}

// A row per warp (BLOCK = false: four rows per block) or per block, NV pieces per lane, kept in registers between the row's
// one read and its one write.
template <int XT, int RT, bool SHIFT, int NV, bool BLOCK, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 && RowKept<XT, RT>::kType == ROW_BF16 && !(SHIFT && NV == 8) ? 2 : 1) norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 scratch[32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = BLOCK ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= p.rows) return;   // whole warps, never part of a block that synchronises
    const WarpRun<SHIFT> run{BLOCK ? (threadIdx.x >> 5) * 256 * NV : 0u, p.cols};
    RowKept<XT, RT> kept[NV];
    float2 s = (p.mode == NORM_I8 || p.mode == NORM_F8) ? read_row<true, XT, RT, SHIFT, NV>(p, row, run, kept) : read_row<false, XT, RT, SHIFT, NV>(p, row, run, kept);
    s = reduce_row<BLOCK, true>(s.x, s.y, blockDim.x >> 5, scratch);
    const RowFactors f = row_factors(p, s.x, s.y, row);
    if (p.scale && (BLOCK ? threadIdx.x : threadIdx.x & 31) == 0) p.scale[row] = f.scale;
    write_row_any<SHIFT, NV>(p, row_offset(p.out, row, p.dims, p.flat), run, NV, f,
                         [&](uint32_t i, int n, float2 (&v)[4]) { scaled_piece<SHIFT>(p, kept[i], run.col(i), n, v); });
}

// The same with the row kept in shared memory (every lane its own pieces) and the pieces walked by a loop: the form for rows at
// any alignment, whose shifts and ends would not fit the instruction cache unrolled, and for rows so long that registers
// would leave one block per SM.
template <int XT, int RT, bool SHIFT>
__global__ void __launch_bounds__(512, 2) norm_loop_kernel(const __grid_constant__ NormParams p) {
    constexpr int KT = RowKept<XT, RT>::kType, Q = RowKept<XT, RT>::kWords / 4;   // 16-byte words of a kept piece
    __shared__ float2 scratch[32];
    extern __shared__ uint4 keep[];   // [piece of a lane][16-byte word][thread]
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = blockIdx.x, threads = blockDim.x, pieces = (p.cols + threads * 8 - 1) / (threads * 8);   // per lane
    const WarpRun<SHIFT> run{(threadIdx.x >> 5) * 256 * pieces, p.cols};
    const bool tops = p.mode == NORM_I8 || p.mode == NORM_F8;
    float2 sum = both(0.0f);
    float top = 0.0f;
    {
        const RowIn<XT, SHIFT> xin(p.x, row_offset(p.x, row, p.dims, p.flat));
        const RowIn<RT, SHIFT> rin(p.residual, RT != ROW_NONE ? row_offset(p.residual, row, p.dims, p.flat) : 0);
        RowOut<KT, SHIFT> sout(p.sum, RT != ROW_NONE ? row_offset(p.sum, row, p.dims, p.flat) : 0);
        const bool has_sum = RT != ROW_NONE && p.sum.ptr != nullptr;
#pragma unroll 1
        for (uint32_t i0 = 0; i0 < pieces; i0 += 2) {
            typename RowIn<XT, SHIFT>::Raw x[2];
            typename RowIn<RT, SHIFT>::Raw r[2];
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j)
                if (i0 + j < pieces && run.size(i0 + j)) {
                    xin.load(x[j], run.col(i0 + j));
                    rin.load(r[j], run.col(i0 + j));
                }
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                const uint32_t i = i0 + j;
                if (i < pieces && run.any(i)) {
                    const int n = run.size(i);
                    RowKept<XT, RT> kept;
                    if (n) {
                        stream_piece<XT, RT, SHIFT>(xin, x[j], rin, r[j], kept);
                        if (SHIFT && n < 8) clear_missing(kept, n);
#pragma unroll
                        for (int k = 0; k < Q; ++k)
                            keep[(i * Q + k) * threads + threadIdx.x] = make_uint4(kept.w[4 * k], kept.w[4 * k + 1], kept.w[4 * k + 2], kept.w[4 * k + 3]);
                        if (tops) sum_piece<true, SHIFT>(p, kept, run.col(i), n, sum, top);
                        else sum_piece<false, SHIFT>(p, kept, run.col(i), n, sum, top);
                    }
                    if constexpr (RT != ROW_NONE) {
                        if (has_sum && (SHIFT || n)) sout.store(run.col(i), n, kept.w, run.whole(i), i == 0, run.last(i, pieces));
                    }
                }
            }
        }
    }
    const float2 s = reduce_row<true, true>(sum.x + sum.y, top, threads >> 5, scratch);
    const RowFactors f = row_factors(p, s.x, s.y, row);
    if (p.scale && threadIdx.x == 0) p.scale[row] = f.scale;
    write_row_any<SHIFT, 1>(p, row_offset(p.out, row, p.dims, p.flat), run, pieces, f, [&](uint32_t i, int n, float2 (&v)[4]) {
        RowKept<XT, RT> kept;
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const uint4 q = n ? keep[(i * Q + k) * threads + threadIdx.x] : make_uint4(0, 0, 0, 0);
            kept.w[4 * k] = q.x; kept.w[4 * k + 1] = q.y; kept.w[4 * k + 2] = q.z; kept.w[4 * k + 3] = q.w;
        }
        scaled_piece<SHIFT>(p, kept, run.col(i), n, v);
    });
}

// Rows too long for shared memory: the row is read a second time (from L2, mostly) once its sums are known. The second read
// takes the stream from `sum` where it was written (in place, x and the residual may be gone by then). A warp reads and
// writes the same elements in both passes.
template <int XT, int RT, bool SHIFT>
__global__ void __launch_bounds__(1024) norm_long_kernel(const __grid_constant__ NormParams p) {
    constexpr int KT = RowKept<XT, RT>::kType;
    __shared__ float2 scratch[32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = blockIdx.x, pieces = (p.cols + 32 * 256 - 1) / (32 * 256);   // per lane
    const WarpRun<SHIFT> run{(threadIdx.x >> 5) * 256 * pieces, p.cols};
    const RowIn<XT, SHIFT> xin(p.x, row_offset(p.x, row, p.dims, p.flat));
    const RowIn<RT, SHIFT> rin(p.residual, RT != ROW_NONE ? row_offset(p.residual, row, p.dims, p.flat) : 0);
    const uint64_t so = RT != ROW_NONE ? row_offset(p.sum, row, p.dims, p.flat) : 0;
    const bool tops = p.mode == NORM_I8 || p.mode == NORM_F8, has_sum = RT != ROW_NONE && p.sum.ptr != nullptr;
    float2 sum = both(0.0f);
    float top = 0.0f;
    {
        RowOut<KT, SHIFT> sout(p.sum, so);
#pragma unroll 1
        for (uint32_t i = 0; i < pieces && run.any(i); ++i) {
            const int n = run.size(i);
            RowKept<XT, RT> kept;
            if (n) {
                typename RowIn<XT, SHIFT>::Raw x;
                typename RowIn<RT, SHIFT>::Raw r;
                xin.load(x, run.col(i));
                rin.load(r, run.col(i));
                stream_piece<XT, RT, SHIFT>(xin, x, rin, r, kept);
                if (SHIFT && n < 8) clear_missing(kept, n);
                if (tops) sum_piece<true, SHIFT>(p, kept, run.col(i), n, sum, top);
                else sum_piece<false, SHIFT>(p, kept, run.col(i), n, sum, top);
            }
            if constexpr (RT != ROW_NONE) {
                if (has_sum && (SHIFT || n)) sout.store(run.col(i), n, kept.w, run.whole(i), i == 0, run.last(i, pieces));
            }
        }
    }
    const float2 s = reduce_row<true, true>(sum.x + sum.y, top, 32, scratch);   // its barrier also orders the stores of `sum` and the reads below
    const RowFactors f = row_factors(p, s.x, s.y, row);
    if (p.scale && threadIdx.x == 0) p.scale[row] = f.scale;
    const RowIn<KT, SHIFT> again(p.sum, so);
    const uint64_t oo = row_offset(p.out, row, p.dims, p.flat);
    write_row_any<SHIFT, 1>(p, oo, run, pieces, f, [&](uint32_t i, int n, float2 (&v)[4]) {
        RowKept<XT, RT> kept;
#pragma unroll
        for (int k = 0; k < RowKept<XT, RT>::kWords; ++k) kept.w[k] = 0;
        if (n) {
            if (has_sum) {
                typename RowIn<KT, SHIFT>::Raw h;
                again.load(h, run.col(i));
                again.words(h, kept.w);
            } else {
                typename RowIn<XT, SHIFT>::Raw x;
                typename RowIn<RT, SHIFT>::Raw r;
                xin.load(x, run.col(i));
                rin.load(r, run.col(i));
                stream_piece<XT, RT, SHIFT>(xin, x, rin, r, kept);
            }
        }
        scaled_piece<SHIFT>(p, kept, run.col(i), n, v);
    });
}

// ------------------------------------------------------------------------------------------ gradient
// With a = dy * gamma, u = x * inv:  dx = inv * (a - u * mean(a * u)) + dsum,  dgamma = sum over rows of dy * u.
// mean(a * u) = inv * mean(a * x), so both sums of a row (x^2 and a * x) are taken in one pass. A block walks rows b, b +
// blocks, ...; every thread keeps the sums of its own columns of dgamma, and the block's partial sums (one row of `partial`)
// are added in a fixed order by column_sums: results do not depend on timing.
__device__ __forceinline__ void clear_missing(float2 (&x)[4], float2 (&y)[4], int n) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (2 * k >= n) x[k].x = y[k].x = 0.0f;
        if (2 * k + 1 >= n) x[k].y = y[k].y = 0.0f;
    }
}
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
// XT: type of x, dy, dsum and dx; DSUM: whether there is a gradient of the sum. A row per warp or per block, as in norm_kernel.
template <int XT, bool DSUM, bool SHIFT, int NV, bool BLOCK, int THREADS>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) norm_grad_kernel(const __grid_constant__ NormGradParams p) {
    constexpr int kRowsPerBlock = BLOCK ? 1 : 4, ST = DSUM ? XT : ROW_NONE, W = 2 * RowElem<XT>::kBytes;
    __shared__ float2 scratch[2][32];
    extern __shared__ float block_sums[];   // a row per warp: [cols], the four warps' sums of dgamma
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t sub = BLOCK ? 0 : (threadIdx.x >> 5);
    const WarpRun<SHIFT> run{BLOCK ? (threadIdx.x >> 5) * 256 * NV : 0u, p.cols};
    float2 acc[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][k] = both(0.0f);
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x * kRowsPerBlock + sub; row < p.rows; row += gridDim.x * kRowsPerBlock, turn ^= 1) {
        const RowIn<XT, SHIFT> xin(p.x, row_offset(p.x, row, p.dims, p.flat)), yin(p.dy, row_offset(p.dy, row, p.dims, p.flat));
        const RowIn<ST, SHIFT> sin(p.dsum, DSUM ? row_offset(p.dsum, row, p.dims, p.flat) : 0);
        uint32_t xs[NV][W], ys[NV][W];
        typename RowIn<ST, SHIFT>::Raw ds[NV];
        {
            typename RowIn<XT, SHIFT>::Raw xr[NV], yr[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (run.size(i)) {
                    xin.load(xr[i], run.col(i));
                    yin.load(yr[i], run.col(i));
                    sin.load(ds[i], run.col(i));
                }
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (run.any(i)) {
                    xin.words(xr[i], xs[i]);
                    yin.words(yr[i], ys[i]);
                }
        }
        float2 squares = both(0.0f), dot = both(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = run.size(i);
            if (n) {
                float2 g[4], x[4], y[4];
                unpack<XT>(xs[i], x);
                unpack<XT>(ys[i], y);
                if (SHIFT && n < 8) clear_missing(x, y, n);
                if (p.gamma_type != ROW_NONE) {
                    load_gamma<SHIFT>(g, p.gamma, p.gamma_type, p.gamma_whole, run.col(i), n);
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] = __fmul2_rn(y[k], g[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    squares = __ffma2_rn(x[k], x[k], squares);
                    dot = __ffma2_rn(y[k], x[k], dot);
                }
            }
        }
        // two buffers: the next row's sums may start before all have read
        const float2 s = reduce_row<BLOCK, false>(squares.x + squares.y, dot.x + dot.y, blockDim.x >> 5, scratch[turn]);
        const float inv = inverse_rms(s.x, p.per_col, p.eps);
        const float mean_au = s.y * p.per_col * inv;
        RowOut<XT, SHIFT> out(p.dx, row_offset(p.dx, row, p.dims, p.flat));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = run.size(i);
            if (SHIFT ? run.any(i) : n != 0) {
                float2 x[4], y[4], a[4], add[4];
                unpack<XT>(xs[i], x);
                unpack<XT>(ys[i], y);
                if constexpr (DSUM) {
                    uint32_t sw[W];
                    sin.words(ds[i], sw);
                    unpack<XT>(sw, add);
                }
                if (p.gamma_type != ROW_NONE) {
                    load_gamma<SHIFT>(a, p.gamma, p.gamma_type, p.gamma_whole, run.col(i), n);
#pragma unroll
                    for (int k = 0; k < 4; ++k) a[k] = __fmul2_rn(a[k], y[k]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) a[k] = y[k];
                }
                grad_piece<DSUM>(x, y, a, add, inv, mean_au, acc[i]);   // the sums of missing elements are never read
                uint32_t w[W];
                pack<XT>(a, w);
                out.store(run.col(i), n, w, run.whole(i), i == 0, run.last(i, NV));
            }
        }
    }
    if (!p.partial) return;
    float* mine = p.partial + uint64_t(blockIdx.x) * p.cols;
    if constexpr (!BLOCK) {
        for (uint32_t w = 0; w < 4; ++w) {   // the warps add their sums in turn: the order is fixed
            if (sub == w) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t c = run.col(i) + e;
                        const float mine_c = (e & 1) ? acc[i][e >> 1].y : acc[i][e >> 1].x;
                        if (c < p.cols) block_sums[c] = w ? block_sums[c] + mine_c : mine_c;
                    }
            }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < p.cols; c += blockDim.x) mine[c] = block_sums[c];
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = run.col(i);
            if (!SHIFT && c < p.cols) {   // cols is a multiple of eight, and a block's row of `partial` starts on 16 bytes
                reinterpret_cast<float4*>(mine + c)[0] = make_float4(acc[i][0].x, acc[i][0].y, acc[i][1].x, acc[i][1].y);
                reinterpret_cast<float4*>(mine + c)[1] = make_float4(acc[i][2].x, acc[i][2].y, acc[i][3].x, acc[i][3].y);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < p.cols) mine[c + e] = (e & 1) ? acc[i][e >> 1].y : acc[i][e >> 1].x;
            }
        }
    }
}
// Rows too long for registers: both passes read from memory, the sums of dgamma are kept in the block's row of `partial`
// (every lane its own columns, so no two threads touch a word).
template <int XT, bool DSUM, bool SHIFT>
__global__ void __launch_bounds__(1024) norm_grad_long_kernel(const __grid_constant__ NormGradParams p) {
    constexpr int ST = DSUM ? XT : ROW_NONE, W = 2 * RowElem<XT>::kBytes;
    __shared__ float2 scratch[2][32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t pieces = (p.cols + 32 * 256 - 1) / (32 * 256);
    const WarpRun<SHIFT> run{(threadIdx.x >> 5) * 256 * pieces, p.cols};
    float* mine = p.partial ? p.partial + uint64_t(blockIdx.x) * p.cols : nullptr;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const RowIn<XT, SHIFT> xin(p.x, row_offset(p.x, row, p.dims, p.flat)), yin(p.dy, row_offset(p.dy, row, p.dims, p.flat));
        const RowIn<ST, SHIFT> sin(p.dsum, DSUM ? row_offset(p.dsum, row, p.dims, p.flat) : 0);
        auto read = [&](uint32_t i, int n, float2 (&x)[4], float2 (&y)[4], float2 (&a)[4]) {
            typename RowIn<XT, SHIFT>::Raw xr, yr;
            uint32_t xw[W], yw[W];
            xin.load(xr, run.col(i));
            yin.load(yr, run.col(i));
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = both(1.0f);
            if (p.gamma_type != ROW_NONE) load_gamma<SHIFT>(a, p.gamma, p.gamma_type, p.gamma_whole, run.col(i), n);
            xin.words(xr, xw);
            yin.words(yr, yw);
            unpack<XT>(xw, x);
            unpack<XT>(yw, y);
            if (SHIFT && n < 8) clear_missing(x, y, n);
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = __fmul2_rn(a[k], y[k]);
        };
        float2 squares = both(0.0f), dot = both(0.0f);
#pragma unroll 1
        for (uint32_t i = 0; i < pieces && run.any(i); ++i) {
            const int n = run.size(i);
            if (n) {
                float2 x[4], y[4], a[4];
                read(i, n, x, y, a);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    squares = __ffma2_rn(x[k], x[k], squares);
                    dot = __ffma2_rn(a[k], x[k], dot);
                }
            }
        }
        const float2 s = reduce_row<true, false>(squares.x + squares.y, dot.x + dot.y, 32, scratch[turn]);
        const float inv = inverse_rms(s.x, p.per_col, p.eps);
        const float mean_au = s.y * p.per_col * inv;
        const bool first = row == blockIdx.x;
        RowOut<XT, SHIFT> out(p.dx, row_offset(p.dx, row, p.dims, p.flat));
#pragma unroll 1
        for (uint32_t i = 0; i < pieces && run.any(i); ++i) {
            const uint32_t c = run.col(i);
            const int n = run.size(i);
            uint32_t w[W];
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] = 0;
            if (n) {
                float2 x[4], y[4], a[4], add[4], acc[4];
                read(i, n, x, y, a);
                if constexpr (DSUM) {
                    typename RowIn<ST, SHIFT>::Raw sr;
                    uint32_t sw[W];
                    sin.load(sr, c);
                    sin.words(sr, sw);
                    unpack<XT>(sw, add);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = both(0.0f);
                if (mine && !first) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < n) ((e & 1) ? acc[e >> 1].y : acc[e >> 1].x) = mine[c + e];
                }
                grad_piece<DSUM>(x, y, a, add, inv, mean_au, acc);
                if (mine) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < n) mine[c + e] = (e & 1) ? acc[e >> 1].y : acc[e >> 1].x;
                }
                pack<XT>(a, w);
            }
            if (SHIFT || n) out.store(c, n, w, run.whole(i), i == 0, run.last(i, pieces));
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
// x is read twice; the second pass walks the rows from the end, so that it begins with what the first left in L2.
template <int XT, bool SHIFT>
__device__ __forceinline__ void column_values(const QuantTransParams& p, uint32_t row, const typename RowIn<XT, SHIFT>::Raw& x, float2 (&v)[4]) {
    const RowIn<XT, SHIFT> in(p.x, uint64_t(row) * p.x_ld);
    uint32_t w[RowIn<XT, SHIFT>::kWords];
    in.words(x, w);
    unpack<XT>(w, v);
}
template <int XT, bool SHIFT>
__global__ void __launch_bounds__(256) column_max_kernel(const __grid_constant__ QuantTransParams p) {
    __shared__ float part[8][257];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 256 + lane * 8;
    const int n = piece_size(c, p.cols);
    const uint32_t rows_per = (p.rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * rows_per, r1 = min(p.rows, r0 + rows_per);
    float2 top[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) top[k] = both(0.0f);
    if (n) {
#pragma unroll 1
        for (uint32_t r = r0 + warp; r < r1; r += 32) {
            typename RowIn<XT, SHIFT>::Raw x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r + 8 * j < r1) RowIn<XT, SHIFT>(p.x, uint64_t(r + 8 * j) * p.x_ld).load(x[j], c);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r + 8 * j < r1) {
                    float2 v[4];
                    column_values<XT, SHIFT>(p, r + 8 * j, x[j], v);
#pragma unroll
                    for (int k = 0; k < 4; ++k)   // of missing columns: never read
                        top[k] = make_float2(max_nan(top[k].x, fabsf(v[k].x)), max_nan(top[k].y, fabsf(v[k].y)));
                }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[warp][e * 32 + lane] = (e & 1) ? top[e >> 1].y : top[e >> 1].x;
    __syncthreads();
    const uint32_t mine = blockIdx.x * 256 + (threadIdx.x & 31) * 8 + (threadIdx.x >> 5);
    float t = part[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 8; ++i) t = max_nan(t, part[i][threadIdx.x]);
    if (mine < p.cols) atomicMax(reinterpret_cast<uint32_t*>(p.scale) + mine, __float_as_uint(t) & 0x7FFFFFFFu);
}
// Tiles of 128 rows x 64 columns, kTransTiles of them one below the other per block: a thread takes four rows of eight
// columns, whose codes make one word per column. A tile's columns leave as aligned 16-byte words (byte by byte at their ends).
constexpr uint32_t kTransTiles = 4;
template <int XT, bool SHIFT, bool I8, bool GIVEN>
__global__ void __launch_bounds__(256) quant_trans_kernel(const __grid_constant__ QuantTransParams p) {
    constexpr uint32_t kPitch = 33;   // words: 128 rows and one word that keeps the banks apart
    __shared__ uint32_t tile[64 * kPitch + 4];
    __shared__ CodeStep steps[64];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t c0 = blockIdx.x * 64;
    if (threadIdx.x < 64) {
        const uint32_t c = c0 + threadIdx.x;
        float s = 0.0f;
        if (c < p.cols) s = GIVEN ? p.given[uint64_t(c) * p.given_stride] : __fdiv_rn(p.scale[c], p.top);
        steps[threadIdx.x] = make_code_step(s);
    }
    const uint32_t cg = threadIdx.x & 7, rq = threadIdx.x >> 3, cc = c0 + cg * 8;
    const bool exists = cc < p.cols;
#pragma unroll 1
    for (uint32_t t = 0; t < kTransTiles; ++t) {
        const uint32_t block = gridDim.y - 1 - blockIdx.y, r0 = (block * kTransTiles + (kTransTiles - 1 - t)) * 128;
        if (r0 >= p.rows) continue;   // uniform over the block
        const uint32_t r = r0 + rq * 4;
        typename RowIn<XT, SHIFT>::Raw x[4];
        float2 v[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (exists && r + j < p.rows) RowIn<XT, SHIFT>(p.x, uint64_t(p.row0 + r + j) * p.x_ld).load(x[j], cc);
        __syncthreads();   // the steps are there, and the tile before has left
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (exists && r + j < p.rows) column_values<XT, SHIFT>(p, p.row0 + r + j, x[j], v[j]);
            else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[j][k] = both(0.0f);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t c = cg * 8 + 2 * k;
            tile[c * kPitch + rq] = make_codes<I8, GIVEN>(make_float2(v[0][k].x, v[1][k].x), make_float2(v[2][k].x, v[3][k].x), steps[c], p.hw);
            tile[(c + 1) * kPitch + rq] = make_codes<I8, GIVEN>(make_float2(v[0][k].y, v[1][k].y), make_float2(v[2][k].y, v[3][k].y), steps[c + 1], p.hw);
        }
        __syncthreads();
        const uint32_t rows = min(128u, p.rows - r0), cols = min(64u, p.cols - c0);
        // nine 16-byte words cover a column's 128 bytes at any alignment
        for (uint32_t i = threadIdx.x; i < cols * 9; i += 256) {
            const uint32_t col = i / 9, k = i % 9;
            uint8_t* a = static_cast<uint8_t*>(p.out) + uint64_t(c0 + col) * p.out_ld + p.row0 + r0;
            const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(a)) & 15u;
            const int begin = int(16 * k) - int(off);   // first row of the word
            if (begin >= int(rows)) continue;
            const uint32_t* column = tile + col * kPitch;
            if (begin >= 0 && begin + 16 <= int(rows)) {
                const uint32_t q = uint32_t(begin) >> 2, sh = (uint32_t(begin) & 3u) * 8;
                uint32_t w[5], o[4];
    #pragma unroll
                for (int j = 0; j < 5; ++j) w[j] = column[q + j];   // the fifth word (the padding, at the end) counts only when sh != 0
    #pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = __funnelshift_r(w[j], w[j + 1], sh);
                *reinterpret_cast<uint4*>(a + begin) = make_uint4(o[0], o[1], o[2], o[3]);
            } else {
                for (int r = max(begin, 0); r < min(begin + 16, int(rows)); ++r) a[r] = uint8_t(column[r >> 2] >> (8 * (r & 3)));
            }
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
