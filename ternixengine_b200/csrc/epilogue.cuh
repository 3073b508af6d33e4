// What a product kernel does with a finished sum: either store it as int32 (the product itself), or take it through
// the rest of a layer's linear step in registers,
//     y[m][n] = T( act( (float(c) * row_scale[m]) * col_scale[n] + bias[n] ) + residual[m][n] ),
// so that the int32 product never reaches global memory.  All arithmetic is fp32 with every operation rounded on its
// own (no contraction into fused multiply-adds), in this order, in every kernel: the result does not depend on which
// kernel the dispatch picked.  There is one rounding to fewer bits, at the end, to the output's type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

namespace tb200 {

// TERNIX_B200_DTYPE_* and TERNIX_B200_ACT_* of the C ABI
constexpr int kDtypeF32 = 0, kDtypeBf16 = 1, kDtypeF16 = 2;
constexpr int kActNone = 0, kActRelu = 1, kActRelu2 = 2, kActSilu = 3, kActGelu = 4, kActGeluTanh = 5;

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// One instruction each: maximum that keeps a NaN, 2^x (relative error 2^-22) and 1 / x (1 ulp), subnormals flushed.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// v / (1 + exp(-u)).  The exponential's error, 2^-22 and |u| 2^-23 from its argument, is weighed by exp(-u) / (1 + exp(-u));
// a denominator above 2^126 gives 0 (the quotient is below |v| 2^-126).
__device__ __forceinline__ float logistic_times(float v, float u) {
    return v * rcp_approx(1.0f + exp2_approx(-1.44269504f * u));
}
// log2 of P(v) / P(-v) over v, P the normal distribution: v P(v), the exact GELU, is v / (1 + 2^(-that v)).  Odd in v and smooth, so
// a polynomial in v^2; this one is a least-squares fit in Chebyshev points of v^2 on [0, 32], weighted by |v| P(v) P(-v) and
// reweighted (Lawson's method) until the error in v P(v) is level.  With the coefficients as float32, v P(v) is off by at most
// 1.2e-8 for every v: beyond v^2 = 32 the logit stays constant, P(-v) goes on falling, and what it is off by is below that too.
__device__ __forceinline__ float gelu_logit(float v) {
    const float u = fminf(__fmul_rn(v, v), 32.0f);
    float r = 4.3443146e-13f;
    r = fmaf(r, u, -4.3081289e-11f);
    r = fmaf(r, u, 1.6313341e-09f);
    r = fmaf(r, u, -2.5466631e-08f);
    r = fmaf(r, u, -7.5623149e-08f);
    r = fmaf(r, u, 9.7798011e-06f);
    r = fmaf(r, u, -1.5490042e-04f);
    r = fmaf(r, u, -1.0019503e-04f);
    r = fmaf(r, u, 0.10483802f);
    return fmaf(r, u, 2.3022091f);
}
// The same three functions for float32 data, where the roundings of sum, reciprocal and product above would show: with e the
// exponential of minus the argument's absolute value, v / (1 + e) is v - v e / (1 + e) for v > 0 and v e / (1 + e) below, so
// that every rounding but the last is of something small.  v P(v) is then off by at most 2^-24 of itself, the fit, and 9 x
// 2^-24 and the argument's rounding as parts of |v| P(-|v|), which is at most 0.17 (0.28 for SiLU).  Largest error on the CPU
// restatement with exact exponentials, fine | short | v (1 + erf) / 2: GELU 1.0e-7 | 2.3e-7 | 1.6e-7 for v in 1 .. 2, 2.5e-7 |
// 5.3e-7 | 4.5e-7 in 4 .. 6, 5.2e-8 | 4.7e-8 | 4.7e-8 in -2 .. -1, 2.6e-8 | 2.5e-8 | 4.8e-8 in -3 .. -2.
// An infinity below gives NaN (the product of infinity and zero), as in the short forms; one above stays.
__device__ __forceinline__ float fine_times(float v, float e) {
    const float q = e * rcp_approx(1.0f + e), a = fmaxf(-v, fminf(v, 128.0f));        // |v|; e is 0 beyond 128
    return fmaf(-a, q, max_nan(v, 0.0f));
}
// exp(-|u|): what the argument loses by its rounding is put back in first order.
__device__ __forceinline__ float exp_fine(float u) {
    const float a = fminf(fabsf(u), 128.0f), t = __fmul_rn(a, -1.44269504f), e = exp2_approx(t);
    return fmaf(e, fmaf(t, -0.69314718f, -a), e);
}
// act(v) on N values at once: the choice is the same for the whole launch, so it is made once per N values.  A NaN stays
// a NaN in every activation.  kFine: for float32 data; 16-bit data round 2^13 times and more coarser than the short forms.
template <bool kFine, int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
    switch (act) {
        case kActRelu:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = max_nan(v[i], 0.0f);
            break;
        case kActRelu2:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float r = max_nan(v[i], 0.0f);
                v[i] = __fmul_rn(r, r);
            }
            break;
        case kActSilu:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (kFine) v[i] = fine_times(v[i], exp_fine(v[i]));
                else v[i] = logistic_times(v[i], v[i]);
            }
            break;
        case kActGelu:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (kFine) v[i] = fine_times(v[i], exp2_approx(-__fmul_rn(fabsf(v[i]), gelu_logit(v[i]))));
                else v[i] = v[i] * rcp_approx(1.0f + exp2_approx(-__fmul_rn(v[i], gelu_logit(v[i]))));
            }
            break;
        case kActGeluTanh:       // 0.5 v (1 + tanh u) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float u2 = 1.5957691f * fmaf(__fmul_rn(0.044715f * v[i], v[i]), v[i], v[i]);
                if constexpr (kFine) v[i] = fine_times(v[i], exp_fine(u2));
                else v[i] = logistic_times(v[i], u2);
            }
            break;
        default: break;
    }
}

// The int32 product itself: the kernels keep their own stores.
struct StoreInt32 {
    static constexpr bool kFused = false;
};

// k32: the output and the residual are float32; else 16 bits wide, bfloat16 or float16 by out_dtype.
// All its operands may have been written by the kernel before, which this one may have overlapped up to dependent_wait():
// they are read with ordinary loads, never through the read-only path (whose loads a compiler may move and whose data has
// to hold for the kernel's whole life).
template <bool k32>
struct FusedEpilogue {
    static constexpr bool kFused = true;
    using Raw = std::conditional_t<k32, uint4, uint2>;       // four residual values as they lie in memory
    const float* row_scale;        // [M]
    const float* col_scale;        // [N], or null: w_scale for every column
    const void* bias;              // [N] of bias_dtype, or null
    const void* residual;          // [M][ldr] of out_dtype, or null; may be `out` itself (an element is read before it is written)
    void* out;                     // [M][ldo] of out_dtype
    long long ldo, ldr;
    float w_scale;
    int bias_dtype, act, out_dtype;
    int vec4;                      // four columns from a multiple of four can be moved as one access (out and residual)

    __device__ __forceinline__ float column_scale(int col) const { return col_scale ? col_scale[col] : w_scale; }
    __device__ __forceinline__ float column_bias(int col) const {
        if (!bias) return 0.0f;
        if (bias_dtype == kDtypeF32) return static_cast<const float*>(bias)[col];
        if (bias_dtype == kDtypeBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[col]);
        return __half2float(static_cast<const __half*>(bias)[col]);
    }
    template <int N>
    __device__ __forceinline__ void activate(float (&v)[N]) const { tb200::activate<k32>(act, v); }
    // Before the activation.  Without a bias 0 is added, which only turns -0 into +0.
    __device__ __forceinline__ float linear(int32_t c, float rs, float cs, float b) const {
        return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(c), rs), cs), b);
    }

    __device__ __forceinline__ float from_bits(uint32_t b) const {           // low 16 bits
        return out_dtype == kDtypeBf16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(b)));
    }
    __device__ __forceinline__ uint32_t to_bits(float v) const {
        return out_dtype == kDtypeBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
    }
    // One activated value: residual and store.
    __device__ __forceinline__ void finish(int row, int col, float v) const {
        const size_t at_r = static_cast<size_t>(row) * ldr + col, at_o = static_cast<size_t>(row) * ldo + col;
        if constexpr (k32) {
            if (residual) v = __fadd_rn(v, static_cast<const float*>(residual)[at_r]);
            static_cast<float*>(out)[at_o] = v;
        } else {
            if (residual) v = __fadd_rn(v, from_bits(static_cast<const uint16_t*>(residual)[at_r]));
            static_cast<uint16_t*>(out)[at_o] = static_cast<uint16_t>(to_bits(v));
        }
    }
    __device__ __forceinline__ void store(int row, int col, int32_t c) const {
        float v[1] = {linear(c, row_scale[row], column_scale(col), column_bias(col))};
        activate(v);
        finish(row, col, v[0]);
    }

    // The residual of columns col .. col + 3 (col a multiple of four): issued early, used by finish4().
    __device__ __forceinline__ Raw load_residual4(int row, int col) const {
        Raw raw{};
        if (!residual) return raw;
        const size_t at = static_cast<size_t>(row) * ldr + col;
        if constexpr (k32) {
            const float* p = static_cast<const float*>(residual) + at;
            if (vec4) raw = *reinterpret_cast<const uint4*>(p);
            else raw = make_uint4(__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3]));
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(residual) + at;
            if (vec4) raw = *reinterpret_cast<const uint2*>(p);
            else raw = make_uint2(p[0] | static_cast<uint32_t>(p[1]) << 16, p[2] | static_cast<uint32_t>(p[3]) << 16);
        }
        return raw;
    }
    // Asks for `count` residual values of a row to be brought into L2.
    __device__ __forceinline__ void prefetch_residual(int row, int col, int count) const {
        constexpr int kBytes = k32 ? 4 : 2;
        const char* p = static_cast<const char*>(residual) + (static_cast<size_t>(row) * ldr + col) * kBytes;
        for (int b = 0; b < count * kBytes; b += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + b));
    }
    // Four activated values of columns col .. col + 3.
    __device__ __forceinline__ void finish4(int row, int col, const float* v, const Raw& raw) const {
        const size_t at = static_cast<size_t>(row) * ldo + col;
        if constexpr (k32) {
            float4 y = make_float4(v[0], v[1], v[2], v[3]);
            if (residual)
                y = make_float4(__fadd_rn(y.x, __uint_as_float(raw.x)), __fadd_rn(y.y, __uint_as_float(raw.y)),
                                __fadd_rn(y.z, __uint_as_float(raw.z)), __fadd_rn(y.w, __uint_as_float(raw.w)));
            float* o = static_cast<float*>(out) + at;
            if (vec4) *reinterpret_cast<float4*>(o) = y;
            else { o[0] = y.x; o[1] = y.y; o[2] = y.z; o[3] = y.w; }
        } else {
            float y[4] = {v[0], v[1], v[2], v[3]};
            if (residual) {
                y[0] = __fadd_rn(y[0], from_bits(raw.x & 0xffffu));
                y[1] = __fadd_rn(y[1], from_bits(raw.x >> 16));
                y[2] = __fadd_rn(y[2], from_bits(raw.y & 0xffffu));
                y[3] = __fadd_rn(y[3], from_bits(raw.y >> 16));
            }
            uint32_t lo, hi;             // two roundings and the packing are one instruction
            if (out_dtype == kDtypeBf16) {
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(y[1]), "f"(y[0]));
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y[3]), "f"(y[2]));
            } else {
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(y[1]), "f"(y[0]));
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y[3]), "f"(y[2]));
            }
            uint16_t* o = static_cast<uint16_t*>(out) + at;
            if (vec4) *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
            else { o[0] = lo & 0xffffu; o[1] = lo >> 16; o[2] = hi & 0xffffu; o[3] = hi >> 16; }
        }
    }
    // The residual of R rows, all inside the output, vec4 only.
    template <int R>
    __device__ __forceinline__ void load_residual_rows(int row, int col, Raw* raw) const {
        constexpr int kBytes = k32 ? 4 : 2;
        const char* p = static_cast<const char*>(residual) + (static_cast<size_t>(row) * ldr + col) * kBytes;
        const size_t step = static_cast<size_t>(ldr) * kBytes;
#pragma unroll
        for (int j = 0; j < R; ++j) raw[j] = *reinterpret_cast<const Raw*>(p + j * step);
    }
    // R rows of four activated values (fp32 bits) each, all inside the output, vec4 only: the choices are made once.
    template <int R, bool kRes>
    __device__ __forceinline__ void finish_rows(int row, int col, const uint4 (&y)[R], const Raw* raw) const {
        constexpr int kBytes = k32 ? 4 : 2;
        char* o = static_cast<char*>(out) + (static_cast<size_t>(row) * ldo + col) * kBytes;
        const size_t step = static_cast<size_t>(ldo) * kBytes;
        float v[R][4];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            v[j][0] = __uint_as_float(y[j].x); v[j][1] = __uint_as_float(y[j].y);
            v[j][2] = __uint_as_float(y[j].z); v[j][3] = __uint_as_float(y[j].w);
        }
        if constexpr (k32) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if constexpr (kRes) {
                    v[j][0] = __fadd_rn(v[j][0], __uint_as_float(raw[j].x)); v[j][1] = __fadd_rn(v[j][1], __uint_as_float(raw[j].y));
                    v[j][2] = __fadd_rn(v[j][2], __uint_as_float(raw[j].z)); v[j][3] = __fadd_rn(v[j][3], __uint_as_float(raw[j].w));
                }
                *reinterpret_cast<float4*>(o + j * step) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
            }
        } else if (out_dtype == kDtypeBf16) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if constexpr (kRes) {
                    v[j][0] = __fadd_rn(v[j][0], __uint_as_float(raw[j].x << 16)); v[j][1] = __fadd_rn(v[j][1], __uint_as_float(raw[j].x & 0xffff0000u));
                    v[j][2] = __fadd_rn(v[j][2], __uint_as_float(raw[j].y << 16)); v[j][3] = __fadd_rn(v[j][3], __uint_as_float(raw[j].y & 0xffff0000u));
                }
                uint2 b;
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.x) : "f"(v[j][1]), "f"(v[j][0]));
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.y) : "f"(v[j][3]), "f"(v[j][2]));
                *reinterpret_cast<uint2*>(o + j * step) = b;
            }
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if constexpr (kRes) {
                    v[j][0] = __fadd_rn(v[j][0], from_bits(raw[j].x & 0xffffu)); v[j][1] = __fadd_rn(v[j][1], from_bits(raw[j].x >> 16));
                    v[j][2] = __fadd_rn(v[j][2], from_bits(raw[j].y & 0xffffu)); v[j][3] = __fadd_rn(v[j][3], from_bits(raw[j].y >> 16));
                }
                uint2 b;
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(b.x) : "f"(v[j][1]), "f"(v[j][0]));
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(b.y) : "f"(v[j][3]), "f"(v[j][2]));
                *reinterpret_cast<uint2*>(o + j * step) = b;
            }
        }
    }
    __device__ __forceinline__ void store4(int row, int col, const int32_t (&c)[4]) const {
        const Raw raw = load_residual4(row, col);
        const float rs = row_scale[row];
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = linear(c[i], rs, column_scale(col + i), column_bias(col + i));
        activate(v);
        finish4(row, col, v, raw);
    }
};

}  // namespace tb200
