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

// act(v) on N values at once: the choice is the same for the whole launch, so it is made once per N values.  A NaN stays
// a NaN in every activation.  The logistic function is v / (1 + exp(-v)) on the hardware's exponential: its error, a
// few units in the 24th bit for arguments that matter, is weighed by v * exp(-v) for positive v and by the result's own
// smallness for negative v, and stays under 3e-7 of the result's scale.
__device__ __forceinline__ float logistic_times(float v, float u) { return __fdividef(v, 1.0f + __expf(-u)); }
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
    switch (act) {
        case kActRelu:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
            break;
        case kActRelu2:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float r = v[i] < 0.0f ? 0.0f : v[i];
                v[i] = __fmul_rn(r, r);
            }
            break;
        case kActSilu:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = logistic_times(v[i], v[i]);
            break;
        case kActGelu:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678f));
            break;
        case kActGeluTanh:       // 0.5 v (1 + tanh u) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
#pragma unroll
            for (int i = 0; i < N; ++i)
                v[i] = logistic_times(v[i], 1.5957691f * fmaf(__fmul_rn(0.044715f * v[i], v[i]), v[i], v[i]));
            break;
        default: break;
    }
}

// The int32 product itself: the kernels keep their own stores.
struct StoreInt32 {
    static constexpr bool kFused = false;
};

struct FusedEpilogue {
    static constexpr bool kFused = true;
    const float* row_scale;        // [M]
    const float* col_scale;        // [N], or null: w_scale for every column
    const void* bias;              // [N] of bias_dtype, or null
    const void* residual;          // [M][ldr] of out_dtype, or null; may be `out` itself (an element is read before it is written)
    void* out;                     // [M][ldo] of out_dtype
    long long ldo, ldr;
    float w_scale;
    int bias_dtype, act, out_dtype;
    int vec4;                      // four columns from a multiple of four can be moved as one access (out and residual)

    __device__ __forceinline__ float column_scale(int col) const { return col_scale ? __ldg(col_scale + col) : w_scale; }
    __device__ __forceinline__ float column_bias(int col) const {
        if (!bias) return 0.0f;
        if (bias_dtype == kDtypeF32) return __ldg(static_cast<const float*>(bias) + col);
        if (bias_dtype == kDtypeBf16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(bias) + col));
        return __half2float(__ldg(static_cast<const __half*>(bias) + col));
    }
    // Before the activation.  Without a bias nothing is added (0 would turn -0 into +0: harmless, and one instruction).
    __device__ __forceinline__ float linear(int32_t c, float rs, float cs, float b) const {
        return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(c), rs), cs), b);
    }

    template <typename T>
    __device__ __forceinline__ void finish_t(int row, int col, float v) const {
        T* o = static_cast<T*>(out) + static_cast<size_t>(row) * ldo + col;
        if (residual) v = __fadd_rn(v, to_float<T>(static_cast<const T*>(residual)[static_cast<size_t>(row) * ldr + col]));
        *o = from_float<T>(v);
    }
    // One activated value: residual and store.
    __device__ __forceinline__ void finish(int row, int col, float v) const {
        if (out_dtype == kDtypeBf16) finish_t<__nv_bfloat16>(row, col, v);
        else if (out_dtype == kDtypeF16) finish_t<__half>(row, col, v);
        else finish_t<float>(row, col, v);
    }
    __device__ __forceinline__ void store(int row, int col, int32_t c) const {
        float v[1] = {linear(c, __ldg(row_scale + row), column_scale(col), column_bias(col))};
        activate(act, v);
        finish(row, col, v[0]);
    }

    // The residual of four columns, as it lies in memory (vec4 only): issued early, used by finish4().
    __device__ __forceinline__ uint4 load_residual4(int row, int col) const {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (!residual || !vec4) return raw;
        const size_t at = static_cast<size_t>(row) * ldr + col;
        if (out_dtype == kDtypeF32) {
            raw = *reinterpret_cast<const uint4*>(static_cast<const float*>(residual) + at);
        } else {
            const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(residual) + at);
            raw.x = r.x;
            raw.y = r.y;
        }
        return raw;
    }
    template <typename T>
    __device__ __forceinline__ void finish4_half(int row, int col, float (&v)[4], const uint4& raw) const {
        union { uint2 u; T t[4]; } x;
        if (residual) {
            x.u = make_uint2(raw.x, raw.y);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(v[i], to_float<T>(x.t[i]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x.t[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint2*>(static_cast<T*>(out) + static_cast<size_t>(row) * ldo + col) = x.u;
    }
    // Four activated values of columns col .. col + 3 (col a multiple of four).
    __device__ __forceinline__ void finish4(int row, int col, float (&v)[4], const uint4& raw) const {
        if (!vec4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) finish(row, col + i, v[i]);
        } else if (out_dtype == kDtypeBf16) {
            finish4_half<__nv_bfloat16>(row, col, v, raw);
        } else if (out_dtype == kDtypeF16) {
            finish4_half<__half>(row, col, v, raw);
        } else {
            if (residual) {
                v[0] = __fadd_rn(v[0], __uint_as_float(raw.x));
                v[1] = __fadd_rn(v[1], __uint_as_float(raw.y));
                v[2] = __fadd_rn(v[2], __uint_as_float(raw.z));
                v[3] = __fadd_rn(v[3], __uint_as_float(raw.w));
            }
            *reinterpret_cast<float4*>(static_cast<float*>(out) + static_cast<size_t>(row) * ldo + col) =
                make_float4(v[0], v[1], v[2], v[3]);
        }
    }
    __device__ __forceinline__ void store4(int row, int col, const int32_t (&c)[4]) const {
        const uint4 raw = load_residual4(row, col);
        const float rs = __ldg(row_scale + row);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = linear(c[i], rs, column_scale(col + i), column_bias(col + i));
        activate(act, v);
        finish4(row, col, v, raw);
    }
};

}  // namespace tb200
