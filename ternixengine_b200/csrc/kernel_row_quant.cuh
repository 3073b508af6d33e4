// The steps that produce a product's int8 activations, one pass over the data each:
//
//   norm      h = T(x + residual);  t = f32(h * w);              s = 1 / sqrt(mean(h^2) + eps)
//   gate      z = act(g) * u;       t = f32(z * w) or z;         s = 1 / sqrt(mean(z^2) + eps) or 1
//   both      m = max|t|;  q = rint(t * (127 / m));  row_scale = (m / 127) * s
//
// The norm's factor s is common to a row, so it cancels out of the codes: q depends on t and m only, and s goes into
// row_scale.  One reduction therefore gives both the maximum and the sum of squares, and a row is read once and held in
// registers until its codes are written.  Statistics and products are fp32; t is rounded to fp32 once.
//
// A row of zeros gets codes 0 and row_scale 1.  A row in which some t is infinite or NaN, or whose sum of squares
// leaves fp32, gets codes 0 and row_scale NaN, so that everything computed from it is NaN.  The maximum is taken with
// the NaN-propagating instruction and carried between lanes as bits (|NaN| > inf > any finite as integers).
// 127 / m would overflow for m below 2^-121; such rows are scaled up by 2^100 first, which is exact.
//
// One CTA per row, the row spread over its threads as VPT vectors of 16 bytes each.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "epilogue.cuh"

namespace tb200 {

constexpr int kRowNorm = 0, kRowNormResidual = 1, kRowGate = 2;

struct RowQuantArgs {
    const void* x;             // x, or the gate
    const void* y;             // the residual, or up
    const void* w;             // norm weight [K] of w_dtype, or null
    void* h;                   // x + residual (may be x or y itself: an element is read before it is written)
    int8_t* q;                 // [M][K]
    float* row_scale;          // [M]
    long long ldx, ldy, ldh;
    int M, K;
    float eps;                 // negative (gate only): no norm
    int w_dtype, act;
};

template <typename T>
constexpr int kRowVec = 16 / static_cast<int>(sizeof(T));      // elements of a 16-byte vector

// V elements as they lie in memory: a 16-byte vector, or one element.
template <typename T, int V>
union RowRaw {
    uint4 u;
    T t[16 / sizeof(T)];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V == 1) t[0] = *p;
        else u = *reinterpret_cast<const uint4*>(p);
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (V == 1) *p = t[0];
        else *reinterpret_cast<uint4*>(p) = u;
    }
};
template <typename T, int V>
__device__ __forceinline__ void row_load_weight(const void* w, int w_is_f32, int k, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = w_is_f32 ? __ldg(static_cast<const float*>(w) + k) : to_float<T>(static_cast<const T*>(w)[k]);
    } else {
        if (w_is_f32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + k);
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const float4 f = __ldg(p + i);
                v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
            }
        } else {
            union { uint4 u; T t[V]; } x;
            x.u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + k));
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = to_float<T>(x.t[i]);
        }
    }
}
// V elements of a row from column k, loaded as x and y: what is normalised and quantised (h or z).  Writes h on the way.
template <typename T, int MODE, int V>
__device__ __forceinline__ void row_element(const RowQuantArgs& p, int row, int k, RowRaw<T, V>& x, const RowRaw<T, V>& y,
                                            float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_float<T>(x.t[i]);
    if constexpr (MODE == kRowNormResidual) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            x.t[i] = from_float<T>(__fadd_rn(v[i], to_float<T>(y.t[i])));
            v[i] = to_float<T>(x.t[i]);
        }
        x.store(static_cast<T*>(p.h) + static_cast<size_t>(row) * p.ldh + k);
    } else if constexpr (MODE == kRowGate) {
        activate(p.act, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __fmul_rn(v[i], to_float<T>(y.t[i]));
    }
}
// Codes as the low bytes of t * inv + 1.5 * 2^23: the addition rounds to the nearest integer, ties to even, and leaves
// it in two's complement in the low bits; |t * inv| <= 127 (1 + 2^-22).
__device__ __forceinline__ uint32_t row_code(float t, float inv) {
    return __float_as_uint(__fadd_rn(__fmul_rn(t, inv), 12582912.0f));
}
__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Maximum (as bits) and sum over the CTA, in every thread.  One barrier; `turn` alternates between two sets of slots, so
// that the next row's partial results cannot overtake this row's readers.
__device__ __forceinline__ void row_reduce(uint32_t& top, float& sum, uint2 (*slots)[32], int turn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (warps == 1) return;
    if (lane == 0) slots[turn][warp] = make_uint2(top, __float_as_uint(sum));
    __syncthreads();
    const uint2 s = lane < warps ? slots[turn][lane] : make_uint2(0, 0);
    top = __reduce_max_sync(0xffffffffu, s.x);
    sum = __uint_as_float(s.y);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
}

// What the statistics of a row say about its codes.
struct RowScale {
    float lift, inv, scale;    // q = rint((t * lift) * inv)
    uint32_t keep;             // 0: the row's codes are all zero
};
__device__ __forceinline__ RowScale row_scale_of(uint32_t top, float sum, const RowQuantArgs& p) {
    RowScale r{1.0f, 0.0f, 1.0f, 0xffffffffu};
    const float m = __uint_as_float(top);
    const bool normed = p.eps >= 0.0f;
    if (top >= 0x7f800000u || (normed && !(sum < __uint_as_float(0x7f800000u)))) {
        r.scale = __uint_as_float(0x7fc00000u);
        r.keep = 0;
    } else if (m > 0.0f) {
        if (m < 1e-30f) r.lift = 1.2676506e30f;        // 2^100
        const float top_l = __fmul_rn(m, r.lift);
        r.inv = __fdiv_rn(127.0f, top_l);
        r.scale = __fdiv_rn(top_l, 127.0f);
        if (normed) r.scale = __fmul_rn(r.scale, __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.K)), p.eps))));
        if (r.lift != 1.0f) r.scale = __fmul_rn(r.scale, 7.8886091e-31f);      // 2^-100: the one rounding to a subnormal
    }
    return r;
}

template <typename T, int MODE, int VPT, bool kVec>
__global__ void __launch_bounds__(1024)
row_quant_kernel(const __grid_constant__ RowQuantArgs p) {
    constexpr int V = kVec ? kRowVec<T> : 1;
    __shared__ uint2 slots[2][32];
    const int w_is_f32 = p.w_dtype == kDtypeF32;
    int turn = 0;
    for (int row = blockIdx.x; row < p.M; row += gridDim.x, turn ^= 1) {
        float t[VPT][V];
        float top_f = 0.0f, sum = 0.0f;
        // all of the row's loads first: a store of h between them would hold the next ones back (h may be x or y)
        RowRaw<T, V> x[VPT], y[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int k = (threadIdx.x + j * blockDim.x) * V;
            x[j].u = y[j].u = make_uint4(0, 0, 0, 0);
            if (k < p.K) {
                x[j].load(static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx + k);
                if constexpr (MODE != kRowNorm) y[j].load(static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy + k);
            }
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int k = (threadIdx.x + j * blockDim.x) * V;
            if (k < p.K) {
                row_element<T, MODE, V>(p, row, k, x[j], y[j], t[j]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) t[j][i] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int k = (threadIdx.x + j * blockDim.x) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) sum = fmaf(t[j][i], t[j][i], sum);
            if (p.w && k < p.K) {
                float w[V];
                row_load_weight<T, V>(p.w, w_is_f32, k, w);
#pragma unroll
                for (int i = 0; i < V; ++i) t[j][i] = __fmul_rn(t[j][i], w[i]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) top_f = max_nan(top_f, fabsf(t[j][i]));
        }
        uint32_t top = __float_as_uint(top_f);
        row_reduce(top, sum, slots, turn);
        const RowScale r = row_scale_of(top, sum, p);
        if (threadIdx.x == 0) p.row_scale[row] = r.scale;
        int8_t* q = p.q + static_cast<size_t>(row) * p.K;
        if (r.lift != 1.0f) {
#pragma unroll
            for (int j = 0; j < VPT; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) t[j][i] *= r.lift;
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int k = (threadIdx.x + j * blockDim.x) * V;
            if (k >= p.K) continue;
            if constexpr (V == 1) {
                q[k] = static_cast<int8_t>(row_code(t[j][0], r.inv) & r.keep);
            } else {
                uint32_t c[V / 4];
#pragma unroll
                for (int i = 0; i < V / 4; ++i)
                    c[i] = pack_codes(row_code(t[j][4 * i], r.inv), row_code(t[j][4 * i + 1], r.inv),
                                      row_code(t[j][4 * i + 2], r.inv), row_code(t[j][4 * i + 3], r.inv)) & r.keep;
                if constexpr (V == 8) *reinterpret_cast<uint2*>(q + k) = make_uint2(c[0], c[1]);
                else *reinterpret_cast<uint32_t*>(q + k) = c[0];
            }
        }
    }
}

// Rows that do not fit the registers of a CTA: the same arithmetic, with the row computed twice.  The second pass reads
// h back instead of adding again (it may have replaced the residual).
template <typename T, int MODE>
__global__ void __launch_bounds__(1024)
row_quant_long_kernel(const __grid_constant__ RowQuantArgs p) {
    __shared__ uint2 slots[2][32];
    const int w_is_f32 = p.w_dtype == kDtypeF32;
    int turn = 0;
    for (int row = blockIdx.x; row < p.M; row += gridDim.x, turn ^= 1) {
        float top_f = 0.0f, sum = 0.0f;
        for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
            RowRaw<T, 1> x, y;
            float t[1];
            x.load(static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx + k);
            if constexpr (MODE != kRowNorm) y.load(static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy + k);
            row_element<T, MODE, 1>(p, row, k, x, y, t);
            sum = fmaf(t[0], t[0], sum);
            if (p.w) {
                float w[1];
                row_load_weight<T, 1>(p.w, w_is_f32, k, w);
                t[0] = __fmul_rn(t[0], w[0]);
            }
            top_f = max_nan(top_f, fabsf(t[0]));
        }
        uint32_t top = __float_as_uint(top_f);
        row_reduce(top, sum, slots, turn);
        const RowScale r = row_scale_of(top, sum, p);
        if (threadIdx.x == 0) p.row_scale[row] = r.scale;
        int8_t* q = p.q + static_cast<size_t>(row) * p.K;
        for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
            RowRaw<T, 1> x, y;
            float t[1];
            if constexpr (MODE == kRowNormResidual) {
                t[0] = to_float<T>(static_cast<const T*>(p.h)[static_cast<size_t>(row) * p.ldh + k]);
            } else {
                x.load(static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx + k);
                if constexpr (MODE == kRowGate) y.load(static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy + k);
                row_element<T, MODE, 1>(p, row, k, x, y, t);
            }
            if (p.w) {
                float w[1];
                row_load_weight<T, 1>(p.w, w_is_f32, k, w);
                t[0] = __fmul_rn(t[0], w[0]);
            }
            q[k] = static_cast<int8_t>(row_code(t[0] * r.lift, r.inv) & r.keep);
        }
    }
}

}  // namespace tb200
