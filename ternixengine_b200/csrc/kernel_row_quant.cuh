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
// A row belongs to one CTA (a cluster, where rows are few and long), spread over its threads as VPT vectors of 16 bytes each.  Where rows start or end off a 16-byte
// boundary the vectors are laid out so that their codes are aligned (the first and the last one may be partial), and a
// vector of an input is put together from the two aligned pieces that it lies in: odd rows, and the halves of a product's
// output with an odd width.  Two float32 inputs, and short rows of 16 bits, are taken as single elements there (launch_row_quant).
//
// Bound by memory: each input once, each output once.  Measured on B200 (copy rate 6.55 TB/s): gate 4096 x 28672 bfloat16 with
// squared ReLU 91 us = 6.4 TB/s; with SiLU 115.5 us, GELU 127 (two MUFU instructions an element, and an SM has room for one row, so its
// phases do not overlap); norm with residual 4096 x 8192 bfloat16 41.4 us = 5.7 TB/s, float32 70.5 us = 6.2 TB/s; 4096 x 2560
// bfloat16 15.5 us.  One row: 1.8 us (2560), 2.2 us (6912 gate with the norm, a
// cluster of eight), 2.3 us (28672), the launch and two trips through the reduction.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>
#include "epilogue.cuh"
#include "ptx_sm100.cuh"

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
// The V elements as fp32; a bfloat16 is the upper half of its float: one instruction each.
template <typename T, int V>
__device__ __forceinline__ void row_unpack(const RowRaw<T, V>& x, float (&v)[V]) {
    if constexpr (V == 8 && std::is_same_v<T, __nv_bfloat16>) {
        const uint32_t w[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else if constexpr (V == 8) {
        const uint32_t w[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_float<T>(x.t[i]);
    }
}
// ... and back, rounded to T.
template <typename T, int V>
__device__ __forceinline__ void row_pack(RowRaw<T, V>& x, const float (&v)[V]) {
    if constexpr (V == 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>)
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
            else
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
        }
        x.u = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x.t[i] = from_float<T>(v[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void row_load_weight(const void* w, int w_is_f32, int k, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = w_is_f32 ? static_cast<const float*>(w)[k] : to_float<T>(static_cast<const T*>(w)[k]);
    } else {
        if (w_is_f32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + k);
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const float4 f = p[i];
                v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
            }
        } else {
            RowRaw<T, V> x;
            x.u = *reinterpret_cast<const uint4*>(static_cast<const T*>(w) + k);
            row_unpack<T, V>(x, v);
        }
    }
}
// 16 bytes at any element's address: the two aligned pieces that hold them (requested first, put together by shift16() when
// they have arrived), or, where a piece reaches beyond [lo, hi), element by element with zeros outside; nothing outside is read.
struct Piece16 {
    uint4 a, b;
    bool whole;
};
template <typename E, bool kAligned>
__device__ __forceinline__ Piece16 load16(const char* at, const char* lo, const char* hi) {
    Piece16 r;
    const char* a = kAligned ? at : at - (reinterpret_cast<uintptr_t>(at) & 15);
    r.whole = a >= lo && a + (kAligned ? 16 : 32) <= hi;
    if (r.whole) {
        r.a = *reinterpret_cast<const uint4*>(a);
        r.b = kAligned ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(a + 16);
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; i += static_cast<int>(sizeof(E))) {
            if (at + i < lo || at + i >= hi) continue;
            if constexpr (sizeof(E) == 4) w[i / 4] = *reinterpret_cast<const uint32_t*>(at + i);
            else w[i / 4] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at + i)) << (8 * (i & 3));
        }
        r.a = make_uint4(w[0], w[1], w[2], w[3]);
        r.b = make_uint4(0, 0, 0, 0);
    }
    return r;
}
__device__ __forceinline__ uint4 shift16(const Piece16& p, const char* at) {
    const uint32_t off = p.whole ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at)) & 15 : 0;
    const uint32_t w[8] = {p.a.x, p.a.y, p.a.z, p.a.w, p.b.x, p.b.y, p.b.z, p.b.w};
    uint32_t v[6], z[5];
#pragma unroll
    for (int i = 0; i < 6; ++i) v[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) z[i] = off & 4 ? v[i + 1] : v[i];
    const uint32_t bits = (off & 3) * 8;
    return make_uint4(__funnelshift_r(z[0], z[1], bits), __funnelshift_r(z[1], z[2], bits), __funnelshift_r(z[2], z[3], bits),
                      __funnelshift_r(z[3], z[4], bits));
}
// The weights of columns k .. k + V - 1 where they are not a vector of their own; zeros outside the row.
template <typename T, int V>
__device__ __forceinline__ void row_load_weight_shifted(const void* w, int w_is_f32, int k, int K, float (&v)[V]) {
    const char* lo = static_cast<const char*>(w);
    if (w_is_f32) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const char* at = lo + (static_cast<long long>(k) + i) * 4;
            const uint4 u = shift16(load16<float, false>(at, lo, lo + static_cast<long long>(K) * 4), at);
            v[i] = __uint_as_float(u.x); v[i + 1] = __uint_as_float(u.y); v[i + 2] = __uint_as_float(u.z); v[i + 3] = __uint_as_float(u.w);
        }
    } else {
        RowRaw<T, V> x;
        const char* at = lo + static_cast<long long>(k) * static_cast<int>(sizeof(T));
        x.u = shift16(load16<T, false>(at, lo, lo + static_cast<long long>(K) * static_cast<int>(sizeof(T))), at);
        row_unpack<T, V>(x, v);
    }
}
// A thread's part of a row, loaded as x and y, as what is normalised and quantised (h or z); h is written on the way.  Vector
// j starts at column (threadIdx.x + j blockDim.x) V - shift; kVec: shift is 0 and every vector whole and aligned.
// `have`: how many of its VPT vectors lie inside the row; the others are zero and stay zero under every activation.
template <typename T, int MODE, int VPT, int V, bool kVec>
__device__ __forceinline__ void row_values(const RowQuantArgs& p, int row, int have, int shift, RowRaw<T, V> (&x)[VPT],
                                           const RowRaw<T, V> (&y)[VPT], float (&t)[VPT][V]) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) row_unpack<T, V>(x[j], t[j]);
    if constexpr (MODE == kRowGate) activate<std::is_same_v<T, float>>(p.act, reinterpret_cast<float (&)[VPT * V]>(t));       // one choice for all of them
    if constexpr (MODE != kRowNorm) {
        T* h = MODE == kRowNormResidual ? static_cast<T*>(p.h) + static_cast<long long>(row) * p.ldh + static_cast<int>(threadIdx.x * V) - shift : nullptr;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float o[V];
            row_unpack<T, V>(y[j], o);
            if constexpr (MODE == kRowNormResidual) {
#pragma unroll
                for (int i = 0; i < V; ++i) t[j][i] = __fadd_rn(t[j][i], o[i]);
                row_pack<T, V>(x[j], t[j]);
                row_unpack<T, V>(x[j], t[j]);
                if constexpr (kVec) {
                    if (j < have) x[j].store(h + j * blockDim.x * V);
                } else {
                    const int k = static_cast<int>((threadIdx.x + j * blockDim.x) * V) - shift;
                    T* at = h + j * blockDim.x * V;
                    if (k >= 0 && k + V <= p.K && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
                        x[j].store(at);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            if (k + i >= 0 && k + i < p.K) at[i] = x[j].t[i];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) t[j][i] = __fmul_rn(t[j][i], o[i]);
            }
        }
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

// The same over the CTAs of a cluster, at most 64 warps in all: a warp's result goes into its slot in every CTA, and each adds
// up the same slots in the same order.  The caller has arrived at the cluster's barrier once, so that nobody is written to
// before it runs; behind the second round nobody touches a peer again.
constexpr int kWideSlots = 64;
__device__ __forceinline__ void row_reduce_cluster(uint32_t& top, float& sum, uint2* slots, uint32_t rank, uint32_t ctas) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, n = warps * static_cast<int>(ctas);
    top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    cluster_wait();
    if (lane < static_cast<int>(ctas))
        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(dsmem_map(smem_u32(&slots[rank * warps + warp]), lane)), "r"(top),
                     "r"(__float_as_uint(sum)) : "memory");
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const uint2 a = lane < n ? slots[lane] : make_uint2(0, 0), b = lane + 32 < n ? slots[lane + 32] : make_uint2(0, 0);
    top = __reduce_max_sync(0xffffffffu, max(a.x, b.x));
    sum = __uint_as_float(a.y) + __uint_as_float(b.y);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
}

// What the statistics of a row say about its codes: q = rint((t * lift) * inv), all zero where keep is 0.
struct RowScale {
    float lift, inv;
    uint32_t keep;
};
__device__ __forceinline__ RowScale row_scale_of(uint32_t top, float sum, const RowQuantArgs& p) {
    RowScale r{1.0f, 0.0f, 0xffffffffu};
    const float m = __uint_as_float(top);
    if (top >= 0x7f800000u || (p.eps >= 0.0f && !(sum < __uint_as_float(0x7f800000u)))) {
        r.keep = 0;
    } else if (m > 0.0f) {
        if (m < 1e-30f) r.lift = 1.2676506e30f;        // 2^100
        r.inv = __fdiv_rn(127.0f, __fmul_rn(m, r.lift));
    }
    return r;
}
// The row's scale: three divisions and a root, a hundred instructions, for one thread of the CTA only.
__device__ __forceinline__ void row_store_scale(const RowQuantArgs& p, int row, uint32_t top, float sum, const RowScale& r) {
    float scale = 1.0f;
    if (!r.keep) {
        scale = __uint_as_float(0x7fc00000u);
    } else if (top) {
        scale = __fdiv_rn(__fmul_rn(__uint_as_float(top), r.lift), 127.0f);
        if (p.eps >= 0.0f) scale = __fmul_rn(scale, __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.K)), p.eps))));
        if (r.lift != 1.0f) scale = __fmul_rn(scale, 7.8886091e-31f);      // 2^-100: the one rounding to a subnormal
    }
    p.row_scale[row] = scale;
}

// One row (or a CTA's part of it), held in registers as t: statistics, scale, codes.  reduce(top, sum): as row_reduce().
template <typename T, int VPT, int V, bool kVec, typename Reduce>
__device__ __forceinline__ void row_finish(const RowQuantArgs& p, int row, int have, int shift, float (&t)[VPT][V], bool store_scale,
                                           const Reduce& reduce) {
    const int w_is_f32 = p.w_dtype == kDtypeF32;
    float top_f = 0.0f, sum = 0.0f;
    if (p.eps >= 0.0f) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) sum = fmaf(t[j][i], t[j][i], sum);
    }
    if (p.w) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if (j >= have) continue;
            float w[V];
            if constexpr (kVec) row_load_weight<T, V>(p.w, w_is_f32, static_cast<int>((threadIdx.x + j * blockDim.x) * V) - shift, w);
            else row_load_weight_shifted<T, V>(p.w, w_is_f32, static_cast<int>((threadIdx.x + j * blockDim.x) * V) - shift, p.K, w);
#pragma unroll
            for (int i = 0; i < V; ++i) t[j][i] = __fmul_rn(t[j][i], w[i]);
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) top_f = max_nan(top_f, fabsf(t[j][i]));
    uint32_t top = __float_as_uint(top_f);
    reduce(top, sum);
    const RowScale r = row_scale_of(top, sum, p);
    if (threadIdx.x == 0 && store_scale) row_store_scale(p, row, top, sum, r);
    int8_t* q = p.q + static_cast<long long>(row) * p.K + static_cast<int>(threadIdx.x * V) - shift;
    if (r.lift != 1.0f) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) t[j][i] *= r.lift;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        if (j >= have) continue;
        int8_t* at = q + j * blockDim.x * V;
        if constexpr (V == 1) {
            *at = static_cast<int8_t>(row_code(t[j][0], r.inv) & r.keep);
        } else {
            uint32_t c[V / 4];
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                c[i] = pack_codes(row_code(t[j][4 * i], r.inv), row_code(t[j][4 * i + 1], r.inv),
                                  row_code(t[j][4 * i + 2], r.inv), row_code(t[j][4 * i + 3], r.inv)) & r.keep;
            if constexpr (!kVec) {
                const int k = static_cast<int>((threadIdx.x + j * blockDim.x) * V) - shift;
                if (k < 0 || k + V > p.K) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (k + i >= 0 && k + i < p.K) at[i] = static_cast<int8_t>(c[i / 4] >> (8 * (i & 3)));
                    continue;
                }
            }
            if constexpr (V == 8) *reinterpret_cast<uint2*>(at) = make_uint2(c[0], c[1]);
            else *reinterpret_cast<uint32_t*>(at) = c[0];
        }
    }
}
// Of `items` vectors those that fall to this thread: threadIdx.x, threadIdx.x + blockDim.x, ...
__device__ __forceinline__ int row_have(int items) {
    const int left = items - static_cast<int>(threadIdx.x);
    return left <= 0 ? 0 : (left + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
}

// One row per CTA.  Of a row's operands and codes: all on vector boundaries; all equally far off one; anything else.
// kRowElements takes the last kind too, a row as single elements instead of vectors.
constexpr int kRowAligned = 0, kRowSamePhase = 1, kRowAnyPhase = 2, kRowElements = 3;
template <typename T, int MODE, int VPT, int kForm>
__global__ void __launch_bounds__(1024)
row_quant_kernel(const __grid_constant__ RowQuantArgs p) {
    constexpr int V = kForm == kRowElements ? 1 : kRowVec<T>;
    constexpr bool kVec = kForm == kRowAligned || kForm == kRowElements, kSame = kForm == kRowSamePhase;
    __shared__ uint2 slots[2][32];
    const int row = blockIdx.x;
    int shift = 0;
    if constexpr (!kVec) shift = static_cast<int>((reinterpret_cast<uintptr_t>(p.q) + static_cast<uintptr_t>(row) * p.K) & (V - 1));
    const int have = row_have(kVec ? p.K / V : (shift + p.K + V - 1) / V);
    dependent_wait();
    float t[VPT][V];
    // all of the row's loads first: a store of h between them would hold the next ones back (h may be x or y)
    RowRaw<T, V> x[VPT], y[VPT];
    const T* px = static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx;
    const T* py = MODE == kRowNorm ? nullptr : static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy;
    if constexpr (kVec) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            x[j].u = y[j].u = make_uint4(0, 0, 0, 0);
            if (j < have) {
                x[j].load(px + (threadIdx.x + j * blockDim.x) * V);
                if constexpr (MODE != kRowNorm) y[j].load(py + (threadIdx.x + j * blockDim.x) * V);
            }
        }
    } else {
        const char *xl = reinterpret_cast<const char*>(px), *yl = reinterpret_cast<const char*>(py);
        const long long bytes = static_cast<long long>(p.K) * static_cast<int>(sizeof(T));
        auto offset = [&](int j) {
            return (static_cast<long long>(threadIdx.x + j * blockDim.x) * V - shift) * static_cast<int>(sizeof(T));
        };
        Piece16 a[VPT], b[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            a[j].a = a[j].b = b[j].a = b[j].b = make_uint4(0, 0, 0, 0);
            a[j].whole = b[j].whole = false;
            if (j < have) {
                a[j] = load16<T, kSame>(xl + offset(j), xl, xl + bytes);
                if constexpr (MODE != kRowNorm) b[j] = load16<T, kSame>(yl + offset(j), yl, yl + bytes);
            }
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            x[j].u = kSame ? a[j].a : shift16(a[j], xl + offset(j));
            y[j].u = MODE == kRowNorm ? make_uint4(0, 0, 0, 0) : kSame ? b[j].a : shift16(b[j], yl + offset(j));
        }
    }
    row_values<T, MODE, VPT, V, kVec>(p, row, have, shift, x, y, t);
    row_finish<T, VPT, V, kVec>(p, row, have, shift, t, true, [&](uint32_t& top, float& sum) { row_reduce(top, sum, slots, 0); });
}

// A few long rows, all on vector boundaries: a row belongs to a cluster, each CTA has a part of it.
template <typename T, int MODE, int VPT>
__global__ void __launch_bounds__(256)
row_quant_wide_kernel(const __grid_constant__ RowQuantArgs p) {
    constexpr int V = kRowVec<T>;
    __shared__ uint2 slots[kWideSlots];
    const uint32_t rank = cluster_ctarank(), ctas = cluster_nctarank();
    const int row = blockIdx.x / ctas, items = p.K / V, part = (items + static_cast<int>(ctas) - 1) / static_cast<int>(ctas);
    const int first = static_cast<int>(rank) * part, have = row_have(min(part, items - first));
    cluster_arrive();
    dependent_wait();
    float t[VPT][V];
    RowRaw<T, V> x[VPT], y[VPT];
    const T* px = static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx + (first + static_cast<int>(threadIdx.x)) * V;
    const T* py = MODE == kRowNorm ? nullptr : static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy + (first + static_cast<int>(threadIdx.x)) * V;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        x[j].u = y[j].u = make_uint4(0, 0, 0, 0);
        if (j < have) {
            x[j].load(px + j * blockDim.x * V);
            if constexpr (MODE != kRowNorm) y[j].load(py + j * blockDim.x * V);
        }
    }
    row_values<T, MODE, VPT, V, true>(p, row, have, -first * V, x, y, t);
    row_finish<T, VPT, V, true>(p, row, have, -first * V, t, rank == 0,
                                [&](uint32_t& top, float& sum) { row_reduce_cluster(top, sum, slots, rank, ctas); });
}

// Many rows: persistent CTAs that have the next row under way while they reduce and quantise this one.  A thread copies
// its own vectors of the next row into shared memory with cp.async and reads only what it copied itself, so the copies
// need no barrier; its slots are free as soon as this row's values are in registers.  (Without this an SM that holds one
// row of 28672 in its registers has no load in flight from the reduction to the last store.)
template <typename T, int MODE, int VPT>
__global__ void __launch_bounds__(VPT == 2 ? 512 : 1024, VPT == 2 ? 3 : 1)
row_quant_stream_kernel(const __grid_constant__ RowQuantArgs p) {
    constexpr int V = kRowVec<T>;
    constexpr int kIn = MODE == kRowNorm ? 1 : 2;
    extern __shared__ __align__(16) uint4 row_stage[];             // [VPT][kIn][threads]
    __shared__ uint2 slots[2][32];
    const uint32_t mine = smem_u32(row_stage) + threadIdx.x * 16, step = blockDim.x * 16;
    const int have = row_have(p.K / V);
    const size_t stride = static_cast<size_t>(blockDim.x) * 16;              // bytes between a thread's vectors
    auto fetch = [&](const char* x, const char* y, int j) {
        if (j >= have) return;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (j * kIn) * step), "l"(x + j * stride) : "memory");
        if constexpr (MODE != kRowNorm)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (j * kIn + 1) * step), "l"(y + j * stride) : "memory");
    };
    auto row_x = [&](int row) { return static_cast<const char*>(p.x) + (static_cast<size_t>(row) * p.ldx + threadIdx.x * V) * sizeof(T); };
    auto row_y = [&](int row) {
        return MODE == kRowNorm ? nullptr : static_cast<const char*>(p.y) + (static_cast<size_t>(row) * p.ldy + threadIdx.x * V) * sizeof(T);
    };
    dependent_wait();
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        fetch(row_x(blockIdx.x), row_y(blockIdx.x), j);
        if (j >= have) {             // slots that no copy writes are read as zero
            sts_v4(mine + (j * kIn) * step, make_uint4(0, 0, 0, 0));
            if constexpr (kIn == 2) sts_v4(mine + (j * kIn + 1) * step, make_uint4(0, 0, 0, 0));
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    int turn = 0;
    for (int row = blockIdx.x; row < p.M; row += gridDim.x, turn ^= 1) {
        float t[VPT][V];
        RowRaw<T, V> x[VPT], y[VPT];
        const int next = row + static_cast<int>(gridDim.x);
        const char *nx = row_x(next), *ny = row_y(next);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // Each vector's slots are requested again as soon as they have been read, before any arithmetic on this row.  A copy is
        // not ordered behind its thread's own earlier loads by itself; the warp's barrier orders what its lanes read in front
        // of it before what they do behind it, starting copies included.  (One barrier behind all vectors' loads instead: gate
        // 4096 x 28672 with SiLU 120 us, as it is 115.5; the norms the same.)
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            x[j].u = lds_v4(mine + (j * kIn) * step);
            y[j].u = kIn == 2 ? lds_v4(mine + (j * kIn + 1) * step) : make_uint4(0, 0, 0, 0);
            __syncwarp();
            if (next < p.M) fetch(nx, ny, j);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        row_values<T, MODE, VPT, V, true>(p, row, have, 0, x, y, t);
        row_finish<T, VPT, V, true>(p, row, have, 0, t, true, [&](uint32_t& top, float& sum) { row_reduce(top, sum, slots, turn); });
    }
}

// Rows that do not fit the registers of a CTA: the same arithmetic, with the row computed twice.  The second pass reads
// h back instead of adding again (it may have replaced the residual).
template <typename T, int MODE>
__device__ __forceinline__ void row_single(const RowQuantArgs& p, int row, int k, RowRaw<T, 1>& x, const RowRaw<T, 1>& y, float (&t)[1]) {
    t[0] = to_float<T>(x.t[0]);
    if constexpr (MODE == kRowNormResidual) {
        x.t[0] = from_float<T>(__fadd_rn(t[0], to_float<T>(y.t[0])));
        t[0] = to_float<T>(x.t[0]);
        x.store(static_cast<T*>(p.h) + static_cast<size_t>(row) * p.ldh + k);
    } else if constexpr (MODE == kRowGate) {
        activate<std::is_same_v<T, float>>(p.act, t);
        t[0] = __fmul_rn(t[0], to_float<T>(y.t[0]));
    }
}
template <typename T, int MODE>
__global__ void __launch_bounds__(1024)
row_quant_long_kernel(const __grid_constant__ RowQuantArgs p) {
    __shared__ uint2 slots[2][32];
    const int w_is_f32 = p.w_dtype == kDtypeF32;
    int turn = 0;
    dependent_wait();
    for (int row = blockIdx.x; row < p.M; row += gridDim.x, turn ^= 1) {
        float top_f = 0.0f, sum = 0.0f;
        for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
            RowRaw<T, 1> x, y;
            float t[1];
            x.load(static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx + k);
            if constexpr (MODE != kRowNorm) y.load(static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy + k);
            row_single<T, MODE>(p, row, k, x, y, t);
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
        if (threadIdx.x == 0) row_store_scale(p, row, top, sum, r);
        int8_t* q = p.q + static_cast<size_t>(row) * p.K;
        for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
            RowRaw<T, 1> x, y;
            float t[1];
            if constexpr (MODE == kRowNormResidual) {
                t[0] = to_float<T>(static_cast<const T*>(p.h)[static_cast<size_t>(row) * p.ldh + k]);
            } else {
                x.load(static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx + k);
                if constexpr (MODE == kRowGate) y.load(static_cast<const T*>(p.y) + static_cast<size_t>(row) * p.ldy + k);
                row_single<T, MODE>(p, row, k, x, y, t);
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
