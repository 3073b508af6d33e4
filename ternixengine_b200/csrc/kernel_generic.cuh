// Generic exact kernel: any M >= 1, K >= 1, N % 4 == 0, any row pitch, any pointer alignment.
//
// This is the path for shapes whose packed rows are not 16-byte multiples (TMA cannot describe
// them) and for K so deep that the scaled accumulators of the fast kernels could overflow.  It
// uses byte loads with predicated tails only, plain int32 multiply-adds and no scaling, so it has
// no limits beyond int32 itself (|C| <= 128*K < 2^31 for K < 2^24).
//
// CTA = 32 x 8 threads, output tile 32 rows x 128 columns, K walked in slabs of 64 through
// shared memory.  Thread (tx, ty) owns rows 4*ty..4*ty+3 and the four columns of packed byte tx.
// Problems with few output tiles (ragged decode shapes: a handful of rows, a thousand columns) are cut along K
// over blockIdx.z; the slices then add into a C that the host has zeroed (integer adds: still exact).
#pragma once
#include <cstdint>
#include "epilogue.cuh"
#include "ptx_sm100.cuh"

namespace tb200 {

constexpr int kGenRows = 32;    // rows of C per CTA
constexpr int kGenBytes = 32;   // packed bytes (x4 columns) per CTA
constexpr int kGenK = 64;       // k-slab
constexpr int kGenThreads = 256;

__global__ void __launch_bounds__(kGenThreads)
ternary_generic_kernel(const int8_t* __restrict__ A, const uint8_t* __restrict__ W, int32_t* __restrict__ C,
                       int M, int K, int N, long long ldc, int k_per_slice) {
    __shared__ __align__(16) int8_t sA[kGenRows][kGenK];
    __shared__ __align__(16) uint8_t sW[kGenK][kGenBytes];

    const int tx = threadIdx.x & 31;
    const int ty = threadIdx.x >> 5;
    const int tid = threadIdx.x;
    const int pitch = N >> 2;                         // packed bytes per k-row
    const int row0 = blockIdx.y * kGenRows;
    const int byte0 = blockIdx.x * kGenBytes;

    int32_t acc[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = 0;

    // staging assignments: 2048 bytes of each tile, 8 per thread
    const int a_row = tid >> 3, a_k = (tid & 7) * 8;
    const int w_k = tid >> 2, w_b = (tid & 3) * 8;

    // this CTA's k-range: all of K, or slice blockIdx.z of it (k_per_slice is a multiple of the slab)
    const bool sliced = gridDim.z > 1;
    const int k_begin = sliced ? static_cast<int>(blockIdx.z) * k_per_slice : 0;
    const int k_end = sliced ? min(K, k_begin + k_per_slice) : K;

    for (int k0 = k_begin; k0 < k_end; k0 += kGenK) {
        {
            const int grow = row0 + a_row;
            const int8_t* src = A + static_cast<size_t>(grow) * K + k0 + a_k;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sA[a_row][a_k + i] = (grow < M && k0 + a_k + i < k_end) ? src[i] : int8_t(0);
            const int gk = k0 + w_k;
            const uint8_t* wsrc = W + static_cast<size_t>(gk) * pitch + byte0 + w_b;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sW[w_k][w_b + i] = (gk < k_end && byte0 + w_b + i < pitch) ? wsrc[i] : uint8_t(0);
        }
        __syncthreads();

#pragma unroll 4
        for (int kk = 0; kk < kGenK; kk += 4) {
            int a4[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) a4[r] = *reinterpret_cast<const int*>(&sA[ty * 4 + r][kk]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int wb = sW[kk + q][tx];
                int w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) w[c] = (wb << (30 - 2 * c)) >> 30;   // 00->0, 01->+1, 11->-1
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int a = (a4[r] << (24 - 8 * q)) >> 24;                 // sign-extended byte q
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[r][c] += a * w[c];
                }
            }
        }
        __syncthreads();
    }

    const int col = (byte0 + tx) * 4;
    if (col < N) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + ty * 4 + r;
            if (row < M) {
                int32_t* out = C + static_cast<size_t>(row) * ldc + col;
                if (sliced) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) atomicAdd(out + c, acc[r][c]);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) out[c] = acc[r][c];
                }
            }
        }
    }
}

// The same shapes and alignments with the fused epilogue.  Byte loads as above, but a packed byte column of four
// consecutive k-rows is put into one word while it is staged, so that a field of it is one shift and mask away from a
// dp4a operand (0, +64, -64 as int8, as in the one-row kernel): 29 instructions per 64 products and thread instead of 120.
// The sums are 64 times too large and are taken down (exactly) every kGenFlush k-rows, so K stays unbounded.
// K is not cut between CTAs: a product large enough to want that is served by an aligned copy and the kernels behind it.
constexpr int kGenFlush = 131072;      // 64 * 128 * 131072 = 2^30
static_assert(kGenFlush % kGenK == 0, "flushes fall between slabs");

template <typename Epi>
__global__ void __launch_bounds__(kGenThreads)
ternary_generic_fused_kernel(const int8_t* A, const uint8_t* W, int M, int K, int N, const Epi epi) {        // no __restrict__: see epilogue.cuh
    __shared__ __align__(16) uint32_t sA[kGenRows][kGenK / 4];
    __shared__ uint32_t sW[kGenK / 4][kGenBytes];

    const int tid = threadIdx.x, tx = tid & 31, ty = tid >> 5;
    const int pitch = N >> 2;
    // tiles numbered along x only, columns fastest: the grid's y would end at 65535 row tiles
    const int tiles_x = (pitch + kGenBytes - 1) / kGenBytes;
    const int row0 = static_cast<int>(blockIdx.x) / tiles_x * kGenRows, byte0 = static_cast<int>(blockIdx.x) % tiles_x * kGenBytes;
    dependent_wait();

    int32_t acc[4][4] = {}, total[4][4] = {};
    const int a_row = tid >> 3, a_k = (tid & 7) * 8;
    int since = 0;
    for (int k0 = 0; k0 < K; k0 += kGenK) {
        {
            const int8_t* src = A + static_cast<size_t>(row0 + a_row) * K + k0 + a_k;
            uint32_t w[2] = {0, 0};
            if (row0 + a_row < M) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + a_k + i < K) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(src[i])) << (8 * (i & 3));
            }
            sA[a_row][a_k / 4] = w[0];
            sA[a_row][a_k / 4 + 1] = w[1];
#pragma unroll
            for (int g = ty; g < kGenK / 4; g += kGenThreads / 32) {
                uint32_t t = 0;
                if (byte0 + tx < pitch) {
                    const uint8_t* col = W + static_cast<size_t>(k0 + 4 * g) * pitch + byte0 + tx;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (k0 + 4 * g + i < K) t |= static_cast<uint32_t>(col[static_cast<size_t>(i) * pitch]) << (8 * i);
                }
                sW[g][tx] = t;
            }
        }
        __syncthreads();
        const int groups = row0 + ty * 4 < M ? kGenK / 4 : 0;        // a warp without rows only helps to stage
#pragma unroll 4
        for (int g = 0; g < groups; ++g) {
            const uint32_t t = sW[g][tx];
            int a4[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) a4[r] = static_cast<int>(sA[ty * 4 + r][g]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int x = static_cast<int>((t << (6 - 2 * c)) & 0xC0C0C0C0u);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r][c] = __dp4a(x, a4[r], acc[r][c]);
            }
        }
        __syncthreads();
        since += kGenK;
        if (since == kGenFlush) {
            since = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) { total[r][c] += acc[r][c] >> 6; acc[r][c] = 0; }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) total[r][c] += acc[r][c] >> 6;

    const int col = (byte0 + tx) * 4;
    if (col < N) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (row0 + ty * 4 + r < M) epi.store4(row0 + ty * 4 + r, col, total[r]);
    }
}

// Rows of `width` bytes at any address, copied to rows at a pitch (and base) of 16 bytes, which is what the TMA unit can
// describe.  A thread writes 16 bytes and reads them as aligned words; a word that is not wholly inside the source is put
// together from its bytes.  What lies between the width and the pitch is zeroed.  One launch copies both operands of a
// product: the first a.blocks CTAs the one, the others the other.
struct AlignJob {
    const uint8_t* src;      // [rows][width], no gaps
    uint8_t* dst;            // [rows][pitch]
    long long rows;
    int width, pitch, blocks;
};
__global__ void __launch_bounds__(256)
align_rows_kernel(const __grid_constant__ AlignJob a, const __grid_constant__ AlignJob b) {
    const bool first = static_cast<int>(blockIdx.x) < a.blocks;
    const AlignJob& job = first ? a : b;
    const int per_row = job.pitch / 16, width = job.width;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(job.src), hi = lo + static_cast<uintptr_t>(job.rows) * width;
    const long long total = job.rows * per_row, block = first ? blockIdx.x : blockIdx.x - a.blocks;
    dependent_wait();
    for (long long i = block * 256 + threadIdx.x; i < total; i += job.blocks * 256LL) {
        const long long r = i / per_row;
        const int x = static_cast<int>(i - r * per_row) * 16;
        const uintptr_t at = lo + static_cast<uintptr_t>(r) * width + x, word = at & ~uintptr_t(3);
        const int shift = static_cast<int>(at & 3) * 8;
        uint32_t w[5];
#pragma unroll
        for (int j = 0; j < 5; ++j) {
            const uintptr_t p = word + 4 * j;
            w[j] = 0;
            if (x + 4 * j - shift / 8 >= width) continue;
            if (p >= lo && p + 4 <= hi) {
                w[j] = *reinterpret_cast<const uint32_t*>(p);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (p + c >= lo && p + c < hi) w[j] |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t*>(p + c)) << (8 * c);
            }
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = __funnelshift_r(w[j], w[j + 1], shift);
            const int left = width - x - 4 * j;             // bytes of this word that belong to the row
            if (left < 4) o[j] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        }
        *reinterpret_cast<uint4*>(job.dst + r * job.pitch + x) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace tb200
