// Few output tiles, fused epilogue: the paired-CTA product of kernel_gemm_tc3.cuh with K cut between the pairs of a cluster.
//
// What bounds a product of some dozens to a few hundred rows is neither memory nor the tensor cores of the whole GPU but
// the few SMs that have a tile: 256 x 6912 x 2560, say, is ten 256 x 256 tiles, ten pairs out of 74, and each works through 27
// k-blocks of 0.5 us.  So a tile belongs to a cluster of `cut` pairs (2, 4, 6 or 8 CTAs); pair p multiplies the p-th share of
// the k-blocks with the machinery of the prefill kernel (weights decoded into tensor memory as the A operand, activations
// from TMA as the B operand, cta_group::2), moves its partial sums to its own shared memory, row-major, over the
// activation ring, which is idle by then, and after a cluster barrier every CTA adds up its share of the tile's rows over
// the pairs through distributed shared memory and takes the sums through the epilogue: four columns to a lane, a row to a
// warp, coalesced residual loads and stores.  Integer sums: any order gives the same bits.  One tile per cluster, no
// persistence: there is nothing after it to overlap with.
//
// Measured on B200 (launches in a graph, weights in L2): a cluster takes 5 to 8 us from its launch to its last store and
// 0.3 us per k-block of its pairs up to 128 rows (two issuers; with one 0.5), 0.55 us at 256 rows.  256 x 6912 x 2560 onto a
// residual 10.9 us, cut 3 (cut 2 12.0; persistent 23 us; 1.9 us at the rate of the instruction, below, on all SMs); 32 x 4096 x 11008 with bias and SiLU 11 us
// (mma.sync 15 us); 64 x 2560 x 2560 6.8 us.  The 0.3 us are the tensor pipe:
// a k-block of 128 rows is 8 MMAs of 256 x 128 x 32, at 8192 products a clock and SM 64 clocks each, 0.27 us in all, and MMAs
// of 64 rows take as long (256 rows: 0.54 us; measured 0.55).  Four issuers, a deeper operand ring (6 slots) and more expander
// warps accordingly change nothing; what is left is SMs without a tile and the way in and out.
// TA: activation rows of a tile (64, 128 or 256), the pair instruction's N.
#pragma once
#include <cuda.h>
#include <cstdint>
#include "epilogue.cuh"
#include "kernel_gemm_tc3.cuh"
#include "ptx_sm100.cuh"

namespace tb200 {

constexpr int kSpTurns = 4;                                       // expander warps per lane quarter: they take the stages in turn
constexpr int kSpFirstExpandWarp = 4;                             // warps 0-3 control; the expanders also read the accumulator
constexpr int kSpWarps = kSpFirstExpandWarp + 4 * kSpTurns, kSpThreads = kSpWarps * 32;
constexpr int kSpMaxCut = 4;                                      // pairs of a cluster: 8 CTAs, the portable limit
constexpr int kSpWStages = 8, kSpTStages = 4;                     // packed-weight ring; operand ring in tensor memory
template <int TA>
struct SpGeom {
    static_assert(TA == 64 || TA == 128 || TA == 256, "activation rows of a tile");
    static constexpr int kRowsPerCta = TA / 2;
    static constexpr int kActBox = kRowsPerCta * 128;             // rows x 128 K-bytes, 128-byte swizzle
    static constexpr int kActBytes = 2 * kActBox;
    static constexpr int kStages = TA == 256 ? 4 : 8;
    // Two MMA issuers take the k-blocks in turn, each into an accumulator of its own, where two of them fit beside the operand
    // ring (256 columns): a k-block costs one thread 8 MMAs of 60-90 cycles whatever their N, a commit of 180 and a wait.
    static constexpr int kIssuers = TA <= 128 ? 2 : 1;
    static constexpr int kPartBytes = TA * 128 * 4;               // this CTA's half of the tile as int32
    static_assert(kStages * kActBytes >= kPartBytes, "the partial tile lies over the activation ring");
    // an expander warp meets every phase of the barriers it waits on
    static_assert(kStages % kSpTurns == 0 && kStages >= kSpTStages && kSpTStages % kSpTurns == 0 && kSpWStages % kSpTurns == 0, "ring sizes");
    static constexpr size_t kSmemBytes = 1024 + size_t(kStages) * kActBytes + size_t(kSpWStages) * kTc3WpBytes + 512;
    static constexpr uint32_t kIdesc = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(TA >> 3) << 17) | (uint32_t(256 >> 4) << 24);
};
static_assert(SpGeom<256>::kSmemBytes <= 227 * 1024, "shared memory: 227 KB per CTA");

template <int TA, typename Epi>
__global__ void __launch_bounds__(kSpThreads, 1)
ternary_gemm_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w, int M, int K,
                          int N, int cut, int32_t* __restrict__ status, const __grid_constant__ Epi epi) {
    using G = SpGeom<TA>;
    constexpr int S = G::kStages, TS = kSpTStages, WS = kSpWStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sAct = base;                                    // [S][2 boxes][rows][128 k], later [TA][128] int32
    uint8_t* sWp = sAct + S * G::kActBytes;                  // [WS][256 k][32]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sWp + WS * kTc3WpBytes);
    uint64_t* full = bars;                   // [S]  this CTA's activations of a stage have landed
    uint64_t* empty = full + S;              // [S]  the pair's MMAs on a stage have retired
    uint64_t* ready = empty + S;             // [TS] (leader) both CTAs' operands of a stage are in place
    uint64_t* w_full = ready + TS;           // [WS] a packed-weight stage has landed
    uint64_t* w_empty = w_full + WS;         // [WS] this CTA's four lane quarters have read it
    uint64_t* acc_full = w_empty + WS;       // all of the pair's MMAs have retired
    uint64_t* drain = acc_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t crank = cluster_ctarank();                // 2 x pair + half
    const uint32_t half = crank & 1, pair = crank >> 1, lead = crank & ~1u;
    const bool leader = half == 0;
    const uint16_t pair_mask = static_cast<uint16_t>(3u << lead);
    const int a_tiles = (M + TA - 1) / TA;
    const int tile = static_cast<int>(blockIdx.x) / (2 * cut);
    const int row0 = (tile % a_tiles) * TA, col0 = (tile / a_tiles) * kTc3TileW + static_cast<int>(half) * 128;
    const int blocks = (K + kTc3BK - 1) / kTc3BK;            // the host cuts no further than one k-block per pair
    const int kb0 = static_cast<int>(pair) * blocks / cut, kb1 = (static_cast<int>(pair) + 1) * blocks / cut;
    const uint32_t n_kb = static_cast<uint32_t>(kb1 - kb0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < TS; ++s) mbar_init(&ready[s], 2 * 4);
        for (int s = 0; s < WS; ++s) { mbar_init(&w_full[s], 1); mbar_init(&w_empty[s], 4); }
        mbar_init(acc_full, G::kIssuers);
        mbar_init(drain, G::kIssuers);
        *abort_flag = 0;
        mbar_init_fence();
    }
    auto load_act = [&](uint32_t it) {
        const uint32_t s = it % S;
        mbar_arrive_expect_tx(&full[s], G::kActBytes);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            tma_load_2d(sAct + s * G::kActBytes + j * G::kActBox, &tmap_a, (kb0 + static_cast<int>(it)) * kTc3BK + j * 128,
                        row0 + static_cast<int>(half) * G::kRowsPerCta, &full[s]);
    };
    auto load_weights = [&](uint32_t it) {
        const uint32_t sw = it % WS;
        mbar_arrive_expect_tx(&w_full[sw], kTc3WpBytes);
        tma_load_2d(sWp + sw * kTc3WpBytes, &tmap_w, col0 / 4, (kb0 + static_cast<int>(it)) * kTc3BK, &w_full[sw]);
    };
    if (warp == 1) {
        tmem_alloc_pair<512>(tmem_slot);
        tmem_relinquish_pair();
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    // The CTAs of the cluster meet here, but nobody waits for the others yet: loads and expansion touch this CTA only.  The
    // first thing that needs a peer is the arrival on the leader's `ready` barrier.
    cluster_arrive();
    dependent_wait();

    if (warp == 0) {
        // ================================================================ activations
        if (lane == 0) {
            uint32_t it = 0;
            for (; it < n_kb; ++it) {
                if (!mbar_wait_backoff(&empty[it % S], ((it / S) & 1) ^ 1, abort_flag, 32)) break;
                load_act(it);
            }
            if (*abort_flag) {
                const uint32_t first = it > static_cast<uint32_t>(S) ? it - S : 0;
                for (uint32_t j = first; j < it; ++j) mbar_drain(&full[j % S], (j / S) & 1);
            }
        }
        __syncwarp();
        cluster_wait();
    } else if (warp == 1 || warp == 3) {
        // ================================================================ MMA issuers (leader CTA of the pair)
        const uint32_t who = warp >> 1;                       // warps 1 and 3
        cluster_wait();
        if (leader && lane == 0 && who < static_cast<uint32_t>(G::kIssuers)) {
            bool ok = true;
            const uint32_t acc = tmem_base + who * TA;
            for (uint32_t it = who; it < n_kb; it += G::kIssuers) {
                const uint32_t s = it % S, ts = it % TS;
                if (!mbar_wait(&ready[ts], (it / TS) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t act_addr = smem_u32(sAct + s * G::kActBytes);
                const uint32_t a_col = tmem_base + kTc3ARingCol + ts * kTc3AStageCols;
#pragma unroll
                for (int g = 0; g < kTc3BK / 32; ++g) {
                    const uint64_t db = umma_desc_sw128(act_addr + (g >> 2) * G::kActBox + (g & 3) * 32, 16, 1024);
                    tc_mma_i8_pair_tmem_a(acc, a_col + 8 * g, db, G::kIdesc, (it != who || g != 0) ? 1u : 0u);
                }
                tc_commit_pair_both(&empty[s], pair_mask);
            }
            if (ok) tc_commit_pair_both(acc_full, pair_mask);
            tc_commit_pair(drain);
            mbar_wait(drain, 0, abort_flag);
        }
    } else if (warp == 2) {
        // ================================================================ packed weights
        if (lane == 0) {
            uint32_t it = 0;
            for (; it < n_kb; ++it) {
                if (!mbar_wait_backoff(&w_empty[it % WS], ((it / WS) & 1) ^ 1, abort_flag, 32)) break;
                load_weights(it);
            }
            if (*abort_flag) {
                const uint32_t first = it > static_cast<uint32_t>(WS) ? it - WS : 0;
                for (uint32_t j = first; j < it; ++j) mbar_drain(&w_full[j % WS], (j / WS) & 1);
            }
        }
        __syncwarp();
        cluster_wait();
    } else if (warp >= kSpFirstExpandWarp) {
        // ================================================================ expanders, as in kernel_gemm_tc3.cuh
        const uint32_t q = warp & 3;
        const uint32_t slot = (warp - kSpFirstExpandWarp) >> 2;
        const uint32_t r_in = lane & 15;
        const uint32_t ld_off = (lane >> 4) * 512 + r_in * 32 + (((q >> 1) ^ ((r_in >> 2) & 1)) << 4);
        const bool odd = (q & 1) != 0;
        const uint32_t wp_sa = smem_u32(sWp);
        const uint32_t t_lane = (q * 32) << 16;
        bool met = false;
        for (uint32_t it = slot; it < n_kb; it += kSpTurns) {
            const uint32_t s = it % S, ts = it % TS, sw = it % WS;
            if (!mbar_wait_backoff(&w_full[sw], (it / WS) & 1, abort_flag, 32)) break;
            const uint32_t wp = wp_sa + sw * kTc3WpBytes + ld_off;
            uint32_t X[kTc3BK / 32], Y[kTc3BK / 32];
#pragma unroll
            for (int g = 0; g < kTc3BK / 32; ++g) {
                uint32_t m[4];
                ldmatrix_x2_trans_b8_nc(m, wp + g * 1024);
                X[g] = odd ? m[1] : m[0];
                Y[g] = odd ? m[3] : m[2];
            }
            // the operand slot is free once the MMAs of stage it - TS have retired (the barrier of that stage's activation slot)
            if (it >= static_cast<uint32_t>(TS)) {
                const uint32_t j = it - TS;
                if (!mbar_wait_backoff(&empty[j % S], (j / S) & 1, abort_flag, 32)) break;
            }
            tc_fence_after_sync();
            const uint32_t a_col = tmem_base + kTc3ARingCol + ts * kTc3AStageCols + t_lane;
#pragma unroll
            for (int g = 0; g < kTc3BK / 32; ++g) {
                tmem_st_16x128_x2(a_col + 8 * g, decode_field_x64<0>(X[g]), decode_field_x64<1>(X[g]), decode_field_x64<0>(Y[g]),
                                  decode_field_x64<1>(Y[g]));
                tmem_st_16x128_x2(a_col + (16u << 16) + 8 * g, decode_field_x64<2>(X[g]), decode_field_x64<3>(X[g]),
                                  decode_field_x64<2>(Y[g]), decode_field_x64<3>(Y[g]));
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&w_empty[sw]);
            tmem_st_wait();
            tc_fence_before_sync();
            if (q == 0 && !mbar_wait_backoff(&full[s], (it / S) & 1, abort_flag, 32)) break;
            if (!met) cluster_wait();
            met = true;
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(&ready[ts]);
                else mbar_arrive_remote(&ready[ts], lead);
            }
        }
        if (!met) cluster_wait();
        // ================================================================ partial sums: tensor memory -> shared memory
        // The tile's residual comes into L2 meanwhile: the rows this CTA will finish, one per thread.
        const int share = (TA + cut - 1) / cut, first = row0 + static_cast<int>(pair) * share;
        const int mine = static_cast<int>(threadIdx.x) - kSpFirstExpandWarp * 32;
        if (epi.residual && mine < share && first + mine < min(M, row0 + TA) && col0 < N) epi.prefetch_residual(first + mine, col0, min(128, N - col0));
        __syncwarp();
        const uint32_t colp = q * 32 + 4 * (lane & 7) + (lane >> 3);       // the column numbering above
        const uint32_t part = smem_u32(sAct);
        if (mbar_wait_backoff(acc_full, 0, abort_flag, 64)) {
            tc_fence_after_sync();
            __syncwarp();
#pragma unroll 1
            for (int c = static_cast<int>(slot); c < TA / 32; c += kSpTurns) {
                uint32_t r[32];
                tmem_ld_32x32(tmem_base + ((q * 32) << 16) + 32 * c, r);
                tmem_ld_wait();
                if (G::kIssuers > 1 && n_kb > 1) {            // an issuer without a k-block left its accumulator untouched
                    uint32_t r1[32];
                    tmem_ld_32x32(tmem_base + ((q * 32) << 16) + TA + 32 * c, r1);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] += r1[j];
                }
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    sts_u32(part + (((32 * c + j) * 128 + colp) << 2), static_cast<uint32_t>(static_cast<int32_t>(r[j]) >> 6));
            }
            tc_fence_before_sync();
        }
    }
    __syncwarp();                      // the roles above part the lanes of their warps
    if (*abort_flag && lane == 0 && status) atomicMax(status, kStatusTimeout);
    __syncwarp();
    cluster_sync_all();                // every pair's partial tile is in place

    // ---- the pair's share of the tile's rows, this CTA's 128 columns: sums over the pairs, epilogue
    {
        const int per_pair = (TA + cut - 1) / cut, first = static_cast<int>(pair) * per_pair, share = min(per_pair, TA - first);
        const int col = col0 + 4 * lane;
        const uint32_t part = smem_u32(sAct) + 16 * lane;
        float cs[4], b[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            cs[x] = col < N ? epi.column_scale(col + x) : 0.0f;
            b[x] = col < N ? epi.column_bias(col + x) : 0.0f;
        }
        for (int j0 = warp; j0 < share; j0 += 2 * kSpWarps) {           // two rows of a warp at a time
            float v[8];
            typename Epi::Raw raw[2];
            int row[2];
            float rs[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = j0 + u * kSpWarps;
                row[u] = j < share ? row0 + first + j : M;
                raw[u] = typename Epi::Raw{};
                rs[u] = 0.0f;
                if (row[u] < M && col < N) {
                    raw[u] = epi.load_residual4(row[u], col);
                    rs[u] = epi.row_scale[row[u]];
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                int32_t sum[4] = {0, 0, 0, 0};
                if (row[u] < M) {
                    const uint32_t at = part + (first + j0 + u * kSpWarps) * 512;
                    int4 x[kSpMaxCut];           // all loads before any is used
#pragma unroll
                    for (int p = 0; p < kSpMaxCut; ++p) {
                        x[p] = make_int4(0, 0, 0, 0);
                        if (p < cut)
                            asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(x[p].x), "=r"(x[p].y), "=r"(x[p].z), "=r"(x[p].w)
                                         : "r"(dsmem_map(at, 2 * p + half)));
                    }
#pragma unroll
                    for (int p = 0; p < kSpMaxCut; ++p) {
                        sum[0] += x[p].x; sum[1] += x[p].y; sum[2] += x[p].z; sum[3] += x[p].w;
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) v[4 * u + x] = epi.linear(sum[x], rs[u], cs[x], b[x]);
            }
            epi.activate(v);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (row[u] < M && col < N) epi.finish4(row[u], col, v + 4 * u, raw[u]);
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    cluster_sync_threads();            // nobody leaves, or frees tensor memory, while a peer may still read or signal it
    __syncwarp();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair<512>(tmem_base);
    }
}

}  // namespace tb200
