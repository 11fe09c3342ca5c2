// linear.cu - K9: matrix product with its epilogue on the tensor cores (TMA +
// tcgen05, TMEM accumulators, sm_100a), bf16 or e4m3 operands.
//
//   v = (sum_k x[m][k] W[n][k]) sx[m] sw[n] + bias[n]
//   u = (sum_k x[m][k] G[n][k]) sx[m] sg[n] + gate_bias[n]        (gated)
//   y[m][n] = bf16_rn((gated ? act(u) v : act(v)) + residual[m][n])
//
// sums and everything after them in fp32, one rounding. The projections of the
// reference's forward_layer (engine/pipeline.py:364-373, 403-405, 407-447:
// torch.matmul, + bias, silu(gate) * up, h + ...). Semantics: include/a11spec.h
// (a11s_linear).
//
// Three kernels, chosen in launch_linear by a cost model of their tiles:
//   linear_skinny (linear_skinny.cu)  up to 32 rows: HBM-bound weight streaming
//   linear_tile   128 rows x 32, 64 or 128 weight rows a CTA, K split over the CTAs
//                 of a cluster (1 to 8): sizes whose tiles alone would leave most
//                 SMs idle. The partial sums meet in distributed shared memory,
//                 added in rank order.
//   linear_pair   persistent CTA pairs (cta_group::2), 256 x 256 tiles: sizes
//                 that fill the GPU. Tensor-bound; structure as in lm_head.cu.
// Measured (one B200): 2048 x 8192 -> 2048 with a residual 60 us = 1.14 PFLOP/s (64 tiles on
// 74 pairs), 8192 x 2048 -> 8192 gated e4m3 237 to 242 us = 2.3 PFLOP/s (2.15 GB of operands
// from L2 into the SMs, 9 TB/s; 10.6 in a cold launch of 203 us), 197 x 1000 -> 1531 9.4 us,
// 64 x 8192 -> 2048 bf16 13.0 us, e4m3 9.6.
// A gated product takes gate and weight rows side by side in one tile (half the
// columns each), so x is staged once for both and act(u) v is formed from two
// column ranges of one accumulator: the 2 N intermediate is never written.
// Operand tiles are 128 bytes of K per row (64 bf16, 128 e4m3), 128-byte
// swizzle: the types differ in the instruction and the tensor maps only.
// Every mbarrier wait is bounded; a timeout sets ETIMEOUT, and the CTA drains
// its copies and MMAs and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "epilogue.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace a11s {

namespace {
constexpr int kThreads = 192;                    // TMA warp, MMA warp, 4 epilogue warps
constexpr int kSliceBytes = 128;                 // bytes of K per row and slice
constexpr long long kWaitBudget = 2000000000ll;  // ~1 s of SM clock

struct LinParams {
    const float *x_scale;
    ColumnParams col;
    const __nv_bfloat16 *residual;
    __nv_bfloat16 *out;
    int64_t res_stride, out_stride;
    int32_t rows, N, act, m_tiles, n_tiles, slices, split;
    int32_t vec4;              // linear_tile: out and residual rows take 8-byte accesses, N a multiple of 4
    int32_t tma_out, vec_res;  // linear_pair: out takes a tensor map; residual rows are read 16 bytes at a time
    StatusWord *status;
};

struct BarsCommon {
    int32_t abort;
    uint32_t tmem_base;
};
__device__ __forceinline__ bool aborted(BarsCommon *bs) { return *reinterpret_cast<volatile int32_t *>(&bs->abort) != 0; }
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, BarsCommon *bs, StatusWord *st) {
    if (tc::mbar_wait(bar, parity, kWaitBudget)) return true;
    *reinterpret_cast<volatile int32_t *>(&bs->abort) = 1;
    report(st, A11S_ETIMEOUT, (int32_t)blockIdx.x);
    return false;
}
// The same by a whole warp, with one answer for all its lanes (a converged warp stays one).
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, BarsCommon *bs, StatusWord *st) {
    return __all_sync(0xffffffffu, wait_or_abort(bar, parity, bs, st));
}
__device__ __forceinline__ bool warp_aborted(BarsCommon *bs) { return __any_sync(0xffffffffu, aborted(bs)); }
// The status word is cleared by the launch's first thread: a report can only
// follow a wait of about a second, long after every CTA of the launch started.
__device__ __forceinline__ void clear_status(StatusWord *st) {
    if (st && blockIdx.x == 0 && threadIdx.x == 0) *st = StatusWord{0, 0};
}
}  // namespace

// ---------------------------------------------------------------------------- linear_tile
namespace {
constexpr int kTileM = 128;
constexpr uint32_t kTileABytes = kTileM * kSliceBytes;  // 16 KB
template <int BN>
struct TileShape {
    static constexpr uint32_t kStage = kTileABytes + BN * kSliceBytes;
    static constexpr int kStages = BN == 128 ? 6 : 8;
    static constexpr uint32_t kRing = kStages * kStage;  // 160 to 192 KB
    static constexpr uint32_t kOffCols = kRing;       // 4 x 128 column parameters, 128 row scales
    static constexpr uint32_t kOffBars = kRing + 2560;
    static constexpr uint32_t kSmem = kOffBars + 512 + 1024;
};
struct TileBars : BarsCommon {
    uint64_t full[8], empty[8], acc_full, drain;
};
static_assert(sizeof(TileBars) <= 512, "barrier block");
}  // namespace

// Barrier of the epilogue warps only.
template <int THREADS>
__device__ __forceinline__ void epilogue_barrier() {
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}
// A warp's 32 rows of 16 consecutive outputs from shared memory (rows 17 floats
// apart), two rows an access: the residual is added and the row segments written.
__device__ __forceinline__ void write_rows(const float *stage, const LinParams &p, int m0, int n0, int lane) {
    constexpr int kSteps = 16, kBatch = 8;
    const int r0 = lane >> 4, c = lane & 15;
#pragma unroll 1
    for (int i0 = 0; i0 < kSteps; i0 += kBatch) {
        // all of a batch's residual loads (absent elements: the last one again) before
        // its stores, since out may be the residual
        __nv_bfloat16 res[kBatch];
        if (p.residual) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                res[i] = p.residual[(int64_t)min(m0 + 2 * (i0 + i) + r0, p.rows - 1) * p.res_stride + min(n0 + c, p.N - 1)];
        } else {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) res[i] = __float2bfloat16_rn(0.0f);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = 2 * (i0 + i) + r0;
            const float y = stage[r * 17 + c] + __bfloat162float(res[i]);
            if (m0 + r < p.rows && n0 + c < p.N) p.out[(int64_t)(m0 + r) * p.out_stride + n0 + c] = __float2bfloat16_rn(y);
        }
    }
}

// What the 128 epilogue threads t of linear_tile do: under the wait for the
// accumulator they fetch the residual; then the sums go to shared memory
// (part, [128][BN + 4] fp32), and this CTA's share of the tile (kOut / SPLIT
// columns) is added up over the cluster's CTAs in rank order, finished and
// written. There a thread takes four columns of every kPer-th group of rows, so
// that a warp's loads from the other CTAs run along rows (whole lines: with a row
// per lane they took 2400 cycles a step of 8 columns) and its columns' parameters
// stay in registers. Reading another CTA's sums runs at some 10 bytes per cycle:
// splits that leave a CTA few columns are the cheap ones.
template <bool GATED, int BN, int SPLIT>
__device__ __forceinline__ void tile_epilogue(TileBars *bs, float *part, const float *cols_sm, const float *xs_sm, const LinParams &p,
                                              uint32_t tmem, int ns, int rank, int t, int m0, int n0, bool params) {
    constexpr int kOut = GATED ? BN / 2 : BN;
    constexpr int kCols = kOut / SPLIT, kPer = kCols / 4, kStep = kTileM / kPer;  // threads of a row, rows of a pass
    constexpr int kPitch = BN + 4;
    constexpr int kBatch = kPer < 2 ? 1 : SPLIT * (GATED ? 2 : 1) <= 8 && kPer >= 4 ? 4 : 2;  // passes in flight
    const int c = rank * kCols + t % kPer * 4, r0 = t / kPer, n = n0 + c;
    uint2 res[kBatch];  // four bf16 of each pass of the next batch; absent elements: the last ones again
    auto load_residual = [&](int i0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            res[i] = make_uint2(0, 0);
            if (!p.residual) continue;
            const __nv_bfloat16 *row = p.residual + (int64_t)min(m0 + r0 + (i0 + i) * kStep, p.rows - 1) * p.res_stride;
            if (p.vec4) {
                res[i] = *reinterpret_cast<const uint2 *>(row + min(n, p.N - 4));
            } else {
                const uint16_t *e = reinterpret_cast<const uint16_t *>(row);
                res[i].x = e[min(n, p.N - 1)] | (uint32_t)e[min(n + 1, p.N - 1)] << 16;
                res[i].y = e[min(n + 2, p.N - 1)] | (uint32_t)e[min(n + 3, p.N - 1)] << 16;
            }
        }
    };
    load_residual(0);
    const bool ok = warp_wait(&bs->acc_full, 0, bs, p.status);
    tc::tc_fence_after();
    const int row = ((threadIdx.x >> 5) & 3) * 32 + (t & 31);  // TMEM lane = tile row: warp % 4 chooses the lanes
    if (ok) {
#pragma unroll
        for (int e0 = 0; e0 < BN; e0 += 32) {
            float v[32];
            if (ns > 0) {
                tc::tmem_ld32(tmem + ((uint32_t)(row & 96) << 16) + e0, v);
            } else {  // no K slice fell to this CTA
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4 *>(part + row * kPitch + e0 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
    }
    __syncwarp();
    // every CTA's sums are in shared memory (after a timeout nobody waits for them)
    if (SPLIT == 1) epilogue_barrier<128>();
    else tc::cluster_sync();
    if (!ok) return;
    float4 ws = make_float4(1, 1, 1, 1), wb = make_float4(0, 0, 0, 0), gs = ws, gb = wb;
    if (params) {
        ws = *reinterpret_cast<const float4 *>(cols_sm + c);
        wb = *reinterpret_cast<const float4 *>(cols_sm + kOut + c);
        if constexpr (GATED) {
            gs = *reinterpret_cast<const float4 *>(cols_sm + 2 * kOut + c);
            gb = *reinterpret_cast<const float4 *>(cols_sm + 3 * kOut + c);
        }
    }
    uint32_t src[SPLIT];
#pragma unroll
    for (int r = 0; r < SPLIT; ++r) src[r] = tc::cluster_addr(part, r) + (uint32_t)(r0 * kPitch + c) * 4;
    // rolled: code that runs once costs its fetching (unrolled, 32 passes took 6 us longer)
#pragma unroll 1
    for (int i0 = 0; i0 < kPer; i0 += kBatch) {
        uint2 add[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) add[i] = res[i];
        if (i0 + kBatch < kPer) load_residual(i0 + kBatch);  // rows that this batch does not write
        float4 a[kBatch][SPLIT], g[GATED ? kBatch : 1][GATED ? SPLIT : 1];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int r = 0; r < SPLIT; ++r) {
                const uint32_t at = src[r] + (uint32_t)((i0 + i) * kStep * kPitch) * 4;
                a[i][r] = tc::ld_cluster_v4(at + (GATED ? kOut * 4 : 0));
                if constexpr (GATED) g[i][r] = tc::ld_cluster_v4(at);
            }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int rr = r0 + (i0 + i) * kStep, m = m0 + rr;
            const float xs = params ? xs_sm[rr] : 1.0f;
            float4 v = a[i][0], u = make_float4(0, 0, 0, 0);
            if constexpr (GATED) u = g[i][0];
#pragma unroll
            for (int r = 1; r < SPLIT; ++r) {
                v = make_float4(v.x + a[i][r].x, v.y + a[i][r].y, v.z + a[i][r].z, v.w + a[i][r].w);
                if constexpr (GATED) u = make_float4(u.x + g[i][r].x, u.y + g[i][r].y, u.z + g[i][r].z, u.w + g[i][r].w);
            }
            const uint2 w = add[i];
            const float y0 = finish<GATED>(v.x, u.x, xs, Column{ws.x, wb.x, gs.x, gb.x}, p.act) + bf16lo(w.x);
            const float y1 = finish<GATED>(v.y, u.y, xs, Column{ws.y, wb.y, gs.y, gb.y}, p.act) + bf16hi(w.x);
            const float y2 = finish<GATED>(v.z, u.z, xs, Column{ws.z, wb.z, gs.z, gb.z}, p.act) + bf16lo(w.y);
            const float y3 = finish<GATED>(v.w, u.w, xs, Column{ws.w, wb.w, gs.w, gb.w}, p.act) + bf16hi(w.y);
            if (m < p.rows) {
                __nv_bfloat16 *o = p.out + (int64_t)m * p.out_stride + n;
                if (p.vec4) {
                    if (n < p.N) *reinterpret_cast<uint2 *>(o) = make_uint2(tc::cvt_bf16x2(y0, y1), tc::cvt_bf16x2(y2, y3));
                } else {
                    if (n < p.N) o[0] = __float2bfloat16_rn(y0);
                    if (n + 1 < p.N) o[1] = __float2bfloat16_rn(y1);
                    if (n + 2 < p.N) o[2] = __float2bfloat16_rn(y2);
                    if (n + 3 < p.N) o[3] = __float2bfloat16_rn(y3);
                }
            }
        }
    }
}

// One 128 x BN tile (gated: 128 x BN/2 outputs) per cluster of p.split CTAs;
// each CTA multiplies its share of the K slices.
template <bool E4M3, bool GATED, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    linear_tile(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                const __grid_constant__ CUtensorMap tg, const LinParams p) {
    using S = TileShape<BN>;
    constexpr int kOut = GATED ? BN / 2 : BN;  // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    TileBars *bs = reinterpret_cast<TileBars *>(sm + S::kOffBars);
    const int warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % p.split, tile = blockIdx.x / p.split;  // clusters are consecutive CTAs
    const int m0 = (tile % p.m_tiles) * kTileM, n0 = (tile / p.m_tiles) * kOut;
    const int per = (p.slices + p.split - 1) / p.split;
    const int s0 = min(rank * per, p.slices), ns = min(per, p.slices - s0);
    let_next_start();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            tc::mbar_init(&bs->full[s], 1);
            tc::mbar_init(&bs->empty[s], 1);
        }
        tc::mbar_init(&bs->acc_full, 1);
        tc::mbar_init(&bs->drain, 1);
        bs->abort = 0;
        tc::fence_barrier_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&bs->tmem_base, BN);
        tc::tmem_relinquish();
    }
    if (warp == 0 && tc::elect_one()) {
        tc::prefetch_tmap(&tx);
        tc::prefetch_tmap(&tw);
        if (GATED) tc::prefetch_tmap(&tg);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = bs->tmem_base;
    wait_before();
    clear_status(p.status);

    if (warp == 0) {
        constexpr int kElems = E4M3 ? kSliceBytes : kSliceBytes / 2;
        for (int i = 0, s = 0, use = 0; i < ns; ++i) {
            if (use > 0 && !warp_wait(&bs->empty[s], (use - 1) & 1, bs, p.status)) break;
            if (warp_aborted(bs)) break;
            if (tc::elect_one()) {
                uint8_t *a = sm + s * S::kStage;
                const int k = (s0 + i) * kElems;
                tc::mbar_arrive_expect_tx(&bs->full[s], S::kStage);
                tc::tma_load_2d(a, &tx, &bs->full[s], k, m0);
                if constexpr (GATED) {  // gate rows, then weight rows: kOut of each
                    tc::tma_load_2d(a + kTileABytes, &tg, &bs->full[s], k, n0);
                    tc::tma_load_2d(a + kTileABytes + kOut * kSliceBytes, &tw, &bs->full[s], k, n0);
                } else {
                    tc::tma_load_2d(a + kTileABytes, &tw, &bs->full[s], k, n0);
                }
            }
            __syncwarp();
            if (++s == S::kStages) {
                s = 0;
                ++use;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t idesc = E4M3 ? tc::idesc_e4m3_f32(kTileM, BN) : tc::idesc_bf16_f32(kTileM, BN, false);
        const uint64_t ad0 = tc::sdesc_sw128(tc::smem_u32(sm), 16, 1024);  // + 16-byte units: slots, 32 bytes per MMA
        bool ok = true;
        for (int i = 0, s = 0, use = 0; i < ns; ++i) {
            if (!(ok = warp_wait(&bs->full[s], use & 1, bs, p.status))) break;
            tc::tc_fence_after();
            if (tc::elect_one()) {
                const uint64_t ad = ad0 + (uint64_t)(s * (S::kStage / 16)), bd = ad + kTileABytes / 16;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    if constexpr (E4M3) tc::mma_e4m3_ss(tmem, ad + 2 * kk, bd + 2 * kk, idesc, (i | kk) != 0);
                    else tc::mma_bf16_ss(tmem, ad + 2 * kk, bd + 2 * kk, idesc, (i | kk) != 0);
                }
                tc::mma_commit(&bs->empty[s]);
            }
            __syncwarp();
            if (++s == S::kStages) {
                s = 0;
                ++use;
            }
        }
        if (tc::elect_one()) {
            if (ok) tc::mma_commit(&bs->acc_full);
            tc::mma_commit(&bs->drain);
        }
        __syncwarp();
        tc::mbar_wait(&bs->drain, 0, kWaitBudget);
        __syncwarp();
    }
    if (warp >= 2) {
        const int t = threadIdx.x - 64;
        float *cols_sm = reinterpret_cast<float *>(sm + S::kOffCols), *xs_sm = cols_sm + 512, *part = reinterpret_cast<float *>(sm);
        const bool params = p.col.any();
        if (params) {
            stage_columns<GATED, kOut>(cols_sm, p.col, n0, p.N, t, 128);
            xs_sm[t] = E4M3 && m0 + t < p.rows ? p.x_scale[m0 + t] : 1.0f;
        }
        epilogue_barrier<128>();
        auto run = [&](auto split) {
            tile_epilogue<GATED, BN, decltype(split)::value>(bs, part, cols_sm, xs_sm, p, tmem, ns, rank, t, m0, n0, params);
        };
        if (p.split == 1) run(std::integral_constant<int, 1>{});
        else if (p.split == 2) run(std::integral_constant<int, 2>{});
        else if (p.split == 4) run(std::integral_constant<int, 4>{});
        else if constexpr (kOut >= 32) run(std::integral_constant<int, 8>{});
    } else if (p.split > 1) {
        __syncwarp();
        tc::cluster_sync();  // the epilogue warps' one
    }
    // After a timeout copies may still be landing here: give them time (about
    // 0.2 ms) before the shared memory is released.
    if (threadIdx.x == 0 && aborted(bs)) {
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {
        }
    }
    __syncwarp();
    tc::tc_fence_before();
    tc::cluster_sync();  // the others have read this CTA's sums; its TMEM loads are over
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, BN);
    }
}

// ---------------------------------------------------------------------------- linear_pair
namespace {
constexpr int kPairM = 256, kPairN = 256;  // tile of a pair; each CTA holds 128 rows of both operands
constexpr int kPairThreads = 320;                  // TMA warp, MMA warp, 8 epilogue warps
constexpr int kEpiThreads = kPairThreads - 64;
constexpr uint32_t kPairHalf = 128 * kSliceBytes;  // 16 KB
constexpr uint32_t kPairStage = 2 * kPairHalf;
constexpr int kPairStages = 6;
constexpr int kEpiCols = 32;                       // output columns per epilogue step: a box of 32 rows x 64 bytes
constexpr uint32_t kBoxPitch = 2560;               // 2 KB box (or 32 x 17 floats), on 512 bytes
constexpr uint32_t kOffBox = kPairStages * kPairStage;       // one box per epilogue warp
constexpr uint32_t kOffPairCols = kOffBox + 8 * kBoxPitch;   // column parameters of two tiles: 512 floats each
constexpr uint32_t kOffPairBars = kOffPairCols + 4096;
constexpr uint32_t kPairSmem = kOffPairBars + 512 + 1024;
constexpr uint32_t kPairTmem = 2 * kPairN;
static_assert(kPairSmem <= 232448 && 32 * 17 * 4 <= kBoxPitch, "shared memory budget");

struct PairBars : BarsCommon {
    uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2], drain;
};
static_assert(sizeof(PairBars) <= 512, "barrier block");
}  // namespace

template <bool E4M3, bool GATED>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                const __grid_constant__ CUtensorMap tg, const __grid_constant__ CUtensorMap tout, const LinParams p) {
    constexpr int kOut = GATED ? kPairN / 2 : kPairN;
    constexpr int kSteps = kOut / kEpiCols;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    PairBars *bs = reinterpret_cast<PairBars *>(sm + kOffPairBars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int unit = (int)tc::cluster_id(), units = (int)tc::cluster_count();
    const int total = p.m_tiles * p.n_tiles;
    const int my_tiles = unit < total ? (total - 1 - unit) / units + 1 : 0;
    let_next_start();
    if (my_tiles == 0) return;  // both CTAs of the pair (the launch has no more pairs than tiles)

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            tc::mbar_init(&bs->full[s], 1);
            tc::mbar_init(&bs->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&bs->acc_full[b], 1);
            tc::mbar_init(&bs->acc_empty[b], 16);  // one arrival per epilogue warp of both CTAs
        }
        tc::mbar_init(&bs->drain, 1);
        bs->abort = 0;
        tc::fence_barrier_init();
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(&bs->tmem_base, kPairTmem);
        tc::tmem_relinquish_pair();
    }
    tc::tc_fence_before();
    tc::cluster_sync();  // the even CTA's barriers are ready before the peer signals them
    tc::tc_fence_after();
    const uint32_t tmem = bs->tmem_base;
    wait_before();
    clear_status(p.status);

    if (warp == 0) {
        constexpr int kElems = E4M3 ? kSliceBytes : kSliceBytes / 2;
        // B rows of this CTA: gated, the even CTA stages the gate's rows and the odd one the weight's
        const CUtensorMap *tb = GATED && rank == 0 ? &tg : &tw;
        int s = 0, use = 0;
        bool ok = true;
        for (int i = 0; i < my_tiles && ok; ++i) {
            const int t = unit + i * units;
            const int m0 = (t % p.m_tiles) * kPairM + (int)rank * 128;
            const int nb = (t / p.m_tiles) * kOut + (GATED ? 0 : (int)rank * 128);
            for (int kb = 0; kb < p.slices; ++kb) {
                if (use > 0 && !(ok = warp_wait(&bs->empty[s], (use - 1) & 1, bs, p.status))) break;
                if (warp_aborted(bs)) {
                    ok = false;
                    break;
                }
                if (tc::elect_one()) {
                    uint8_t *a = sm + s * kPairStage;
                    const uint32_t fb = tc::cluster_addr(&bs->full[s], 0);
                    if (rank == 0) tc::mbar_arrive_expect_tx(&bs->full[s], 2 * kPairStage);
                    tc::tma_load_2d_pair(a, &tx, fb, kb * kElems, m0);
                    tc::tma_load_2d_pair(a + kPairHalf, tb, fb, kb * kElems, nb);
                }
                __syncwarp();
                if (++s == kPairStages) {
                    s = 0;
                    ++use;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc = E4M3 ? tc::idesc_e4m3_f32(kPairM, kPairN) : tc::idesc_bf16_f32(kPairM, kPairN, false);
            const uint64_t ad0 = tc::sdesc_sw128(tc::smem_u32(sm), 16, 1024);
            int s = 0, phase = 0;
            bool ok = true;
            for (int i = 0; i < my_tiles && ok; ++i) {
                const int buf = i & 1, use = i >> 1;
                if (use > 0 && !(ok = warp_wait(&bs->acc_empty[buf], (use - 1) & 1, bs, p.status))) break;
                tc::tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(buf * kPairN);
                for (int kb = 0; kb < p.slices; ++kb) {
                    if (!(ok = warp_wait(&bs->full[s], phase, bs, p.status))) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        const uint64_t ad = ad0 + (uint64_t)(s * (kPairStage / 16)), bd = ad + kPairHalf / 16;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            if constexpr (E4M3) tc::mma_e4m3_ss_pair(d, ad + 2 * kk, bd + 2 * kk, idesc, (kb | kk) != 0);
                            else tc::mma_bf16_ss_pair(d, ad + 2 * kk, bd + 2 * kk, idesc, (kb | kk) != 0);
                        }
                        tc::mma_commit_pair_both(&bs->empty[s]);
                    }
                    __syncwarp();
                    if (++s == kPairStages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                if (ok && tc::elect_one()) tc::mma_commit_pair_both(&bs->acc_full[buf]);
                __syncwarp();
            }
            if (tc::elect_one()) tc::mma_commit_pair(&bs->drain);
            __syncwarp();
            tc::mbar_wait(&bs->drain, 0, kWaitBudget);
        }
        __syncwarp();
    } else {
        // epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31 and takes every other
        // step (w / 4) of 32 output columns. The outputs leave through a box of its
        // own (64 bytes a row, 64-byte swizzle) by TMA stores.
        const int q = warp & 3, first = (warp - 2) >> 2;
        const uint32_t lane_base = (uint32_t)(q * 32) << 16;
        uint8_t *box = sm + kOffBox + (warp - 2) * kBoxPitch;
        const uint32_t srow = tc::smem_u32(box) + (uint32_t)lane * 64u;
        const bool params = p.col.any();
        bool ok = true;
        for (int i = 0; i < my_tiles; ++i) {  // to the end also after a timeout: the warps meet at a barrier
            const int t = unit + i * units;
            const int mw = (t % p.m_tiles) * kPairM + (int)rank * 128 + q * 32, n0 = (t / p.m_tiles) * kOut;
            const int buf = i & 1, m = mw + lane;
            float *cols = reinterpret_cast<float *>(sm + kOffPairCols) + buf * 512;
            float xs = 1.0f;
            // under the wait for the accumulator: the tile's column parameters (the
            // buffer's readers, two tiles back, passed the barrier of the tile between)
            if (params) {
                stage_columns<GATED, kOut>(cols, p.col, n0, p.N, threadIdx.x - 64, kEpiThreads);
                epilogue_barrier<kEpiThreads>();
            }
            if (!ok) continue;
            if (E4M3 && m < p.rows) xs = p.x_scale[m];
            uint4 res[4];
            auto load_residual = [&](int n) {  // this row's 32 columns at n; absent ones are never stored
                const bool in = m < p.rows;
                const uint4 *src = reinterpret_cast<const uint4 *>(p.residual + (int64_t)m * p.res_stride + n);
#pragma unroll
                for (int c = 0; c < 4; ++c) res[c] = in && n + 8 * c < p.N ? __ldcs(src + c) : make_uint4(0, 0, 0, 0);
            };
            if (p.vec_res) load_residual(n0 + first * kEpiCols);
            ok = warp_wait(&bs->acc_full[buf], (i >> 1) & 1, bs, p.status);
            if (!ok) continue;
            tc::tc_fence_after();
#pragma unroll 1
            for (int h = first; h < kSteps; h += 2) {
                const int n = n0 + h * kEpiCols;
                float v[32], u[GATED ? 32 : 1];
                if constexpr (GATED) tc::tmem_ld32(tmem + lane_base + (uint32_t)(buf * kPairN + h * kEpiCols), u);
                tc::tmem_ld32(tmem + lane_base + (uint32_t)(buf * kPairN + (GATED ? kOut : 0) + h * kEpiCols), v);
                if (h + 2 >= kSteps) {  // the accumulator is in registers: the next tile may use it
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive_cluster(tc::cluster_addr(&bs->acc_empty[buf], 0));
                }
                finish_columns<GATED, kOut>(v, u, xs, cols, h * kEpiCols, params, p.act);
                if (p.tma_out) {
                    if (p.vec_res) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t w[4] = {res[c].x, res[c].y, res[c].z, res[c].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                v[8 * c + 2 * e] += bf16lo(w[e]);
                                v[8 * c + 2 * e + 1] += bf16hi(w[e]);
                            }
                        }
                        if (h + 2 < kSteps) load_residual(n + 2 * kEpiCols);
                    }
                    if (lane == 0) tc::bulk_wait_read_all();  // the box's last store
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = tc::cvt_bf16x2(v[8 * c + 2 * e], v[8 * c + 2 * e + 1]);
                        tc::st_shared_v4(srow + (((uint32_t)c ^ (uint32_t)((lane >> 1) & 3)) << 4), w);
                    }
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {  // clipped at the last column and row
                        tc::tma_store_2d(&tout, box, n, mw);
                        tc::bulk_commit_group();
                    }
                } else {  // rows that no tensor map can describe (odd pitch or width)
                    float *st = reinterpret_cast<float *>(box);
#pragma unroll
                    for (int e0 = 0; e0 < 32; e0 += 16) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) st[lane * 17 + e] = v[e0 + e];
                        __syncwarp();
                        write_rows(st, p, mw, n + e0, lane);
                        __syncwarp();
                    }
                }
            }
        }
        if (lane == 0) tc::bulk_wait_all();
        __syncwarp();
    }
    if (threadIdx.x == 0 && aborted(bs)) {  // as in linear_tile
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {
        }
    }
    __syncwarp();
    tc::tc_fence_before();
    tc::cluster_sync();  // the pair's MMAs and remote arrivals are over
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc_pair(tmem, kPairTmem);
    }
}

// ---------------------------------------------------------------------------- host side
namespace {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// 2-D row-major [outer][inner] of bf16 or bytes, pitch in elements; boxes of 128 (or 64) bytes x box_rows, swizzled over their width.
bool encode(CUtensorMap *map, bool bytes, const void *base, int64_t inner, int64_t outer, int64_t pitch, uint32_t box_rows,
            int box_bytes = 128) {
    auto fn = encode_fn();
    if (!fn) return false;
    const int es = bytes ? 1 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    // with one row the pitch is never used; it must still be a valid one
    const cuuint64_t str[1] = {(cuuint64_t)pitch * es};
    const cuuint32_t box[2] = {(cuuint32_t)(box_bytes / es), box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base),
              dims, str, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int device_sms() {
    static std::atomic<int> n{0};
    int v = n.load();
    if (!v) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            v = 148;
        n.store(v);
    }
    return v;
}

// Clusters of `split` linear_tile CTAs that can be resident at once.
int tile_slots(int split, int sms) {
    static std::atomic<int> known[4] = {};  // splits 1, 2, 4, 8; every instantiation fills an SM with one CTA
    const int i = split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3;
    int v = known[i].load();
    if (!v) {
        auto kernel = linear_tile<false, false, 64>;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(sms / split * split));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = TileShape<64>::kSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)split;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TileShape<64>::kSmem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&v, kernel, &cfg) != cudaSuccess || v < 1)
            v = std::max(1, sms / split * (split == 8 ? 3 : 4) / 4);
        known[i].store(v);
    }
    return v;
}

// What a tiling takes, in microseconds: waves of tiles, each its K slices and
// what a tile spends besides (filling the ring, exchanging sums, the epilogue).
// Fitted to a sweep of every (BN, split) over 14 sizes of 48 to 2048 rows, K 512
// to 8192 and N 200 to 8192; the choice was the fastest there or within 6 % of it.
// Eleven of them were bf16 and three e4m3; one set of constants serves both types,
// gated or not. For instance 64 x 8192 -> 2048 with a residual: 64/4 14.2 us, 32/2 18.7, 64/1 33.6, pairs 43.9;
// 768 x 4096 -> 4096: pairs 26.3, 128/2 45.5; 197 x 1000 -> 1531: 64/2 10.0, 32/1 10.4.
struct Plan {
    int bn = kPairN, split = 1;
};
Plan choose(const LinearArgs &a, int slices, int sms) {
    const auto tiles = [&](int m, int n) { return (long long)((a.rows + m - 1) / m) * ((a.N + n - 1) / n); };
    Plan best;
    const long long pairs = tiles(kPairM, a.gate ? kPairN / 2 : kPairN);
    double least = (double)((pairs + sms / 2 - 1) / (sms / 2)) * slices * 0.32 + 6.0;
    for (int bn : {32, 64, 128})
        for (int split : {1, 2, 4, 8}) {
            if (split > 1 && (split > slices || (bn == 32 && a.gate && split == 8))) break;
            const double slice = bn == 32 ? 0.20 : bn == 64 ? 0.21 : 0.235;
            const double fixed = split == 1 ? 3.05 + 0.045 * bn : split == 2 ? 3.55 + 0.0266 * bn : split == 4 ? 4.1 + 0.018 * bn
                                                                                                       : 4.9 + 0.03 * bn;
            const long long t = tiles(kTileM, a.gate ? bn / 2 : bn), slots = tile_slots(split, sms);
            const double us = (double)((t + slots - 1) / slots) * ((slices + split - 1) / split * slice + fixed);
            if (us < least) {
                least = us;
                best.bn = bn;
                best.split = split;
            }
        }
    return best;
}

int k_slices(const LinearArgs &a) {
    const int elems = a.e4m3 ? kSliceBytes : kSliceBytes / 2;
    return (a.K + elems - 1) / elems;
}

template <bool E4M3, bool GATED, int BN>
cudaError_t launch_tile(const LinearArgs &a, LinParams p, int split, cudaStream_t s) {
    constexpr int kOut = GATED ? BN / 2 : BN;
    CUtensorMap tx, tw, tg;
    if (!encode(&tx, E4M3, a.x, a.K, a.rows, a.x_stride, kTileM)) return cudaErrorInvalidValue;
    if (!encode(&tw, E4M3, a.weight, a.K, a.N, a.K, kOut)) return cudaErrorInvalidValue;
    tg = tw;
    if (GATED && !encode(&tg, E4M3, a.gate, a.K, a.N, a.K, kOut)) return cudaErrorInvalidValue;
    p.m_tiles = (a.rows + kTileM - 1) / kTileM;
    p.n_tiles = (a.N + kOut - 1) / kOut;
    p.split = split;
    auto vec4 = [&](const void *ptr, int64_t stride) {
        return a.N % 4 == 0 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 7) == 0;
    };
    p.vec4 = vec4(a.out, a.out_stride) && (!a.residual || vec4(a.residual, a.res_stride));
    auto kernel = linear_tile<E4M3, GATED, BN>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TileShape<BN>::kSmem);
    if (e != cudaSuccess) return e;
    return launch_overlapped(kernel, dim3((unsigned)((long long)p.m_tiles * p.n_tiles * split)), kThreads, TileShape<BN>::kSmem,
                             (unsigned)split, s, tx, tw, tg, p);
}

// CTA pairs that can be resident at once (one CTA per SM; an odd SM of a group stays out).
template <typename K>
int pair_slots(K kernel, const cudaLaunchConfig_t &cfg, int sms) {
    static std::atomic<int> n{0};  // the same for every instantiation of the kernel: one CTA per SM by shared memory
    int v = n.load();
    if (!v) {
        if (cudaOccupancyMaxActiveClusters(&v, kernel, &cfg) != cudaSuccess || v < 1) v = sms / 2;
        n.store(v);
    }
    return v;
}

template <bool E4M3, bool GATED>
cudaError_t launch_pair(const LinearArgs &a, LinParams p, int sms, cudaStream_t s) {
    constexpr int kOut = GATED ? kPairN / 2 : kPairN;
    CUtensorMap tx, tw, tg, tout;
    if (!encode(&tx, E4M3, a.x, a.K, a.rows, a.x_stride, 128)) return cudaErrorInvalidValue;
    if (!encode(&tw, E4M3, a.weight, a.K, a.N, a.K, 128)) return cudaErrorInvalidValue;
    tg = tout = tw;
    if (GATED && !encode(&tg, E4M3, a.gate, a.K, a.N, a.K, 128)) return cudaErrorInvalidValue;
    auto mappable = [&](const void *ptr, int64_t stride) {
        return a.N % 8 == 0 && stride % 8 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0;
    };
    p.tma_out = mappable(a.out, a.out_stride) && (!a.residual || mappable(a.residual, a.res_stride));
    p.vec_res = p.tma_out && a.residual;
    if (p.tma_out && !encode(&tout, false, a.out, a.N, a.rows, a.out_stride, 32, kEpiCols * 2)) return cudaErrorInvalidValue;
    p.m_tiles = (a.rows + kPairM - 1) / kPairM;
    p.n_tiles = (a.N + kOut - 1) / kOut;
    auto kernel = linear_pair<E4M3, GATED>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(2 * (sms / 2)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const long long pairs = std::min<long long>((long long)p.m_tiles * p.n_tiles, pair_slots(kernel, cfg, sms));
    return launch_overlapped(kernel, dim3((unsigned)(2 * pairs)), kPairThreads, kPairSmem, 2, s, tx, tw, tg, tout, p);
}

template <bool E4M3, bool GATED>
cudaError_t launch_type(const LinearArgs &a, cudaStream_t s) {
    LinParams p{};
    p.x_scale = a.x_scale;
    p.col = {a.w_scale, a.g_scale, static_cast<const __nv_bfloat16 *>(a.bias), static_cast<const __nv_bfloat16 *>(a.g_bias)};
    p.residual = static_cast<const __nv_bfloat16 *>(a.residual);
    p.out = static_cast<__nv_bfloat16 *>(a.out);
    p.res_stride = a.res_stride;
    p.out_stride = a.out_stride;
    p.rows = a.rows;
    p.N = a.N;
    p.act = a.act;
    p.status = a.status;
    p.slices = k_slices(a);
    const int sms = device_sms();
    const Plan plan = choose(a, p.slices, sms);
    switch (plan.bn) {
        case kPairN: return launch_pair<E4M3, GATED>(a, p, sms, s);
        case 32: return launch_tile<E4M3, GATED, 32>(a, p, plan.split, s);
        case 64: return launch_tile<E4M3, GATED, 64>(a, p, plan.split, s);
        default: return launch_tile<E4M3, GATED, 128>(a, p, plan.split, s);
    }
}
}  // namespace

LinearPlan linear_plan(const LinearArgs &a) {
    if (a.rows <= kSkinnyRows) return {0, 1};
    const Plan plan = choose(a, k_slices(a), device_sms());
    return {plan.bn, plan.split};
}

cudaError_t launch_linear(const LinearArgs &a, cudaStream_t s) {
    if (a.rows <= kSkinnyRows) return launch_linear_skinny(a, s);
    if (a.e4m3) return a.gate ? launch_type<true, true>(a, s) : launch_type<true, false>(a, s);
    return a.gate ? launch_type<false, true>(a, s) : launch_type<false, false>(a, s);
}

}  // namespace a11s
