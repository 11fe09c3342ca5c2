// chunk_attn.cu - K10: attention of a chunk of new tokens over 16-token KV pages,
// TMA + tcgen05 (TMEM accumulators) on sm_100a.
//
// Token i of sequence b (i < n_new[b]) sits at position ctx_lens[b] + i and sees
// the positions 0 .. ctx_lens[b] + i:
//   s_j = scale q . k_j,  out = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
// with query head h on KV head h / (Hq / Hkv). The decode attention of the
// reference's forward_layer (engine/pipeline.py:386-402) for a whole prompt
// chunk, or for one token per sequence. Semantics: include/a11spec.h
// (a11s_chunk_attention).
//
// One CTA = one sequence, one KV head, two Q tiles of 128 rows; a row is one
// query head of one token, so a tile holds 128 / group consecutive tokens and
// the group's heads read each K/V block once (group = Hq / Hkv up to 128; rows
// that no whole token fits into stay idle). The KV range runs in blocks of 128
// keys and stops at the tiles' last visible position: half of the chunk's own
// square is never computed. 384 threads, roles and TMEM layout as in
// tree_attn.cu, whose measurements chose them:
//   warps 0-7  softmax: warp w serves tile w/4, thread = row = TMEM lane
//   warp 8     TMA producer, K and V rings; page ids fetched 4 blocks ahead
//   warp 9     TMEM allocator + S issuer (QK^T, Q and K from shared memory)
//   warp 11    PV issuer (P from TMEM, V from shared memory)
//   warp 10    idle (completes the third warpgroup for the register split)
// Large chunks are bound by the tensor core and the exponentials (128 x 128
// scores: 1024 cycles of MMA at D = 128, 1024 of ex2); a few tokens over a long
// cache by HBM: then only the live tile and its live warps work, and the KV
// range is cut into splits of equal length, merged by chunk_attn_combine in
// split order.
// Statistics, sums and accumulators are fp32; the probabilities are rounded to
// bf16 for the PV product (its operand type), the denominator sums them before
// that rounding. A row's running maximum is renewed when the block maximum
// exceeds it by more than 8 (log2 units), so exponents stay below 2^8.
// V rows past the last visible position are zeroed in shared memory: whatever
// the page holds there (a probability of 0 times a NaN would be NaN).
// Measured (one B200): 4096 tokens over 12288 (32 / 4 heads of 128) 920 to
// 935 us = 1.03 PFLOP/s; 4 x 300 over up to 2000 (24 / 8 heads of 64) 37.8 us. A softmax warp
// spends about 2750 cycles on a block, 1400 of them on the exponentials, and two
// warps share a scheduler and its MUFU: the barriers it waits at are already
// complete. Measured slower: polling them ahead of time (941 us), one tile per CTA
// with two CTAs per SM at D = 64 (55 us), a quarter of the exponentials as a
// polynomial on the FMA units (983 us), two threads a row (1785 us, spills).
// (Spills: 68 bytes at D = 128, 84 at 64.)
// Every mbarrier wait is bounded (clock budget); a timeout sets ETIMEOUT and
// the CTA drains and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace a11s {

namespace {
constexpr int kBlockKV = 128;  // keys per block = 8 pages (the N of the QK^T MMA)
constexpr int kPagesPerBlock = kBlockKV / A11S_PAGE_TOKENS;
constexpr int kTiles = 2;
constexpr int kSoftmaxWarps = 4 * kTiles;
constexpr int kProducerWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1, kPvWarp = kSoftmaxWarps + 3;
constexpr int kThreads = 32 * (kSoftmaxWarps + 4);
constexpr int kRegsSoftmax = 216, kRegsOther = 56;  // setmaxnreg split (multiples of 8)
constexpr long long kRegsNeeded = 32ll * (kSoftmaxWarps * kRegsSoftmax + 4 * kRegsOther);
constexpr uint32_t kHalf = 16384;  // 128 rows x 128 B: 64 dims of a Q tile or of a K or V block
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColO = 128, kColP = 384;  // S (128), O of tile t (D), P of tile t (64: bf16 pairs)
constexpr long long kWaitBudget = 2000000000ll;  // ~1 s of SM clock
constexpr float kRescaleThreshold = 8.0f;
constexpr int kMaxSplits = 64;

template <int D>
struct Shape {
    static constexpr int kHalves = D / 64;
    static constexpr int kKStages = D == 128 ? 2 : 4, kVStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kSlot = kHalves * kHalf;   // one K or V block
    static constexpr uint32_t kQTile = kHalves * kHalf;  // one Q tile
    static constexpr uint32_t kOffK = kTiles * kQTile, kOffV = kOffK + kKStages * kSlot;
    static constexpr uint32_t kOffBar = kOffV + kVStages * kSlot;
    static constexpr uint32_t kSmem = kOffBar + 512 + 1024;
};

struct Bars {
    uint64_t k_full[4], k_empty[4], v_full[6], v_empty[6];
    uint64_t q_ready, s_full[kTiles], s_free, p_full[kTiles], pv_done[kTiles];
    uint64_t drain, drain_pv;
    uint32_t tmem_base;
    int32_t abort;
};
static_assert(sizeof(Bars) <= 512, "barrier block");

struct Params {
    const __nv_bfloat16 *q;
    int64_t q_stride;
    const int32_t *page_table;
    int32_t max_pages, num_pages;
    const int32_t *ctx_lens, *n_new;
    int32_t B, N, Hq, Hkv, group, tokens;  // tokens: of a tile (128 / group)
    int32_t ctiles, splits, split_blocks;  // CTAs along the chunk; at most `splits` splits of split_blocks blocks
    float scale_log2;
    __nv_bfloat16 *out;
    float *lse;
    float *part_o, *part_ml;
    StatusWord *status;
};

__device__ __forceinline__ bool aborted(Bars *bs) { return *reinterpret_cast<volatile int32_t *>(&bs->abort) != 0; }
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, Bars *bs, StatusWord *st) {
    if (tc::mbar_wait(bar, parity, kWaitBudget)) return true;
    *reinterpret_cast<volatile int32_t *>(&bs->abort) = 1;
    report(st, A11S_ETIMEOUT, 0);
    return false;
}
// The same by a whole warp, with one answer for all its lanes (a converged warp stays one).
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, Bars *bs, StatusWord *st) {
    return __all_sync(0xffffffffu, wait_or_abort(bar, parity, bs, st));
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Live tokens of sequence b (0 with EBOUNDS reported when its lengths are impossible) and its context.
__device__ __forceinline__ int live_tokens(const Params &p, int b, int &ctx, bool tell) {
    ctx = p.ctx_lens[b];
    const int n = p.n_new ? p.n_new[b] : p.N;
    if (n < 0 || n > p.N || ctx < 0 || (long long)ctx + n > min((long long)p.max_pages * A11S_PAGE_TOKENS, (long long)kMaxKv)) {
        if (tell) report(p.status, A11S_EBOUNDS, b);
        ctx = 0;
        return 0;
    }
    return n;
}
}  // namespace

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_attn_tc(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const Params p) {
    using S = Shape<D>;
    constexpr int kQ16 = D / 8;  // 16-byte pieces of a head
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars *bs = reinterpret_cast<Bars *>(sm + S::kOffBar);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    let_next_start();
    wait_before();
    // the chunk's last tokens see the most keys: they start first
    int idx = blockIdx.x;
    const int g = idx % p.Hkv;
    idx /= p.Hkv;
    const int split = idx % p.splits;
    idx /= p.splits;
    const int b = idx % p.B, ct = p.ctiles - 1 - idx / p.B;

    int L;
    const int n_live = live_tokens(p, b, L, tid == 0 && ct == 0 && split == 0 && g == 0);
    const int tok0 = ct * kTiles * p.tokens;
    const int last = min(n_live, tok0 + kTiles * p.tokens) - 1;  // last live token of the CTA
    const int kv_len = L + last + 1;
    const int nblk = (kv_len + kBlockKV - 1) / kBlockKV;
    const int blk0 = split * p.split_blocks;
    // the last split goes on to the end: max_kv_len may have been too small
    const int nb = last < tok0 ? 0 : max(0, split == p.splits - 1 ? nblk - blk0 : min(p.split_blocks, nblk - blk0));
    const int nt = last < tok0 + p.tokens ? 1 : kTiles;  // live tiles

    // softmax thread -> (tile, token, query head)
    const int tile = warp / 4 < kTiles ? warp / 4 : 0;
    const int m = tid & 127;
    const int tok_local = m / p.group;
    const bool in_tile = tok_local < p.tokens;
    const int token = tok0 + tile * p.tokens + tok_local;
    const int head = g * p.group + (m - tok_local * p.group);
    const bool write = warp < kSoftmaxWarps && in_tile && token < p.N, live = write && token < n_live;
    const size_t row = write ? ((size_t)b * p.N + token) * p.Hq + head : 0;
    if (nb == 0 || (!live && write)) {
        // a row without work here: zero output (split 0 writes it: the merge skips it)
        if (write && split == 0 && !live) {
            uint4 *o = reinterpret_cast<uint4 *>(p.out + row * D);
            for (int c = 0; c < kQ16; ++c) o[c] = make_uint4(0, 0, 0, 0);
            if (p.lse) p.lse[row] = 0.0f;
        }
        if (nb == 0) return;
    }

    if (tid == 0) {
        for (int s = 0; s < S::kKStages; ++s) {
            tc::mbar_init(&bs->k_full[s], 1);
            tc::mbar_init(&bs->k_empty[s], 1);
        }
        for (int s = 0; s < S::kVStages; ++s) {
            tc::mbar_init(&bs->v_full[s], 1);
            tc::mbar_init(&bs->v_empty[s], 1);
        }
        for (int t = 0; t < kTiles; ++t) {
            tc::mbar_init(&bs->s_full[t], 1);
            tc::mbar_init(&bs->p_full[t], 4);
            tc::mbar_init(&bs->pv_done[t], 1);
        }
        tc::mbar_init(&bs->s_free, 4);
        tc::mbar_init(&bs->q_ready, 4 * nt);
        tc::mbar_init(&bs->drain, 1);
        tc::mbar_init(&bs->drain_pv, 1);
        bs->abort = 0;
        tc::fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        tc::tmem_alloc(&bs->tmem_base, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = bs->tmem_base;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    static_assert(kRegsSoftmax % 8 == 0 && kRegsOther % 8 == 0, "setmaxnreg counts");
    if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp == kProducerWarp) {
            // ---------------- TMA producer ----------------
            if (lane == 0) {
                tc::prefetch_tmap(&tk);
                tc::prefetch_tmap(&tv);
            }
            constexpr int kBlocksPerWindow = 32 / kPagesPerBlock;
            const int32_t *pt = p.page_table + (size_t)b * p.max_pages;
            const int lp0 = blk0 * kPagesPerBlock;
            // past the last visible position: -2, zero-filled. kv_len <= 16 max_pages (live_tokens)
            const int lp_end = min((kv_len + A11S_PAGE_TOKENS - 1) / A11S_PAGE_TOKENS, (blk0 + nb) * kPagesPerBlock);
            auto window = [&](int w) -> int {
                const int lp = lp0 + 32 * w + lane;
                return lp < lp_end ? pt[lp] : -2;
            };
            int cur = window(0), nxt = window(1);
            int nk = 0, nv = 0;
            for (int it = 0; it < nb && !aborted(bs); ++it) {
                const int k = it % kBlocksPerWindow;
                if (k == 0 && it > 0) {
                    cur = nxt;
                    nxt = window(it / kBlocksPerWindow + 1);
                }
                const int id = __shfl_sync(0xffffffffu, cur, (k * kPagesPerBlock + lane) & 31);
                int page = p.num_pages;  // out of range -> zero fill
                if (lane < kPagesPerBlock && id != -2) {
                    if (id < 0 || id >= p.num_pages) report(p.status, A11S_EBOUNDS, b);
                    else page = id;
                }
                const int ks = it % S::kKStages, kuse = it / S::kKStages;
                if (lane == 0 && kuse > 0) wait_or_abort(&bs->k_empty[ks], (kuse - 1) & 1, bs, p.status);
                __syncwarp();
                if (aborted(bs)) break;
                if (lane == 0) tc::mbar_arrive_expect_tx(&bs->k_full[ks], S::kSlot);
                __syncwarp();
                uint8_t *sK = sm + S::kOffK + ks * S::kSlot;
                if (lane < kPagesPerBlock)
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h)
                        tc::tma_load_4d(sK + h * kHalf + lane * 2048, &tk, &bs->k_full[ks], 64 * h, g, 0, page);
                ++nk;
                const int vs = it % S::kVStages, vuse = it / S::kVStages;
                if (lane == 0 && vuse > 0) wait_or_abort(&bs->v_empty[vs], (vuse - 1) & 1, bs, p.status);
                __syncwarp();
                if (aborted(bs)) break;
                if (lane == 0) tc::mbar_arrive_expect_tx(&bs->v_full[vs], S::kSlot);
                __syncwarp();
                uint8_t *sV = sm + S::kOffV + vs * S::kSlot;
                if (lane < kPagesPerBlock)
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h)
                        tc::tma_load_4d(sV + h * kHalf + lane * 2048, &tv, &bs->v_full[vs], 64 * h, g, 0, page);
                ++nv;
            }
            if (aborted(bs) && lane == 0) {
                // copies that may still be landing in this CTA's shared memory
                for (int i = max(0, nk - S::kKStages); i < nk; ++i)
                    tc::mbar_wait(&bs->k_full[i % S::kKStages], (i / S::kKStages) & 1, kWaitBudget);
                for (int i = max(0, nv - S::kVStages); i < nv; ++i)
                    tc::mbar_wait(&bs->v_full[i % S::kVStages], (i / S::kVStages) & 1, kWaitBudget);
            }
        } else if (warp == kMmaWarp) {
            // ---------------- S issuer ----------------
            constexpr uint32_t idesc = tc::idesc_bf16_f32(128, kBlockKV, false);
            const uint64_t qd0 = tc::sdesc_sw128(tc::smem_u32(sm), 16, 1024), kd0 = tc::sdesc_sw128(tc::smem_u32(sm + S::kOffK), 16, 1024);
            bool ok = warp_wait(&bs->q_ready, 0, bs, p.status);
            int ks = 0, kphase = 0, sphase = 1;
            for (int j = 0; j < nb && ok; ++j) {
                for (int t = 0; t < nt; ++t) {
                    if (j + t > 0) ok = warp_wait(&bs->s_free, sphase, bs, p.status);  // the tile before has loaded its S
                    sphase ^= 1;
                    if (ok && t == 0) ok = warp_wait(&bs->k_full[ks], kphase, bs, p.status);
                    if (!ok) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        const uint64_t qd = qd0 + (uint64_t)(t * (S::kQTile / 16)), kd = kd0 + (uint64_t)(ks * (S::kSlot / 16));
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            tc::mma_bf16_ss(tmem + kColS, qd + (kk >> 2) * (kHalf / 16) + (kk & 3) * 2,
                                            kd + (kk >> 2) * (kHalf / 16) + (kk & 3) * 2, idesc, kk > 0);
                        tc::mma_commit(&bs->s_full[t]);
                        if (t == nt - 1) tc::mma_commit(&bs->k_empty[ks]);
                    }
                    __syncwarp();
                }
                if (++ks == S::kKStages) {
                    ks = 0;
                    kphase ^= 1;
                }
            }
            if (tc::elect_one()) tc::mma_commit(&bs->drain);
            __syncwarp();
            tc::mbar_wait(&bs->drain, 0, kWaitBudget);
            __syncwarp();
        } else if (warp == kPvWarp) {
            // ---------------- PV issuer ----------------
            constexpr uint32_t idesc = tc::idesc_bf16_f32(128, D, true);
            const uint64_t vd0 = tc::sdesc_sw128(tc::smem_u32(sm + S::kOffV), kHalf, 1024);
            bool ok = true;
            int vs = 0, vphase = 0;
            for (int j = 0; j < nb && ok; ++j) {
                ok = warp_wait(&bs->v_full[vs], vphase, bs, p.status);
                if (!ok) break;
                // the page that holds the last visible position: zero its rows past it
                const int end = kv_len - (blk0 + j) * kBlockKV;  // visible rows of the block
                if (end < kBlockKV && (end & 15) != 0) {
                    uint8_t *sV = sm + S::kOffV + vs * S::kSlot;
                    const int rows = 16 - (end & 15);
                    for (int i = lane; i < rows * 8 * S::kHalves; i += 32)
                        *reinterpret_cast<uint4 *>(sV + (i / (rows * 8)) * kHalf + end * 128 + (i % (rows * 8)) * 16) =
                            make_uint4(0, 0, 0, 0);
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                }
                for (int t = 0; t < nt; ++t) {
                    ok = warp_wait(&bs->p_full[t], j & 1, bs, p.status);
                    if (!ok) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        const uint64_t vd = vd0 + (uint64_t)(vs * (S::kSlot / 16));
#pragma unroll
                        for (int kk = 0; kk < kBlockKV / 16; ++kk)
                            tc::mma_bf16_ts(tmem + kColO + D * t, tmem + kColP + 64 * t + kk * 8, vd + kk * (2048 / 16), idesc,
                                            (j > 0 || kk > 0) ? 1u : 0u);
                        tc::mma_commit(&bs->pv_done[t]);
                        if (t == nt - 1) tc::mma_commit(&bs->v_empty[vs]);
                    }
                    __syncwarp();
                }
                if (++vs == S::kVStages) {
                    vs = 0;
                    vphase ^= 1;
                }
            }
            if (tc::elect_one()) tc::mma_commit(&bs->drain_pv);
            __syncwarp();
            tc::mbar_wait(&bs->drain_pv, 0, kWaitBudget);
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        if (tile < nt) {
            // ---------------- softmax warps: thread = query row ----------------
            {  // Q row into the tile's 128-byte-swizzled K-major operand, zeros for rows without work
                const uint32_t q_row = tc::smem_u32(sm + tile * S::kQTile + m * 128);
                const uint4 *src = reinterpret_cast<const uint4 *>(p.q + ((int64_t)b * p.N + token) * p.q_stride + head * D);
#pragma unroll
                for (int c = 0; c < kQ16; ++c) {
                    const uint4 v = live ? src[c] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    tc::st_shared_v4(q_row + (uint32_t)(c >> 3) * kHalf + ((uint32_t)((c & 7) ^ (m & 7)) << 4), w);
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bs->q_ready);
            }
            const bool warp_live = __any_sync(0xffffffffu, live);  // a warp without live rows keeps the barriers going only
            const int lim = live ? L + token : INT32_MAX;          // last visible position
            const uint32_t p_cols = tmem + lane_base + kColP + 64 * tile;
            const uint32_t o_cols = tmem + lane_base + kColO + D * tile;
            const float sl2 = p.scale_log2;
            float m_ref = -INFINITY, lsum = 0.0f;
            bool ok = true;
            for (int it = 0; it < nb && ok; ++it) {
                const int p0 = (blk0 + it) * kBlockKV;
                ok = warp_wait(&bs->s_full[tile], it & 1, bs, p.status);
                if (!ok) break;
                tc::tc_fence_after();
                float xa[64], xb[64];
                if (warp_live) {
                    tc::tmem_ld64(tmem + lane_base + kColS, xa);
                    tc::tmem_ld64(tmem + lane_base + kColS + 64, xb);
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bs->s_free);
#define X(c) ((c) < 64 ? xa[(c) & 63] : xb[(c) & 63])
                float alpha = 1.0f, neg = 0.0f;
                bool rescale = false;
                if (warp_live) {
                    if (p0 + kBlockKV - 1 > lim) {
                        const int seen = lim - p0;  // columns up to this one
#pragma unroll
                        for (int c = 0; c < kBlockKV; ++c)
                            if (c > seen) X(c) = -INFINITY;
                    }
                    float mx8[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) mx8[q] = xa[q];
#pragma unroll
                    for (int c = 8; c + 16 <= kBlockKV; c += 16)
#pragma unroll
                        for (int q = 0; q < 8; ++q) mx8[q] = fmax3(mx8[q], X(c + q), X(c + 8 + q));
#pragma unroll
                    for (int q = 0; q < 8; ++q) mx8[q] = fmaxf(mx8[q], X(kBlockKV - 8 + q));
                    const float mx = fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
                    const float mb = mx * sl2;  // scale > 0: max commutes with scaling
                    if (mx > -INFINITY) {
                        if (m_ref == -INFINITY) {
                            m_ref = mb;  // first visible block of this row: its O row is still zero
                        } else if (mb > m_ref + kRescaleThreshold) {
                            alpha = tc::ex2(m_ref - mb);
                            m_ref = mb;
                            rescale = true;
                        }
                    }
                    neg = m_ref == -INFINITY ? 0.0f : -m_ref;
                }
                // PV(it - 1) has read P and accumulated into O
                if (it > 0) {
                    ok = warp_wait(&bs->pv_done[tile], (it - 1) & 1, bs, p.status);
                    if (!ok) break;
                    tc::tc_fence_after();
                }
                if (warp_live) {
                    float2 ls[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                    for (int c32 = 0; c32 < kBlockKV / 32; ++c32) {
                        uint32_t pw[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int c = 32 * c32 + 2 * e;
                            const float2 ev = tc::ffma2(make_float2(X(c), X(c + 1)), make_float2(sl2, sl2), make_float2(neg, neg));
                            const float2 a = make_float2(tc::ex2(ev.x), tc::ex2(ev.y));
                            pw[e] = tc::cvt_bf16x2(a.x, a.y);
                            ls[e & 3] = tc::fadd2(ls[e & 3], a);
                        }
                        tc::tmem_st16u_nowait(p_cols + 16 * c32, pw);
                    }
                    lsum = lsum * alpha + (((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y)) + ((ls[2].x + ls[2].y) + (ls[3].x + ls[3].y)));
                    if (__any_sync(0xffffffffu, rescale) && it > 0) {
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            float o[32];
                            tc::tmem_ld32(o_cols + c * 32, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] *= alpha;
                            tc::tmem_st32(o_cols + c * 32, o);
                        }
                    }
                    tc::tmem_wait_st();
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bs->p_full[tile]);
#undef X
            }
            // ---------------- epilogue ----------------
            if (ok && warp_wait(&bs->pv_done[tile], (nb - 1) & 1, bs, p.status) && warp_live) {
                tc::tc_fence_after();
                // a row whose every score is -inf has no weight: zeros; a NaN stays one
                const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
                if (p.splits == 1) {
                    uint4 *o16 = reinterpret_cast<uint4 *>(p.out + row * D);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float o[32];
                        tc::tmem_ld32(o_cols + c * 32, o);
                        if (live) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    w[e] = tc::cvt_bf16x2(o[q * 8 + 2 * e] * inv, o[q * 8 + 2 * e + 1] * inv);
                                o16[c * 4 + q] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    if (live && p.lse) p.lse[row] = lsum == 0.0f ? 0.0f : (m_ref + log2f(lsum)) * 0.6931471805599453f;
                } else {
                    const size_t prow = (size_t)split * p.B * p.N * p.Hq + row;
                    float4 *po = reinterpret_cast<float4 *>(p.part_o + prow * D);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float o[32];
                        tc::tmem_ld32(o_cols + c * 32, o);
                        if (live)
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                po[c * 8 + q] = make_float4(o[q * 4] * inv, o[q * 4 + 1] * inv, o[q * 4 + 2] * inv, o[q * 4 + 3] * inv);
                    }
                    if (live) {
                        p.part_ml[prow * 2] = lsum == 0.0f ? -INFINITY : m_ref;
                        p.part_ml[prow * 2 + 1] = lsum;
                    }
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

// Merge of the splits of each live row, in split order: one warp per (b, token,
// head); the splits' weights first, one or two per lane.
template <int D>
__global__ void __launch_bounds__(256) chunk_attn_combine(const Params p) {
    constexpr int W = D / 32;  // dims of a lane
    const size_t row = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (size_t)p.B * p.N * p.Hq;
    let_next_start();
    wait_before();
    if (row >= rows) return;
    const int lane = threadIdx.x & 31, b = (int)(row / ((size_t)p.N * p.Hq)), token = (int)((row / p.Hq) % p.N);
    int L;
    const int n_live = live_tokens(p, b, L, false);
    if (token >= n_live) return;  // its zeros are written
    // the splits of the CTA that held this token
    const int per_cta = kTiles * p.tokens, last = min(n_live, (token / per_cta + 1) * per_cta) - 1;
    const int nblk = (L + last + kBlockKV) / kBlockKV;
    const int splits = min(p.splits, (nblk + p.split_blocks - 1) / p.split_blocks);
    // weights 2^(m - M) l over their sum (each split's output is already divided by its l)
    float m[kMaxSplits / 32], w[kMaxSplits / 32], M = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
        const int s = lane + 32 * i;
        const size_t at = ((size_t)min(s, splits - 1) * rows + row) * 2;
        m[i] = p.part_ml[at];
        w[i] = s < splits ? p.part_ml[at + 1] : 0.0f;
        if (w[i] != 0.0f) M = fmaxf(M, m[i]);
    }
    M = warp_fmax(M);
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
        w[i] = w[i] == 0.0f ? 0.0f : w[i] * exp2f(m[i] - M);
        sum += w[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float *po = p.part_o + row * D + lane * W;
    float acc[W] = {};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const float f = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[kMaxSplits / 32 - 1], s & 31);
        float o[W];
        if constexpr (W == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(po + (size_t)s * rows * D);
            o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2 *>(po + (size_t)s * rows * D);
            o[0] = v.x, o[1] = v.y;
        }
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] = fmaf(f, f == 0.0f ? 0.0f : o[e], acc[e]);  // a split that saw nothing takes no part
    }
    uint32_t *out = reinterpret_cast<uint32_t *>(p.out + row * D + lane * W);
#pragma unroll
    for (int e = 0; e < W; e += 2) out[e / 2] = tc::cvt_bf16x2(acc[e] * inv, acc[e + 1] * inv);
    if (p.lse && lane == 0) p.lse[row] = sum == 0.0f ? 0.0f : (M + log2f(sum)) * 0.6931471805599453f;
}
static_assert(kMaxSplits == 64, "two weights per lane");

// ---------------------------------------------------------------------------- host side
// Clears the status word and the merge counters: a kernel and not a memset, so
// that the attention can start over its tail.
namespace {
__global__ void chunk_attn_clear(uint32_t *words, int n) {
    let_next_start();
    wait_before();
    for (int i = threadIdx.x; i < n; i += blockDim.x) words[i] = 0;
}
}  // namespace
cudaError_t launch_chunk_attention_clear(void *workspace, size_t bytes, cudaStream_t s) {
    return launch_overlapped(chunk_attn_clear, dim3(1), 256, 0, 1, s, static_cast<uint32_t *>(workspace), (int)(bytes / 4));
}

ChunkPlan chunk_attention_plan(int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t max_kv_len) {
    int sms = 148, dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    ChunkPlan c;
    if ((long long)N * (Hq / Hkv) <= kChunkRows && B <= kChunkRowsMaxBatch) {
        c.rows = true;
        c.splits = chunk_rows_ctas(sms);
        return c;
    }
    c.tokens = 128 / (Hq / Hkv);
    c.ctiles = (N + kTiles * c.tokens - 1) / (kTiles * c.tokens);
    const long long ctas = (long long)B * Hkv * c.ctiles;
    const int blocks = std::max(1, (max_kv_len + kBlockKV - 1) / kBlockKV);
    double best = 1e300;
    for (int s = 1; s <= std::min(kMaxSplits, blocks); ++s) {
        const int bps = (blocks + s - 1) / s;
        // in units of a block (about 1 us): whole waves while they are few, and 12
        // blocks of fixed cost a CTA; split, the merge and its partial outputs'
        // way through memory (B N Hq rows of D fp32 per split, written and read)
        const double w = (double)(ctas * s) / sms, waves = w <= 3.0 ? std::ceil(w) : w + 0.5;
        const double merge = s > 1 ? 4.0 + (double)B * N * Hq * s * 128 * 8 / 6.5e6 : 0.0;
        const double cost = waves * (bps + 12.0) + merge;
        if (cost < best * 0.98) {
            best = cost;
            c.splits = s;
        }
    }
    c.split_blocks = (blocks + c.splits - 1) / c.splits;
    c.splits = (blocks + c.split_blocks - 1) / c.split_blocks;
    return c;
}

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

// K or V [pages][16][Hkv][D]: box 64 dims x 1 head x 16 tokens x 1 page
bool encode_pool(CUtensorMap *map, const void *base, int D, int Hkv, int pages) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)Hkv, 16, (cuuint64_t)pages};
    const cuuint64_t str[3] = {(cuuint64_t)D * 2, (cuuint64_t)Hkv * D * 2, (cuuint64_t)Hkv * D * 32};
    const cuuint32_t box[4] = {64, 1, 16, 1}, estr[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, str, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch_d(const ChunkAttnArgs &a, const Params &p, cudaStream_t s) {
    CUtensorMap tk, tv;
    if (!encode_pool(&tk, a.k_pool, D, a.Hkv, a.num_pages) || !encode_pool(&tv, a.v_pool, D, a.Hkv, a.num_pages))
        return cudaErrorInvalidValue;
    auto kernel = chunk_attn_tc<D>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes fa{};
    e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return e;
    // setmaxnreg.inc would wait forever if the split needed more registers than the launch holds
    if ((long long)fa.numRegs * kThreads < kRegsNeeded) return cudaErrorInvalidConfiguration;
    e = launch_overlapped(kernel, dim3((unsigned)((long long)p.ctiles * p.B * p.splits * p.Hkv)), kThreads, Shape<D>::kSmem, 1, s,
                          tk, tv, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_overlapped(chunk_attn_combine<D>, dim3((unsigned)(((size_t)p.B * p.N * p.Hq + 7) / 8)), 256, 0, 1, s, p);
}
}  // namespace

cudaError_t launch_chunk_attention(const ChunkAttnArgs &a, cudaStream_t s) {
    if (a.plan.rows) return launch_chunk_attention_rows(a, s);
    Params p{};
    p.q = reinterpret_cast<const __nv_bfloat16 *>(a.q);
    p.q_stride = a.q_stride;
    p.page_table = a.page_table;
    p.max_pages = a.max_pages;
    p.num_pages = a.num_pages;
    p.ctx_lens = a.ctx_lens;
    p.n_new = a.n_new;
    p.B = a.B;
    p.N = a.N;
    p.Hq = a.Hq;
    p.Hkv = a.Hkv;
    p.group = a.Hq / a.Hkv;
    p.tokens = a.plan.tokens;
    p.ctiles = a.plan.ctiles;
    p.splits = a.plan.splits;
    p.split_blocks = a.plan.split_blocks;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.out = reinterpret_cast<__nv_bfloat16 *>(a.out);
    p.lse = a.lse;
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.status = a.status;
    return a.D == 128 ? launch_d<128>(a, p, s) : launch_d<64>(a, p, s);
}

}  // namespace a11s
