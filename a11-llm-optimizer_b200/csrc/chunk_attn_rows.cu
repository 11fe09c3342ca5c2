// chunk_attn_rows.cu - K10 for few query rows (tokens x heads of a KV head at
// most 32: one token per sequence, mostly): the cache is streamed once, all
// else is small.
//
// The formulas of chunk_attn.cu. Bound by HBM: every visible K and V row is read
// once. A tile of 128 query rows would be nearly empty and its chain (S, softmax
// of 128 keys in one thread, PV) takes 2700 cycles per 64 KB whatever the rows,
// so the keys take the tile's place: per page of 16 tokens a warp computes
//   S^T (16 keys x 8 rows) = K Q^T,  O^T (D x 8 rows) += V^T P^T
// with m16n8k16 instructions. A lane then holds 2 keys x 2 rows: the exponentials
// are spread over all lanes, the probabilities become the next operand by two
// 8 x 8 transposes, and the rows' maxima and sums stay in the lanes that own
// those rows of O^T.
// A warp streams its own pages (every eighth of its CTA's share) through a ring
// of its own in shared memory (cp.async, 16-byte pieces, swizzled for ldmatrix),
// with a running maximum of its own: no barrier inside a share.
// One CTA per SM. The pages of all sequences and KV heads, laid end to end, are
// cut into one equal share per CTA, so ragged lengths leave no SM idle: a CTA
// may finish one sequence's tail, whole sequences, and another's head. What it
// has of a sequence that others share goes to the workspace; the last of them to
// finish (a counter) merges the pieces, in order along the sequence. Batches of
// short sequences (16 pages a slot on average, and none above 128) are not cut: a
// CTA takes whole ones. The longest one decides too, since a padded batch may hold
// one long sequence among empty slots. Whole against cut, 64 sequences of 100 tokens
// (32 / 4 heads of 128) some of which have more: four of 900 19.5 / 24.6 us, one of
// 2100 24.3 / 24.6, one of 4000 32.7 / 24.6; 64 slots, one of 15000 and the others
// empty, 76 / 23.
// Tokens past the last visible one are never read: their copies are zero-filled.
// Measured (one B200): 32 sequences of one token over up to 4096 (32 / 4 heads of
// 128, 200 MB) 41 us = 4.9 TB/s, 61 through chunk_attn_tc; one token over 32767
// (67 MB, 37 pieces per KV head) 23.8 us, 33 through chunk_attn_tc with 64 splits; with
// 24 / 8 heads of 64, 32 sequences 43.5 us = 4.6 TB/s, one token over 32767 23.7 us. The
// kernel of 25 to 32 rows of 128 dims spills 160 bytes.
// The probabilities are rounded to bf16 for the product with V, as in chunk_attn.cu.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "mma_sync.cuh"
#include "tc_common.cuh"

namespace a11s {

namespace {
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr float kRescaleThreshold = 8.0f;
constexpr int kMinPages = 16;    // of a CTA's share
constexpr int kWholePages = 128; // of the longest sequence of a batch that is not cut
constexpr int kMaxShares = 256;  // CTAs of a launch

template <int D>
struct Shape {
    static constexpr uint32_t kPage = 16 * D * 2;  // K or V of a page and KV head
    static constexpr uint32_t kStage = 2 * kPage;
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kRing = kStages * kStage;  // of a warp: 24 KB
    static constexpr uint32_t kSmem = kWarps * kRing + (kChunkRowsMaxBatch + 1) * 4;
    static constexpr int kPitch = D + 4;  // floats between rows of O in the merge
};

struct Params {
    const __nv_bfloat16 *q, *k, *v;
    int64_t q_stride;
    const int32_t *page_table;
    int32_t max_pages, num_pages;
    const int32_t *ctx_lens, *n_new;
    int32_t B, N, Hq, Hkv, group;
    float scale_log2;
    __nv_bfloat16 *out;
    float *lse;
    float *part_o, *part_ml;  // [2 per CTA][8 NT][D], [2 per CTA][8 NT][2]
    int32_t *counters;        // [B][Hkv], zero at the launch
    StatusWord *status;
};

// Context and live tokens of sequence b; both 0 when they are impossible.
__device__ __forceinline__ int lengths(const Params &p, int b, int &ctx) {
    ctx = p.ctx_lens[b];
    const int n = p.n_new ? p.n_new[b] : p.N;
    if (n >= 0 && n <= p.N && ctx >= 0 && (long long)ctx + n <= min((long long)p.max_pages * A11S_PAGE_TOKENS, (long long)kMaxKv)) return n;
    ctx = 0;
    return -1;
}
// 2^a with 2^(-inf) = 0 also for a = -inf - (-inf).
__device__ __forceinline__ float weight2(float m, float M) { return m == -INFINITY ? 0.0f : exp2f(m - M); }
}  // namespace

// NT: tiles of 8 query rows.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads, 1) chunk_attn_rows(const Params p) {
    using S = Shape<D>;
    constexpr int kSteps = D / 16, kRows = 8 * NT;
    extern __shared__ __align__(1024) uint8_t smem[];
    int32_t *prefix = reinterpret_cast<int32_t *>(smem + kWarps * S::kRing);  // [B + 1]: pages before sequence b
    __shared__ float2 ml[kWarps][kRows];
    __shared__ int is_last, warp_sum[kWarps], warp_longest[kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, t4 = lane & 3;

    let_next_start();
    wait_before();
    // ---------------- pages of the sequences, summed up ----------------
    {
        const int per = (p.B + kThreads - 1) / kThreads, b0 = tid * per;
        int sum = 0, most = 0;
        for (int b = b0; b < min(b0 + per, p.B); ++b) {
            int ctx;
            const int n = lengths(p, b, ctx);
            if (n < 0 && blockIdx.x == 0) report(p.status, A11S_EBOUNDS, b);
            const int pages = n > 0 ? (ctx + n + A11S_PAGE_TOKENS - 1) / A11S_PAGE_TOKENS : 0;
            prefix[b] = sum;
            sum += pages;
            most = max(most, pages);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) {
            warp_sum[warp] = incl;
            warp_longest[warp] = most;
        }
        __syncthreads();
        int before = incl - sum;
        for (int w = 0; w < warp; ++w) before += warp_sum[w];
        for (int b = b0; b < min(b0 + per, p.B); ++b) prefix[b] += before;
        if (tid == kThreads - 1) prefix[p.B] = before + sum;
        __syncthreads();
    }
    // rows without work: zeros
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        int ctx;
        const int n = max(0, lengths(p, b, ctx));
        const size_t row = ((size_t)b * p.N + n) * p.Hq;
        for (int64_t i = tid; i < (int64_t)(p.N - n) * p.Hq * (D / 8); i += kThreads) {
            reinterpret_cast<uint4 *>(p.out + row * D)[i] = make_uint4(0, 0, 0, 0);
            if (p.lse && i % (D / 8) == 0) p.lse[row + i / (D / 8)] = 0.0f;
        }
    }
    // this CTA's share: pages [r0, r1) of all, or (short sequences) whole units.
    // All counts fit 32 bits (checked on the host).
    const int units = p.B * p.Hkv, total = prefix[p.B] * p.Hkv;
    if (total == 0) return;
    int longest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) longest = max(longest, warp_longest[w]);
    const bool whole = longest <= kWholePages && total <= units * 16ll;
    const int shares = min((int)gridDim.x, whole ? units : (total + kMinPages - 1) / kMinPages), me = blockIdx.x;
    if (me >= shares) return;
    const int each = total / shares, extra = total % shares;  // the first `extra` shares have a page more
    auto share_start = [&](int c) { return each * c + min(c, extra); };
    auto share_of = [&](int x) {  // the CTA whose share holds page x
        const int longer = extra * (each + 1);
        return x < longer ? x / (each + 1) : extra + (x - longer) / each;
    };
    const int r0 = whole ? 0 : share_start(me), r1 = whole ? 0 : share_start(me + 1);
    // the first unit: (b, g), and the page it starts at
    int b, g;
    if (whole) {
        b = me / p.Hkv;
        g = me % p.Hkv;
    } else {
        int lo = 0, hi = p.B - 1;  // the last b with prefix[b] * Hkv <= r0
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (prefix[mid] * p.Hkv <= r0) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        g = (r0 - prefix[b] * p.Hkv) / (prefix[b + 1] - prefix[b]);
    }
    const float sl2 = p.scale_log2;
    const int mrow = lane & 7, mi = lane >> 3;  // ldmatrix: this lane's row of matrix mi
    const uint32_t ring = tc::smem_u32(smem) + warp * S::kRing;
    const int64_t token_stride = (int64_t)p.Hkv * D;
    // copies of a page: lane moves 16 bytes of token (32 c + lane) / (D / 8) in
    // copy c; where they land repeats (but for 512 bytes a copy) with the swizzle
    constexpr int kCopies = S::kPage / 512, kPhases = D == 128 ? 4 : 2;
    const int64_t lane_src = lane / (D / 8) * token_stride + lane % (D / 8) * 8, copy_step = 32 / (D / 8) * token_stride;
    uint32_t lane_dst[kPhases];
#pragma unroll
    for (int c = 0; c < kPhases; ++c) {
        const int row = (c * 32 + lane) / (D / 8);
        lane_dst[c] = row * (D * 2) + (((lane % (D / 8)) ^ (row & 7)) << 4);
    }

    for (;;) {
        int L;
        const int n_live = max(0, lengths(p, b, L));
        const int rows = n_live * p.group, kv_len = L + n_live, pages = prefix[b + 1] - prefix[b];
        const int f0 = prefix[b] * p.Hkv + g * pages, f1 = f0 + pages;  // the unit in the row of pages
        const int first = whole ? 0 : max(f0, r0) - f0, count = whole ? pages : min(f1, r1) - f0 - first;
        const bool shared_unit = count != pages;
        const size_t row0 = (size_t)b * p.N * p.Hq + g * p.group;
        auto row_of = [&](int r) { return row0 + (size_t)(r / p.group) * p.Hq + r % p.group; };
        if (count > 0) {
            const int mine = (count - warp + kWarps - 1) / kWarps;  // pages first + warp, + 8, ...
            const int32_t *table = p.page_table + (size_t)b * p.max_pages + first + warp;
            int ids = lane < mine ? table[kWarps * lane] : 0;  // page ids of 32 of the warp's pages, from ids0 on
            int ids0 = 0;
            auto issue = [&](int i) {  // K and V of the warp's page i into its ring slot
                if (i < mine) {
                    if (i - ids0 >= 32) {
                        ids0 += 32;
                        ids = ids0 + lane < mine ? table[kWarps * (ids0 + lane)] : 0;
                    }
                    int id = __shfl_sync(0xffffffffu, ids, i - ids0);
                    const bool good = id >= 0 && id < p.num_pages;
                    if (!good) {
                        if (lane == 0) report(p.status, A11S_EBOUNDS, b);
                        id = 0;
                    }
                    const int left = kv_len - (first + warp + kWarps * i) * A11S_PAGE_TOKENS;  // tokens of the page
                    const int64_t base = (int64_t)id * A11S_PAGE_TOKENS * token_stride + g * D + lane_src;
                    const uint32_t slot = ring + (i % S::kStages) * S::kStage;
                    const __nv_bfloat16 *ks = p.k + base, *vs = p.v + base;
                    if (good && left >= A11S_PAGE_TOKENS) {
#pragma unroll
                        for (int c = 0; c < kCopies; ++c) {
                            const uint32_t dst = slot + lane_dst[c % kPhases] + c / kPhases * (kPhases * 512);
                            cp_async16(dst, ks, true);
                            cp_async16(dst + S::kPage, vs, true);
                            ks += copy_step;
                            vs += copy_step;
                        }
                    } else {  // the last page, or none: zeros past the end
#pragma unroll
                        for (int c = 0; c < kCopies; ++c) {
                            const uint32_t dst = slot + lane_dst[c % kPhases] + c / kPhases * (kPhases * 512);
                            const bool in = good && (c * 32 + lane) / (D / 8) < left;
                            cp_async16(dst, in ? ks + c * copy_step : p.k, in);
                            cp_async16(dst + S::kPage, in ? vs + c * copy_step : p.v, in);
                        }
                    }
                }
                cp_async_commit();
            };
#pragma unroll
            for (int i = 0; i < S::kStages - 1; ++i) issue(i);
            // (the copies are under way) the CTAs that hold pieces of the unit
            const int c0 = shared_unit ? share_of(f0) : me, n = shared_unit ? share_of(f1 - 1) - c0 + 1 : 1;
            // rows of Q as operand B: column r of tile j is query row 8 j + r
            uint32_t qf[NT][kSteps][2];
            int lim[NT][2];  // last position that rows 8 j + 2 t4, + 1 see
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int r = 8 * j + g4, token = r / p.group;
                const bool in = r < rows;
                const __nv_bfloat16 *src = p.q + ((int64_t)b * p.N + (in ? token : 0)) * p.q_stride + (g * p.group + (in ? r % p.group : 0)) * D;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    qf[j][s][0] = in ? *reinterpret_cast<const uint32_t *>(src + 16 * s + 2 * t4) : 0u;
                    qf[j][s][1] = in ? *reinterpret_cast<const uint32_t *>(src + 16 * s + 8 + 2 * t4) : 0u;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int rr = 8 * j + 2 * t4 + e;
                    lim[j][e] = rr < rows ? L + rr / p.group : kv_len - 1;
                }
            }
            float o[NT][kSteps][4] = {};
            float m_ref[NT][2], lsum[NT][2] = {};
#pragma unroll
            for (int j = 0; j < NT; ++j) m_ref[j][0] = m_ref[j][1] = -INFINITY;
            for (int i = 0; i < mine; ++i) {
                cp_async_wait<S::kStages - 2>();
                __syncwarp();  // every lane's copies of page i, and nobody reads page i - 1 any more
                const uint32_t sk = ring + (i % S::kStages) * S::kStage, sv = sk + S::kPage;
                const int pos0 = (first + warp + kWarps * i) * A11S_PAGE_TOKENS;
                float s[NT][2][4] = {};  // two chains of accumulation
                {
                    const int row = (mi & 1) * 8 + mrow;
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) {
                        uint32_t a[4];
                        ldmatrix4(a, sk + row * (D * 2) + (((2 * ks + (mi >> 1)) ^ (row & 7)) << 4));
#pragma unroll
                        for (int j = 0; j < NT; ++j) mma16816_bf16(s[j][ks & 1], a, qf[j][ks][0], qf[j][ks][1]);
                    }
                }
                issue(i + S::kStages - 1);
                uint32_t pb[NT][2];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float x[4];  // keys g4 and g4 + 8, rows 2 t4 and + 1
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = s[j][0][e] + s[j][1][e];
                    if (pos0 + A11S_PAGE_TOKENS - 1 > L) {  // some row may not see some key
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (pos0 + g4 + 8 * (e >> 1) > lim[j][e & 1]) x[e] = -INFINITY;
                    }
                    // The reference maximum follows lazily (as in chunk_attn.cu): while no
                    // lane is more than 8 above it, the maxima are not even formed.
                    const float mx0 = fmaxf(x[0], x[2]) * sl2, mx1 = fmaxf(x[1], x[3]) * sl2;
                    if (__any_sync(0xffffffffu, mx0 > m_ref[j][0] + kRescaleThreshold || mx1 > m_ref[j][1] + kRescaleThreshold)) {
                        float mx[2] = {mx0, mx1}, alpha[2];
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) {
                            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], d));
                            mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], d));
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            alpha[e] = 1.0f;
                            if (mx[e] > m_ref[j][e] + kRescaleThreshold) {
                                alpha[e] = weight2(m_ref[j][e], mx[e]);
                                m_ref[j][e] = mx[e];
                            }
                        }
                        lsum[j][0] *= alpha[0];
                        lsum[j][1] *= alpha[1];
#pragma unroll
                        for (int mt = 0; mt < kSteps; ++mt) {
                            o[j][mt][0] *= alpha[0];
                            o[j][mt][1] *= alpha[1];
                            o[j][mt][2] *= alpha[0];
                            o[j][mt][3] *= alpha[1];
                        }
                    }
                    const float neg[2] = {m_ref[j][0] == -INFINITY ? 0.0f : -m_ref[j][0], m_ref[j][1] == -INFINITY ? 0.0f : -m_ref[j][1]};
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = tc::ex2(fmaf(x[e], sl2, neg[e & 1]));
                    lsum[j][0] += x[0] + x[2];
                    lsum[j][1] += x[1] + x[3];
                    pb[j][0] = transpose8(tc::cvt_bf16x2(x[0], x[1]));  // row g4, keys 2 t4, + 1
                    pb[j][1] = transpose8(tc::cvt_bf16x2(x[2], x[3]));  // the same, keys + 8
                }
                {
                    const int key = (mi >> 1) * 8 + mrow;
#pragma unroll
                    for (int mt = 0; mt < kSteps; ++mt) {
                        uint32_t a[4];  // V^T: dims 16 mt + g4, + 8; keys
                        ldmatrix4_trans(a, sv + key * (D * 2) + (((2 * mt + (mi & 1)) ^ (key & 7)) << 4));
#pragma unroll
                        for (int j = 0; j < NT; ++j) mma16816_bf16(o[j][mt], a, pb[j][0], pb[j][1]);
                    }
                }
            }
            // ---------------- the warps' results, merged in warp order ----------------
            cp_async_wait<0>();
            __syncthreads();
            float *so = reinterpret_cast<float *>(smem);  // [warp][8 NT rows][kPitch]
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float l = lsum[j][e];
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                    if (g4 == 0) ml[warp][8 * j + 2 * t4 + e] = make_float2(m_ref[j][e], l);
                }
#pragma unroll
                for (int mt = 0; mt < kSteps; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        so[(warp * kRows + 8 * j + 2 * t4 + (e & 1)) * S::kPitch + 16 * mt + g4 + 8 * (e >> 1)] = o[j][mt][e];
            }
            __syncthreads();
            constexpr int kDims4 = D / 4;  // threads of a row, four dims each
            const int d4 = tid % kDims4 * 4;
            // pieces of a unit: slot 1 of the CTA it starts in, slot 0 of those it goes on in
            const size_t slot = 2 * (size_t)me + (f0 < r0 ? 0 : 1);
            for (int r = tid / kDims4; r < rows; r += kThreads / kDims4) {
                float M = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w][r].x);
                float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float2 v = ml[w][r];
                    const float4 a = *reinterpret_cast<const float4 *>(so + (w * kRows + r) * S::kPitch + d4);
                    const float f = weight2(v.x, M);
                    if (v.x == -INFINITY && v.y == 0.0f) continue;  // saw nothing
                    l += f * v.y;
                    acc.x += f * a.x;
                    acc.y += f * a.y;
                    acc.z += f * a.z;
                    acc.w += f * a.w;
                }
                if (!shared_unit) {
                    const size_t row = row_of(r);
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    *reinterpret_cast<uint2 *>(p.out + row * D + d4) =
                        make_uint2(tc::cvt_bf16x2(acc.x * inv, acc.y * inv), tc::cvt_bf16x2(acc.z * inv, acc.w * inv));
                    if (p.lse && d4 == 0) p.lse[row] = l == 0.0f ? 0.0f : (M + log2f(l)) * 0.6931471805599453f;
                } else {
                    __stcg(reinterpret_cast<float4 *>(p.part_o + (slot * kRows + r) * D + d4), acc);
                    if (d4 == 0) __stcg(reinterpret_cast<float2 *>(p.part_ml + (slot * kRows + r) * 2), make_float2(M, l));
                }
            }
            if (shared_unit) {
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    is_last = atomicAdd(p.counters + b * p.Hkv + g, 1) == n - 1;
                    __threadfence();
                }
                __syncthreads();
                if (is_last) {
                    // Weights of the pieces in shared memory, [row][kMaxShares]; behind them the
                    // pieces' outputs, copied there all at once (as many as fit) while the weights
                    // are formed. Every thread copies and later reads elements of its own.
                    float *wgt = reinterpret_cast<float *>(smem);
                    constexpr uint32_t kStageAt = kRows * kMaxShares * 4;
                    constexpr int kRowThreads = kThreads / kDims4;                    // rows side by side
                    constexpr int kNr = (kRows + kRowThreads - 1) / kRowThreads;      // rows of a thread
                    constexpr int kGroup = (kWarps * S::kRing - kStageAt) / (kThreads * 16) / kNr;  // pieces at a time
                    auto my_row = [&](int k) { return min(tid / kDims4 + k * kRowThreads, kRows - 1); };
                    const uint32_t mine16 = tc::smem_u32(smem) + kStageAt + tid * 16;
                    // piece i of the unit sits in slot 2 (c0 + i), the first one in 2 c0 + 1
                    const float *piece0 = p.part_o + (size_t)2 * c0 * kRows * D + d4;
                    const float *ml0 = p.part_ml + (size_t)2 * c0 * kRows * 2;
                    auto fetch = [&](int i0) {
                        const int m = min(kGroup, n - i0);
#pragma unroll 4
                        for (int i = 0; i < m; ++i) {
                            const float *src = piece0 + (2 * (i0 + i) + (i0 + i == 0)) * (kRows * D);
#pragma unroll
                            for (int k = 0; k < kNr; ++k)  // rows past the last hold nothing and are not used
                                cp_async16(mine16 + (i * kNr + k) * (kThreads * 16), src + my_row(k) * D, true);
                        }
                        cp_async_commit();
                    };
                    fetch(0);
                    for (int r = warp; r < rows; r += kWarps) {
                        float2 v[kMaxShares / 32];
                        float M = -INFINITY, sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < kMaxShares / 32; ++i) {
                            const int at = lane + 32 * i;
                            v[i] = make_float2(-INFINITY, 0.0f);
                            if (at < n) v[i] = __ldcg(reinterpret_cast<const float2 *>(ml0 + ((2 * at + (at == 0)) * kRows + r) * 2));
                        }
#pragma unroll
                        for (int i = 0; i < kMaxShares / 32; ++i) M = fmaxf(M, v[i].x);
                        M = warp_fmax(M);
#pragma unroll
                        for (int i = 0; i < kMaxShares / 32; ++i) {
                            if (32 * i >= n) break;
                            v[i].x = v[i].x == -INFINITY && v[i].y == 0.0f ? 0.0f : weight2(v[i].x, M);
                            sum += v[i].x * v[i].y;
                        }
#pragma unroll
                        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                        for (int i = 0; i < kMaxShares / 32; ++i) {
                            if (32 * i >= n) break;
                            if (lane + 32 * i < n) wgt[r * kMaxShares + lane + 32 * i] = v[i].x * inv;
                        }
                        if (p.lse && lane == 0) p.lse[row_of(r)] = sum == 0.0f ? 0.0f : (M + log2f(sum)) * 0.6931471805599453f;
                    }
                    __syncthreads();
                    float4 acc[kNr];
#pragma unroll
                    for (int k = 0; k < kNr; ++k) acc[k] = make_float4(0, 0, 0, 0);
                    for (int i0 = 0; i0 < n; i0 += kGroup) {
                        if (i0 > 0) fetch(i0);
                        cp_async_wait<0>();
                        const int m = min(kGroup, n - i0);
#pragma unroll 8
                        for (int i = 0; i < m; ++i)
#pragma unroll
                            for (int k = 0; k < kNr; ++k) {
                                const float f = wgt[my_row(k) * kMaxShares + i0 + i];
                                const float4 a = *reinterpret_cast<const float4 *>(smem + kStageAt + tid * 16 + (i * kNr + k) * (kThreads * 16));
                                const bool seen = f != 0.0f;  // else whatever is there takes no part
                                acc[k].x = fmaf(f, seen ? a.x : 0.0f, acc[k].x);
                                acc[k].y = fmaf(f, seen ? a.y : 0.0f, acc[k].y);
                                acc[k].z = fmaf(f, seen ? a.z : 0.0f, acc[k].z);
                                acc[k].w = fmaf(f, seen ? a.w : 0.0f, acc[k].w);
                            }
                    }
#pragma unroll
                    for (int k = 0; k < kNr; ++k) {
                        const int r = tid / kDims4 + k * kRowThreads;
                        if (r < rows)
                            *reinterpret_cast<uint2 *>(p.out + row_of(r) * D + d4) =
                                make_uint2(tc::cvt_bf16x2(acc[k].x, acc[k].y), tc::cvt_bf16x2(acc[k].z, acc[k].w));
                    }
                }
            }
        }
        // the next unit of the share
        if (whole) {
            const int64_t u = (int64_t)b * p.Hkv + g + shares;
            if (u >= units) return;
            b = (int)(u / p.Hkv);
            g = (int)(u % p.Hkv);
        } else {
            if (f1 >= r1) return;
            if (++g == p.Hkv) {
                g = 0;
                do ++b;
                while (prefix[b + 1] == prefix[b]);  // a sequence with pages follows: f1 < r1 <= total
            }
        }
        __syncthreads();  // the ring and the merge's scratch are free again
    }
}

// CTAs of a launch: one per SM.
int chunk_rows_ctas(int sms) { return std::min(sms, kMaxShares); }

namespace {
template <int D>
cudaError_t launch_rows_d(const Params &p, int ctas, cudaStream_t s) {
    auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
        if (e != cudaSuccess) return e;
        return launch_overlapped(kernel, dim3(ctas), kThreads, Shape<D>::kSmem, 1, s, p);
    };
    switch ((p.N * p.group + 7) / 8) {
        case 1: return go(chunk_attn_rows<D, 1>);
        case 2: return go(chunk_attn_rows<D, 2>);
        case 3: return go(chunk_attn_rows<D, 3>);
        default: return go(chunk_attn_rows<D, 4>);
    }
}
}  // namespace

cudaError_t launch_chunk_attention_rows(const ChunkAttnArgs &a, cudaStream_t s) {
    Params p{};
    p.q = static_cast<const __nv_bfloat16 *>(a.q);
    p.k = static_cast<const __nv_bfloat16 *>(a.k_pool);
    p.v = static_cast<const __nv_bfloat16 *>(a.v_pool);
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
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.out = static_cast<__nv_bfloat16 *>(a.out);
    p.lse = a.lse;
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.counters = a.counters;
    p.status = a.status;
    return a.D == 128 ? launch_rows_d<128>(p, a.plan.splits, s) : launch_rows_d<64>(p, a.plan.splits, s);
}

}  // namespace a11s
