// linear_skinny.cu - K9 for few rows (single tokens of up to 32 sequences):
// the weights are streamed once, everything else is small.
//
// y[m][n] = act(sum_k x[m][k] W[n][k] ...) as in linear.cu. Bound by HBM: N * K
// weight elements per product; the rows (at most 32) come from L2.
// A block takes 16 or 32 output columns; its warps share the K axis in interleaved
// slices of 128 bytes per weight row and add their sums in shared memory, in
// warp order. With mma.m16n8k16 the 16 weight rows are operand A and 8 rows of
// x operand B: no lane is wasted on absent rows beyond the 8 of a tile, and a
// product of 32 rows costs 4 instructions per 16 x 16 weights. tcgen05 would
// need M = 128 and the weights in shared memory; here they go from HBM straight
// into the registers of the instruction that uses them. That works because the
// order of k inside a slice does not matter as long as A and B agree: a lane
// loads 32 consecutive bytes of its row, and those are its operands of several
// instructions.
// e4m3 values are widened to f16 (exact) for the same instruction: products of
// two e4m3 values are exact in fp32, as are all but the sums.
// Measured (one B200): 1 x 2048 -> 2 x 8192 bf16 12.6 us = 5.3 TB/s (15.4 with 16-byte
// loads and one column tile a block), 32 x 2048 -> 5120 e4m3 7.6 us (9.1 where the
// weights of every call come from HBM), 1 x 8192 -> 2048 bf16 10.1 us. Spills: 24 bytes in
// the e4m3 gated kernel of 25 to 32 rows, 8 in the bf16 one of 9 to 16.
#include <cuda_fp16.h>

#include "epilogue.cuh"
#include "kernels.h"
#include "mma_sync.cuh"

namespace a11s {
namespace {

struct SkinnyParams {
    const uint8_t *x, *weight, *gate;
    const float *x_scale;
    ColumnParams col;
    const __nv_bfloat16 *residual;
    __nv_bfloat16 *out;
    int64_t x_pitch, res_stride, out_stride;  // x: bytes; others: elements
    int32_t rows, k_bytes, N, act;
    StatusWord *status;
};

// Four e4m3 values as two f16 pairs (exact).
__device__ __forceinline__ void widen(uint32_t v, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(v));
}
// 16 bytes of k of weight rows g and g + 8 against 16 bytes of k of 8 rows of x.
template <bool E4M3>
__device__ __forceinline__ void product16(float (&d)[4], const uint4 &w0, const uint4 &w8, const uint4 &x) {
    const uint32_t p[4] = {w0.x, w0.y, w0.z, w0.w}, q[4] = {w8.x, w8.y, w8.z, w8.w}, b[4] = {x.x, x.y, x.z, x.w};
    if constexpr (E4M3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a[4], b0, b1;
            widen(p[i], a[0], a[2]);
            widen(q[i], a[1], a[3]);
            widen(b[i], b0, b1);
            mma16816_f16(d, a, b0, b1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t a[4] = {p[i], q[i], p[i + 1], q[i + 1]};
            mma16816_bf16(d, a, b[i], b[i + 1]);
        }
    }
}
// 32 consecutive bytes, of which those from `left` on are zeros. WIDE: one 32-byte
// access, so that the four lanes of a row ask for a whole 128-byte line at once.
struct Bytes32 {
    uint4 lo, hi;
};
// STREAM: read once (the weights); else kept in L1 (x, which the other blocks of
// the SM read too).
template <bool WIDE, bool STREAM>
__device__ __forceinline__ Bytes32 load32(const uint8_t *p, int left) {
    Bytes32 r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if constexpr (!STREAM) {
        if (left > 0) r.lo = *reinterpret_cast<const uint4 *>(p);
        if (left > 16) r.hi = reinterpret_cast<const uint4 *>(p)[1];
    } else if constexpr (WIDE) {
        if (left > 0)
            asm volatile("ld.global.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(r.lo.x), "=r"(r.lo.y), "=r"(r.lo.z), "=r"(r.lo.w), "=r"(r.hi.x), "=r"(r.hi.y), "=r"(r.hi.z), "=r"(r.hi.w)
                         : "l"(p));
    } else {
        if (left > 0) r.lo = ld_stream(p);
        if (left > 16) r.hi = ld_stream(p + 16);
    }
    return r;
}

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// NT: tiles of 8 rows of x; MT: tiles of 16 weight rows (output columns) of a block.
template <bool E4M3, bool GATED, int NT, int MT, bool WIDE>
__global__ void __launch_bounds__(512) linear_skinny_kernel(const SkinnyParams p) {
    constexpr int P = GATED ? 2 : 1, kCols = 16 * MT;
    extern __shared__ float part[];  // [warps][P][MT][NT][16 columns][8 rows]
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kCols;
    let_next_start();
    wait_before();
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.status) *p.status = StatusWord{0, 0};  // nothing here can fail
    {  // the epilogue's operands into L2 while the weights stream
        const int c = threadIdx.x % kCols, m = threadIdx.x / kCols, n = n0 + c;
        if (n < p.N) {
            if (p.residual && m < p.rows && c == 0) prefetch_l2(p.residual + m * p.res_stride + n);
            if (m == 0 && c % 8 == 0) {
                if (p.col.bias) prefetch_l2(p.col.bias + n);
                if (p.col.w_scale) prefetch_l2(p.col.w_scale + n);
                if (GATED && p.col.g_bias) prefetch_l2(p.col.g_bias + n);
                if (GATED && p.col.g_scale) prefetch_l2(p.col.g_scale + n);
            }
        }
        if (E4M3 && threadIdx.x == 0) prefetch_l2(p.x_scale);
    }
    // this lane's weight rows and NT rows of x; absent ones repeat the last (their results are dropped)
    const uint8_t *w[P][MT][2], *x[NT];
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                w[i][m][h] = (i ? p.gate : p.weight) + (int64_t)min(n0 + 16 * m + g + 8 * h, p.N - 1) * p.k_bytes + 32 * t;
#pragma unroll
    for (int j = 0; j < NT; ++j) x[j] = p.x + (int64_t)min(8 * j + g, p.rows - 1) * p.x_pitch + 32 * t;

    float acc[P][MT][NT][4] = {};
    // slices of 128 bytes of k, 32 bytes a lane; k_bytes is a multiple of 16, so the
    // last slice may end before or within a lane's bytes
#pragma unroll(P * MT * NT <= 2 ? 2 : 1)
    for (int k0 = warp * 128; k0 < p.k_bytes; k0 += warps * 128) {
        const int left = p.k_bytes - k0 - 32 * t;
        Bytes32 a[P][MT][2], b[NT];
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[i][m][h] = load32<WIDE, true>(w[i][m][h] + k0, left);
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = load32<WIDE, false>(x[j] + k0, left);
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    product16<E4M3>(acc[i][m][j], a[i][m][0].lo, a[i][m][1].lo, b[j].lo);
                    product16<E4M3>(acc[i][m][j], a[i][m][0].hi, a[i][m][1].hi, b[j].hi);
                }
    }
    // lane's results: columns 16 m + g and + 8, rows 8 j + 2 t and + 1
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float *d = part + ((((warp * P + i) * MT + m) * NT + j) * 16 + g) * 8 + 2 * t;
                *reinterpret_cast<float2 *>(d) = make_float2(acc[i][m][j][0], acc[i][m][j][1]);
                *reinterpret_cast<float2 *>(d + 64) = make_float2(acc[i][m][j][2], acc[i][m][j][3]);
            }
    __syncthreads();
    for (int o = threadIdx.x; o < NT * 8 * kCols; o += blockDim.x) {
        const int c = o % kCols, m = o / kCols, n = n0 + c;
        if (m >= p.rows || n >= p.N) continue;
        const float *src = part + (((c >> 4) * NT + (m >> 3)) * 16 + (c & 15)) * 8 + (m & 7);
        float s[2] = {0.0f, 0.0f};
#pragma unroll 8
        for (int v = 0; v < warps; ++v)
#pragma unroll
            for (int i = 0; i < P; ++i) s[i] += src[(v * P + i) * MT * NT * 128];
        const float xs = E4M3 ? p.x_scale[m] : 1.0f;
        float y = finish<GATED>(s[0], s[1], xs, column<GATED>(p.col, n), p.act);
        if (p.residual) y += __bfloat162float(p.residual[m * p.res_stride + n]);
        p.out[m * p.out_stride + n] = __float2bfloat16_rn(y);
    }
}

template <bool E4M3, bool GATED, int NT, bool WIDE>
cudaError_t launch_nt(const SkinnyParams &p, cudaStream_t s) {
    // Two column tiles a block where that still gives every SM a block and pays:
    // for a gated product of few rows, gate and weight rows then come in longer runs,
    // and at the rows below x is read half as often; else the registers that a second
    // tile takes cost more. One tile / two, us: gated 2048 -> 8192, bf16 1 row 14.5 / 12.6,
    // 16 rows 16.3 / 15.0, 17 rows 17.7 / 20.3; e4m3 8 rows 9.8 / 8.8, 16 rows 11.1 / 12.5
    // (spills); 2048 -> 5120, bf16 16 rows 6.9 / 8.3, 17 rows 7.2 / 8.9, 25 rows 11.6 /
    // 10.2; e4m3 16 rows 5.3 / 6.1, 17 rows 8.4 / 7.0, 25 rows 8.9 / 9.5. The same side
    // won at K from 1024 to 8192 and N from 5120 to 16384.
    constexpr bool kTwo = GATED ? NT <= (E4M3 ? 1 : 2) : NT == (E4M3 ? 3 : 4);
    const int mt = kTwo && p.N >= 32 * 148 ? 2 : 1;
    const int blocks = (p.N + 16 * mt - 1) / (16 * mt);
    // 8 warps share K; 16 when the blocks do not fill the SMs and K has slices for
    // them (1 x 8192 -> 2048: 10.1 us against 14.7)
    const int warps = blocks < 148 && p.k_bytes >= 16 * 128 ? 16 : 8;
    const size_t smem = (size_t)warps * (GATED ? 2 : 1) * mt * NT * 128 * sizeof(float);
    auto go = [&](auto kernel) {
        if (smem > 48 * 1024) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return e;
        }
        return launch_overlapped(kernel, dim3(blocks), warps * 32, smem, 1, s, p);
    };
    if constexpr (kTwo)
        if (mt == 2) return go(linear_skinny_kernel<E4M3, GATED, NT, 2, WIDE>);
    return go(linear_skinny_kernel<E4M3, GATED, NT, 1, WIDE>);
}
template <bool E4M3, bool GATED>
cudaError_t launch_type(const SkinnyParams &p, cudaStream_t s) {
    auto wide = [](const void *ptr, int64_t pitch) { return (reinterpret_cast<uintptr_t>(ptr) & 31) == 0 && pitch % 32 == 0; };
    const bool w = wide(p.weight, p.k_bytes) && wide(p.gate, 0);
    switch ((p.rows + 7) / 8) {
        case 1: return w ? launch_nt<E4M3, GATED, 1, true>(p, s) : launch_nt<E4M3, GATED, 1, false>(p, s);
        case 2: return w ? launch_nt<E4M3, GATED, 2, true>(p, s) : launch_nt<E4M3, GATED, 2, false>(p, s);
        case 3: return w ? launch_nt<E4M3, GATED, 3, true>(p, s) : launch_nt<E4M3, GATED, 3, false>(p, s);
        default: return w ? launch_nt<E4M3, GATED, 4, true>(p, s) : launch_nt<E4M3, GATED, 4, false>(p, s);
    }
}
}  // namespace

cudaError_t launch_linear_skinny(const LinearArgs &a, cudaStream_t s) {
    const int es = a.e4m3 ? 1 : 2;
    SkinnyParams p{};
    p.x = static_cast<const uint8_t *>(a.x);
    p.weight = static_cast<const uint8_t *>(a.weight);
    p.gate = static_cast<const uint8_t *>(a.gate);
    p.x_scale = a.x_scale;
    p.col = {a.w_scale, a.g_scale, static_cast<const __nv_bfloat16 *>(a.bias), static_cast<const __nv_bfloat16 *>(a.g_bias)};
    p.residual = static_cast<const __nv_bfloat16 *>(a.residual);
    p.out = static_cast<__nv_bfloat16 *>(a.out);
    p.x_pitch = a.x_stride * es;
    p.res_stride = a.res_stride;
    p.out_stride = a.out_stride;
    p.rows = a.rows;
    p.k_bytes = a.K * es;
    p.N = a.N;
    p.act = a.act;
    p.status = a.status;
    if (a.e4m3) return a.gate ? launch_type<true, true>(p, s) : launch_type<true, false>(p, s);
    return a.gate ? launch_type<false, true>(p, s) : launch_type<false, false>(p, s);
}

}  // namespace a11s
