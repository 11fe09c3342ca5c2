// linear_skinny.cu - K9 for few rows (single tokens of up to 32 sequences):
// the weights are streamed once, everything else is small.
//
// y[m][n] = act(sum_k x[m][k] W[n][k] ...) as in linear.cu. Bound by HBM: N * K
// weight elements per product; the rows (at most 32) come from L2.
// A block takes 16 output columns; its warps share the K axis in interleaved
// slices of 128 bytes per weight row and add their sums in shared memory, in
// warp order. With mma.m16n8k16 the 16 weight rows are operand A and 8 rows of
// x operand B: no lane is wasted on absent rows beyond the 8 of a tile, and a
// product of 32 rows costs 4 instructions per 16 x 16 weights. tcgen05 would
// need M = 128 and the weights in shared memory; here they go from HBM straight
// into the registers of the instruction that uses them. That works because the
// order of k inside a slice does not matter as long as A and B agree: a lane
// loads 16 consecutive bytes of its row, and those are its operands of several
// instructions.
// e4m3 values are widened to f16 (exact) for the same instruction: products of
// two e4m3 values are exact in fp32, as are all but the sums.
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

// NT: tiles of 8 rows of x.
template <bool E4M3, bool GATED, int NT>
__global__ void __launch_bounds__(512) linear_skinny_kernel(const SkinnyParams p) {
    constexpr int P = GATED ? 2 : 1;
    extern __shared__ float part[];  // [warps][P][NT][16 columns][8 rows]
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16;
    let_next_start();
    wait_before();
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.status) *p.status = StatusWord{0, 0};  // nothing here can fail
    // this lane's two weight rows and NT rows of x; absent ones repeat the last (their results are dropped)
    const uint8_t *w[P][2], *x[NT];
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[i][h] = (i ? p.gate : p.weight) + (int64_t)min(n0 + g + 8 * h, p.N - 1) * p.k_bytes;
#pragma unroll
    for (int j = 0; j < NT; ++j) x[j] = p.x + (int64_t)min(8 * j + g, p.rows - 1) * p.x_pitch;

    float acc[P][NT][4] = {};
    // slices of 128 bytes of k, bytes 16 t and 64 + 16 t of each; k_bytes is a
    // multiple of 16, so the last slice may end before a lane's bytes
#pragma unroll(NT <= 2 ? 2 : 1)
    for (int k0 = warp * 128; k0 < p.k_bytes; k0 += warps * 128) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        uint4 a[P][2][2], b[NT][2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int k = k0 + 64 * c + 16 * t;
            const bool in = k < p.k_bytes;
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[i][h][c] = in ? ldg_stream(w[i][h] + k) : zero;
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j][c] = in ? __ldg(reinterpret_cast<const uint4 *>(x[j] + k)) : zero;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) product16<E4M3>(acc[i][j], a[i][0][c], a[i][1][c], b[j][c]);
    }
    // lane's results: columns n0 + g and n0 + g + 8, rows 8 j + 2 t and + 1
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float *d = part + (((warp * P + i) * NT + j) * 16 + g) * 8 + 2 * t;
            d[0] = acc[i][j][0];
            d[1] = acc[i][j][1];
            d[64] = acc[i][j][2];
            d[65] = acc[i][j][3];
        }
    __syncthreads();
    for (int o = threadIdx.x; o < NT * 128; o += blockDim.x) {
        const int c = o & 15, m = o >> 4, n = n0 + c;
        if (m >= p.rows || n >= p.N) continue;
        const float *src = part + ((m >> 3) * 16 + c) * 8 + (m & 7);
        float s[2] = {0.0f, 0.0f};
        for (int v = 0; v < warps; ++v)
#pragma unroll
            for (int i = 0; i < P; ++i) s[i] += src[(v * P + i) * NT * 128];
        const float xs = E4M3 ? __ldg(p.x_scale + m) : 1.0f;
        float y = finish<GATED>(s[0], s[1], xs, column<GATED>(p.col, n), p.act);
        if (p.residual) y += __bfloat162float(p.residual[m * p.res_stride + n]);
        p.out[m * p.out_stride + n] = __float2bfloat16_rn(y);
    }
}

template <bool E4M3, bool GATED>
cudaError_t launch_nt(const SkinnyParams &p, cudaStream_t s) {
    const int nt = (p.rows + 7) / 8, blocks = (p.N + 15) / 16;
    // 8 warps share K; 16 when the blocks alone do not fill the SMs and K has slices for them
    const int warps = blocks < 148 && p.k_bytes >= 16 * 256 ? 16 : 8;
    const size_t smem = (size_t)warps * (GATED ? 2 : 1) * nt * 128 * sizeof(float);
    auto go = [&](auto kernel) {
        if (smem > 48 * 1024) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return e;
        }
        return launch_overlapped(kernel, dim3(blocks), warps * 32, smem, 1, s, p);
    };
    switch (nt) {
        case 1: return go(linear_skinny_kernel<E4M3, GATED, 1>);
        case 2: return go(linear_skinny_kernel<E4M3, GATED, 2>);
        case 3: return go(linear_skinny_kernel<E4M3, GATED, 3>);
        default: return go(linear_skinny_kernel<E4M3, GATED, 4>);
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
    if (a.e4m3) return a.gate ? launch_nt<true, true>(p, s) : launch_nt<true, false>(p, s);
    return a.gate ? launch_nt<false, true>(p, s) : launch_nt<false, false>(p, s);
}

}  // namespace a11s
