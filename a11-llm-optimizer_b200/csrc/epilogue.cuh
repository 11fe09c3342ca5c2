// epilogue.cuh - what the linear kernels (K9) apply to an accumulator: the
// e4m3 scales, bias, activation and gate, in fp32.
#pragma once
#include "common.cuh"

namespace a11s {

// Below v = -87.3 the denominator passes 2^126 and the quotient is 0 (of y above -2^-119).
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
// v Phi(v) with Phi(-|v|) = exp(-v^2 / 2) erfcx(|v| / sqrt(2)) / 2, where erfcx(z) =
// exp(z^2) erfc(z) is a polynomial in t = 1 / (1 + 0.38 z) (the form of Hastings'
// approximations; own least-squares fit, reweighted towards the least relative
// error: 2.2e-8 on [0, 12]). Without branches, so that the columns of a step run
// side by side: erff, with its two ranges, took 300 cycles a column in a warp
// that has its scheduler to itself. Relative error in fp32 below 1.0e-6 for v > -4
// and 2.1e-6 down to -6, where v Phi(v) is 6e-9.
__device__ __forceinline__ float gelu(float v) {
    const float t = __fdividef(1.0f, fmaf(0.26870057f, fabsf(v), 1.0f));
    float r = 0.0590475053f;
    r = fmaf(r, t, -0.262688488f);
    r = fmaf(r, t, 0.364739329f);
    r = fmaf(r, t, -0.162510931f);
    r = fmaf(r, t, 0.230789483f);
    r = fmaf(r, t, 0.138305649f);
    r = fmaf(r, t, 0.204000324f);
    r = fmaf(r, t, 0.213905275f);
    r = fmaf(r, t, 0.214411855f);
    const float q = 0.5f * t * r * exp2f(v * v * -0.72134752f);
    return v * (v < 0.0f ? q : 1.0f - q);
}

__device__ __forceinline__ float activate(float v, int act) {
    return act == A11S_ACT_SILU ? silu(v) : act == A11S_ACT_GELU ? gelu(v) : v;
}

struct ColumnParams {  // per output column, nullable
    const float *w_scale, *g_scale;
    const __nv_bfloat16 *bias, *g_bias;
    __host__ __device__ bool any() const { return w_scale || bias || g_bias; }
};
struct Column {
    float w_scale, bias, g_scale, g_bias;
};
template <bool GATED>
__device__ __forceinline__ Column column(const ColumnParams &p, int n) {
    Column c{1.0f, 0.0f, 1.0f, 0.0f};
    if (p.w_scale) c.w_scale = p.w_scale[n];
    if (p.bias) c.bias = __bfloat162float(p.bias[n]);
    if (GATED) {
        if (p.g_scale) c.g_scale = p.g_scale[n];
        if (p.g_bias) c.g_bias = __bfloat162float(p.g_bias[n]);
    }
    return c;
}
// One output before the residual: the accumulator (and, gated, the gate's)
// with scales and biases.
template <bool GATED>
__device__ __forceinline__ float finish(float acc, float gacc, float x_scale, const Column &c, int act) {
    const float v = fmaf(acc, x_scale * c.w_scale, c.bias);
    if (!GATED) return activate(v, act);
    return activate(fmaf(gacc, x_scale * c.g_scale, c.g_bias), act) * v;
}

// Columns of a tile in shared memory ([w_scale | bias | g_scale | g_bias] of
// COLS each), read by whole warps at one column: broadcasts.
template <bool GATED, int COLS>
__device__ __forceinline__ void stage_columns(float *sc, const ColumnParams &p, int n0, int N, int i, int threads) {
    for (; i < COLS; i += threads) {
        Column c{1.0f, 0.0f, 1.0f, 0.0f};
        if (n0 + i < N) c = column<GATED>(p, n0 + i);
        sc[i] = c.w_scale;
        sc[COLS + i] = c.bias;
        if (GATED) {
            sc[2 * COLS + i] = c.g_scale;
            sc[3 * COLS + i] = c.g_bias;
        }
    }
}
// W values of consecutive columns at c0 (a multiple of 4), in place in v; u: the gate's accumulators.
template <bool GATED, int COLS, int W>
__device__ __forceinline__ void finish_columns(float (&v)[W], const float *u, float xs, const float *sc, int c0, bool params, int act) {
    if (params) {
#pragma unroll
        for (int e = 0; e < W; e += 4) {
            const float4 s = *reinterpret_cast<const float4 *>(sc + c0 + e), b = *reinterpret_cast<const float4 *>(sc + COLS + c0 + e);
            v[e] = fmaf(v[e], xs * s.x, b.x);
            v[e + 1] = fmaf(v[e + 1], xs * s.y, b.y);
            v[e + 2] = fmaf(v[e + 2], xs * s.z, b.z);
            v[e + 3] = fmaf(v[e + 3], xs * s.w, b.w);
        }
    }
    if constexpr (GATED) {
#pragma unroll
        for (int e = 0; e < W; e += 4) {
            float g[4] = {u[e], u[e + 1], u[e + 2], u[e + 3]};
            if (params) {
                const float4 s = *reinterpret_cast<const float4 *>(sc + 2 * COLS + c0 + e),
                             b = *reinterpret_cast<const float4 *>(sc + 3 * COLS + c0 + e);
                g[0] = fmaf(g[0], xs * s.x, b.x);
                g[1] = fmaf(g[1], xs * s.y, b.y);
                g[2] = fmaf(g[2], xs * s.z, b.z);
                g[3] = fmaf(g[3], xs * s.w, b.w);
            }
            if (act == A11S_ACT_SILU) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[e + i] *= silu(g[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[e + i] *= activate(g[i], act);
            }
        }
    } else if (act != A11S_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = activate(v[e], act);
    }
}

}  // namespace a11s
