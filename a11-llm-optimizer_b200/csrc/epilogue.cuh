// epilogue.cuh - what the linear kernels (K9) apply to an accumulator: the
// e4m3 scales, bias, activation and gate, in fp32.
#pragma once
#include "common.cuh"

namespace a11s {

__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
__device__ __forceinline__ float gelu(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f)); }

__device__ __forceinline__ float activate(float v, int act) {
    return act == A11S_ACT_SILU ? silu(v) : act == A11S_ACT_GELU ? gelu(v) : v;
}

// One output before the residual: acc (and, gated, the gate's accumulator)
// with their scales and biases.
struct Column {
    float w_scale, g_scale, bias, g_bias;
};
template <bool GATED>
__device__ __forceinline__ float finish(float acc, float gacc, float x_scale, const Column &c, int act) {
    const float v = fmaf(acc, x_scale * c.w_scale, c.bias);
    if (!GATED) return activate(v, act);
    return activate(fmaf(gacc, x_scale * c.g_scale, c.g_bias), act) * v;
}

struct ColumnParams {
    const float *w_scale, *g_scale;
    const __nv_bfloat16 *bias, *g_bias;
};
template <bool GATED>
__device__ __forceinline__ Column column(const ColumnParams &p, int n) {
    Column c{1.0f, 1.0f, 0.0f, 0.0f};
    if (p.w_scale) c.w_scale = __ldg(p.w_scale + n);
    if (p.bias) c.bias = __bfloat162float(__ldg(p.bias + n));
    if (GATED) {
        if (p.g_scale) c.g_scale = __ldg(p.g_scale + n);
        if (p.g_bias) c.g_bias = __bfloat162float(__ldg(p.g_bias + n));
    }
    return c;
}

}  // namespace a11s
