// norm.cu - K8: root-mean-square norm with the residual's addition, output in
// the input's type or in e4m3 with one scale per row.
//
// Per row of `dim` elements, in fp32:
//   h = x + residual                       (h = x without a residual)
//   r = rsqrt(sum(h^2) / dim + eps)
//   y = (h * w) * r
//   scale = max(max|y| / 448, 2^-100), out = e4m3_rn(y / scale)   (e4m3 output)
// The statement pair `h = h + sub_layer(...)`, `_rms_norm(h)` of the reference's
// forward_layer (engine/pipeline.py:403-407, 322-324). Semantics: include/a11spec.h
// (a11s_add_rms_norm).
//
// Bound by HBM: two reads and two writes per element and nothing else of size.
// One pass: a row lives in the registers of its threads between the sums and
// the output, so x and the residual are read once. sum(h^2) and max|h w| are
// reduced together (max|y| = max|h w| * r exactly, since rounding is monotone
// and y is formed in that order), so the e4m3 output costs no second
// reduction. Rows of up to 32 vectors belong to one warp (8 rows a block, no
// block barrier); longer rows to a block of up to 1024 threads with one to four
// 16-byte vectors each.
// Rows of odd length start anywhere, but all tensors' rows at the same distance
// from a 16-byte boundary: the body is moved in vectors from the first boundary
// on, and the up to 2 x 7 elements before and after it by one thread each.
// Where the tensors differ in that distance, every access is one element.
// Measured (one B200): 8190 x 4999 fp32 104 to 109 us = 6.0 to 6.3 TB/s (188 with one element per
// access), 2048 x 2048 bf16 to e4m3 6.9 to 7.0 us, 2048 x 12001 fp32 to e4m3 71 us; one row of
// 2048 2.8 us, which is the host's call.
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"
#include "tc_common.cuh"

namespace a11s {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 0x1p-100f;  // a row whose outputs are all below 448 times this keeps its quotients finite

struct NormParams {
    const void *x, *residual, *weight;
    void *sum, *out;
    float *scales;
    int64_t x_stride, res_stride, sum_stride, out_stride;  // elements
    int32_t rows, dim;
    float eps;
};

// Maximum that keeps a NaN (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// One element. As ld_stream, free to move over the stores, which it never aliases
// before its own element's; not over wait_before().
__device__ __forceinline__ float ld_one(const float *p) {
    float f;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(f) : "l"(p));
    return f;
}
__device__ __forceinline__ float ld_one(const __nv_bfloat16 *p) {
    uint16_t u;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(u) : "l"(p));
    return bf16lo(u);
}
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        f[0] = ld_one(p);
    } else if constexpr (sizeof(T) == 2) {
        const uint4 u = ld_stream(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = bf16lo(w[i]);
            f[2 * i + 1] = bf16hi(w[i]);
        }
    } else {
        const uint4 u = ld_stream(p);
        f[0] = __uint_as_float(u.x);
        f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z);
        f[3] = __uint_as_float(u.w);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(f[0]);
        else *p = f[0];
    } else if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
}
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t *p, const float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        *p = __nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3);
    } else {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
            w[i] = lo | (hi << 16);
        }
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(p) = w[0];
    }
}

// v / scale rounded to nearest, as __fdiv_rn gives it but in four operations, since a
// row's elements share the reciprocal: inv + inv_lo is 1 / scale to 2^-47, so the first
// quotient is off by less than one unit in its last place, and with inv = 1 / scale
// rounded to nearest the correction rounds the quotient correctly (P. Markstein,
// Computation of elementary functions on the IBM RISC System/6000 processor, 1990) -
// as long as no remainder underflows: `scale` within [kFastMin, kFastMax] keeps those
// that can reach an e4m3 value, of v above 2^-10 scale, normal. (Times inv alone, ties
// fall to either side. 2048 x 2048: 7.0 us so, 7.8 with __fdiv_rn, 6.6 times inv.)
constexpr float kFastMin = 0x1p-60f, kFastMax = 0x1p100f;
template <int W>
__device__ __forceinline__ void quotients(float (&v)[W], float scale, float inv, float inv_lo) {
    if constexpr (W == 1) {
        const float q = fmaf(v[0], inv, v[0] * inv_lo);
        v[0] = fmaf(fmaf(q, -scale, v[0]), inv, q);
    } else {
        const float2 neg = make_float2(-scale, -scale), hi = make_float2(inv, inv), lo = make_float2(inv_lo, inv_lo);
#pragma unroll
        for (int e = 0; e < W; e += 2) {
            const float2 a = make_float2(v[e], v[e + 1]);
            const float2 q = tc::ffma2(a, hi, tc::fmul2(a, lo)), d = tc::ffma2(tc::ffma2(q, neg, a), hi, q);
            v[e] = d.x;
            v[e + 1] = d.y;
        }
    }
}

// WARP: a warp per row; otherwise a block per row. NV: vectors a thread holds.
// PEEL: rows start row * x_stride elements (mod VEC) past a vector boundary.
template <typename T, bool E4M3, int VEC, int NV, bool WARP, bool PEEL>
__global__ void __launch_bounds__(WARP ? 256 : 1024) add_rms_norm_kernel(const NormParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
    const int t = WARP ? lane : threadIdx.x, threads = WARP ? 32 : blockDim.x;
    let_next_start();
    wait_before();
    if (WARP && row >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + row * p.res_stride : nullptr;
    const T *wt = static_cast<const T *>(p.weight);
    T *sum = p.sum ? static_cast<T *>(p.sum) + row * p.sum_stride : nullptr;

    // elements [head, head + body) in vectors; `extra`: this thread's one element of the rest, or -1
    int head = 0, body = p.dim, extra = -1;
    if (PEEL) {
        head = min((int)(-(row * p.x_stride) & (VEC - 1)), p.dim);
        body = (p.dim - head) & ~(VEC - 1);
        if (t < head) extra = t;
        else if (t - head < p.dim - head - body) extra = body + t;
    }
    float h[NV][VEC], he = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < body) load_vec<T, VEC>(x + head + c, h[i]);
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[i][e] = 0.0f;
    }
    if (PEEL && extra >= 0) he = (float)x[extra];
    if (res) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * threads + t) * VEC;
            if (c < body) {
                float r[VEC];
                load_vec<T, VEC>(res + head + c, r);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i][e] += r[e];
            }
        }
        if (PEEL && extra >= 0) he += (float)res[extra];
    }
    float ss = 0.0f, mx = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < body) {
            float w[VEC];
            if constexpr (PEEL) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) w[e] = ld_one(wt + head + c + e);
            } else {
                load_vec<T, VEC>(wt + c, w);
            }
            if (sum) store_vec<T, VEC>(sum + head + c, h[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                ss = fmaf(h[i][e], h[i][e], ss);
                h[i][e] *= w[e];
                if (E4M3) mx = max_nan(mx, fabsf(h[i][e]));
            }
        }
    }
    if (PEEL && extra >= 0) {
        const float one[1] = {he};
        if (sum) store_vec<T, 1>(sum + extra, one);
        ss = fmaf(he, he, ss);
        he *= ld_one(wt + extra);
        if (E4M3) mx = max_nan(mx, fabsf(he));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (E4M3) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (!WARP) {
        __shared__ float2 part[32];
        if (lane == 0) part[warp] = make_float2(ss, mx);
        __syncthreads();
        const float2 v = lane < (int)(blockDim.x >> 5) ? part[lane] : make_float2(0.0f, 0.0f);
        ss = v.x;
        mx = v.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (E4M3) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
    }
    const float r = rsqrtf(ss / (float)p.dim + p.eps);
    float scale = 1.0f, inv = 1.0f, inv_lo = 0.0f;
    bool fast = true;
    if (E4M3) {
        scale = mx * r / kE4m3Max;
        if (scale < kMinScale) scale = kMinScale;  // a NaN stays
        inv = __frcp_rn(scale);
        inv_lo = fmaf(-scale, inv, 1.0f) * inv;
        fast = scale >= kFastMin && scale <= kFastMax;
        if (t == 0) p.scales[row] = scale;
    }
    auto put = [&](int c, auto &v) {  // v: VEC or one elements at c
        constexpr int W = sizeof(v) / sizeof(float);
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] *= r;
        if constexpr (E4M3) {
            if (fast) {
                quotients(v, scale, inv, inv_lo);
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e) v[e] = __fdiv_rn(v[e], scale);
            }
        }
        if constexpr (E4M3) store_e4m3<W>(static_cast<uint8_t *>(p.out) + row * p.out_stride + c, v);
        else store_vec<T, W>(static_cast<T *>(p.out) + row * p.out_stride + c, v);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < body) put(head + c, h[i]);
    }
    if (PEEL && extra >= 0) {
        float one[1] = {he};
        put(extra, one);
    }
}

template <typename T, bool E4M3, int VEC, bool PEEL>
cudaError_t launch_vec(const NormParams &p, cudaStream_t s) {
    // values a thread holds: one vector (8 single elements) while 1024 threads
    // cover the row that way, else up to 16 (A11S_NORM_MAX_DIM = 1024 * 16).
    // Holding two or four vectors in fewer threads measured the same at
    // 2048 x 2048 and 1 x 2048 (within 2 %).
    constexpr int kFirst = VEC == 1 ? 8 : 1, kLast = 16 / VEC;
    const int vecs = (p.dim + VEC - 1) / VEC;
    if (vecs <= 32 * kFirst)
        return launch_overlapped(add_rms_norm_kernel<T, E4M3, VEC, kFirst, true, PEEL>, dim3((unsigned)((p.rows + 7ll) / 8)), 256, 0, 1, s, p);
    int nv = kFirst;
    while (vecs > 1024 * nv) nv *= 2;
    const int threads = ((vecs + nv - 1) / nv + 31) / 32 * 32;
    if (nv == kFirst) return launch_overlapped(add_rms_norm_kernel<T, E4M3, VEC, kFirst, false, PEEL>, dim3((unsigned)p.rows), threads, 0, 1, s, p);
    if (nv == 2 * kFirst) return launch_overlapped(add_rms_norm_kernel<T, E4M3, VEC, 2 * kFirst, false, PEEL>, dim3((unsigned)p.rows), threads, 0, 1, s, p);
    if (nv <= kLast) return launch_overlapped(add_rms_norm_kernel<T, E4M3, VEC, kLast, false, PEEL>, dim3((unsigned)p.rows), threads, 0, 1, s, p);
    return cudaErrorInvalidValue;
}

template <typename T, bool E4M3>
cudaError_t launch_type(const NormParams &p, int vec, cudaStream_t s) {
    constexpr int kVec = 16 / (int)sizeof(T);
    if (vec == 2) return launch_vec<T, E4M3, kVec, false>(p, s);
    return vec == 1 ? launch_vec<T, E4M3, kVec, true>(p, s) : launch_vec<T, E4M3, 1, false>(p, s);
}
}  // namespace

cudaError_t launch_add_rms_norm(const NormArgs &a, cudaStream_t s) {
    NormParams p{};
    p.x = a.x;
    p.residual = a.residual;
    p.weight = a.weight;
    p.sum = a.sum;
    p.out = a.out;
    p.scales = a.scales;
    p.x_stride = a.x_stride;
    p.res_stride = a.res_stride;
    p.sum_stride = a.sum_stride;
    p.out_stride = a.out_stride;
    p.rows = a.rows;
    p.dim = a.dim;
    p.eps = a.eps;
    const int es = a.bf16 ? 2 : 4, os = a.e4m3 ? 1 : es, per = 16 / es;
    // 2: rows and lengths in whole vectors; 1: rows of every tensor equally far past a vector boundary; 0: neither
    auto base = [](const void *ptr, int bytes) { return (reinterpret_cast<uintptr_t>(ptr) % bytes) == 0; };
    int vec = 0;
    if (base(a.x, 16) && base(a.residual, 16) && base(a.weight, 16) && base(a.sum, 16) && base(a.out, per * os)) {
        const int64_t d = a.x_stride % per;
        if (a.out_stride % per == d && (!a.residual || a.res_stride % per == d) && (!a.sum || a.sum_stride % per == d))
            vec = d == 0 && a.dim % per == 0 ? 2 : 1;
    }
    if (a.bf16)
        return a.e4m3 ? launch_type<__nv_bfloat16, true>(p, vec, s) : launch_type<__nv_bfloat16, false>(p, vec, s);
    return a.e4m3 ? launch_type<float, true>(p, vec, s) : launch_type<float, false>(p, vec, s);
}

}  // namespace a11s
