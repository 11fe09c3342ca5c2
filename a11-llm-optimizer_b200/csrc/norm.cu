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
// block barrier); longer rows to a block of 128 to 1024 threads, wide enough
// that a thread holds one 16-byte vector where the row allows it (at most 16 values).
// Rows whose start or length is not a multiple of 16 bytes take the same
// kernel with one element per access: a warp still covers consecutive bytes.
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace a11s {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 0x1p-100f;  // keeps 1 / scale finite; a row that small is all zeros but for its scale

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

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        f[0] = (float)__ldg(p);
    } else if constexpr (sizeof(T) == 2) {
        const uint4 u = ldg_stream(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = bf16lo(w[i]);
            f[2 * i + 1] = bf16hi(w[i]);
        }
    } else {
        const uint4 u = ldg_stream(p);
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

// WARP: a warp per row; otherwise a block per row. NV: vectors a thread holds.
template <typename T, bool E4M3, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) add_rms_norm_kernel(const NormParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
    const int t = WARP ? lane : threadIdx.x, threads = WARP ? 32 : blockDim.x;
    if (WARP && row >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + row * p.res_stride : nullptr;
    const T *wt = static_cast<const T *>(p.weight);

    float h[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < p.dim) load_vec<T, VEC>(x + c, h[i]);
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[i][e] = 0.0f;
    }
    if (res) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * threads + t) * VEC;
            if (c < p.dim) {
                float r[VEC];
                load_vec<T, VEC>(res + c, r);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i][e] += r[e];
            }
        }
    }
    float ss = 0.0f, mx = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < p.dim) {
            if (p.sum) store_vec<T, VEC>(static_cast<T *>(p.sum) + row * p.sum_stride + c, h[i]);
            float w[VEC];
            load_vec<T, VEC>(wt + c, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                ss = fmaf(h[i][e], h[i][e], ss);
                h[i][e] *= w[e];
                if (E4M3) mx = max_nan(mx, fabsf(h[i][e]));
            }
        }
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
    float inv = 1.0f;
    if (E4M3) {
        float scale = mx * r / kE4m3Max;
        if (scale < kMinScale) scale = kMinScale;  // a NaN stays
        inv = 1.0f / scale;
        if (t == 0) p.scales[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * threads + t) * VEC;
        if (c < p.dim) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[i][e] *= r;
                if (E4M3) h[i][e] *= inv;
            }
            if constexpr (E4M3) store_e4m3<VEC>(static_cast<uint8_t *>(p.out) + row * p.out_stride + c, h[i]);
            else store_vec<T, VEC>(static_cast<T *>(p.out) + row * p.out_stride + c, h[i]);
        }
    }
}

template <typename T, bool E4M3, int VEC>
cudaError_t launch_vec(const NormParams &p, cudaStream_t s) {
    // values a thread holds: one vector (8 single elements) while 1024 threads
    // cover the row, else 16 (A11S_NORM_MAX_DIM = 1024 * 16)
    constexpr int kFirst = VEC == 1 ? 8 : 1, kLast = 16 / VEC;
    const int vecs = (p.dim + VEC - 1) / VEC;
    if (vecs <= 32 * kFirst) {
        add_rms_norm_kernel<T, E4M3, VEC, kFirst, true><<<(unsigned)((p.rows + 7ll) / 8), 256, 0, s>>>(p);
        return cudaGetLastError();
    }
    int threads = 128;
    while (threads < 1024 && threads * kFirst < vecs) threads *= 2;
    const int nv = (vecs + threads - 1) / threads;
    if (nv <= kFirst) add_rms_norm_kernel<T, E4M3, VEC, kFirst, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
    else if (nv <= 2 * kFirst) add_rms_norm_kernel<T, E4M3, VEC, 2 * kFirst, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
    else if (nv <= kLast) add_rms_norm_kernel<T, E4M3, VEC, kLast, false><<<(unsigned)p.rows, threads, 0, s>>>(p);
    else return cudaErrorInvalidValue;
    return cudaGetLastError();
}

template <typename T, bool E4M3>
cudaError_t launch_type(const NormParams &p, bool vec, cudaStream_t s) {
    return vec ? launch_vec<T, E4M3, 16 / (int)sizeof(T)>(p, s) : launch_vec<T, E4M3, 1>(p, s);
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
    auto ok = [](const void *ptr, int64_t stride, int size, int bytes) {
        return (reinterpret_cast<uintptr_t>(ptr) % bytes) == 0 && (stride * size) % bytes == 0;
    };
    const bool vec = a.dim % per == 0 && ok(a.x, a.x_stride, es, 16) && ok(a.residual, a.res_stride, es, 16) &&
                     ok(a.weight, 0, es, 16) && ok(a.sum, a.sum_stride, es, 16) &&
                     ok(a.out, a.out_stride, os, per * os);
    if (a.bf16)
        return a.e4m3 ? launch_type<__nv_bfloat16, true>(p, vec, s) : launch_type<__nv_bfloat16, false>(p, vec, s);
    return a.e4m3 ? launch_type<float, true>(p, vec, s) : launch_type<float, false>(p, vec, s);
}

}  // namespace a11s
