// RMS norm of rows with the residual's addition and an optional 8-bit output.
//
//   h = x (+ residual)                        (fp32; also stored, rounded to x's type)
//   y = h / sqrt(mean(h^2) + eps) * w
//   out = y in x's type, or e4m3 codes with one fp32 scale per row and block
//         of 128 channels: scale = max|y| / 448, code = e4m3(y * 448 / max|y|)
//
// HBM bound: per channel one read of x and of the residual, one write of the
// sum and of the output.  One block per row keeps the row in registers
// between the two passes the formula needs (sum of squares, then scaling), so
// every byte moves once; h, the sum of squares and y are fp32, and each
// stored value is rounded once from them.  A thread owns vectors of 8
// consecutive channels, so a block of 128 channels is 16 neighbouring lanes
// and its maximum four shuffles.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace vxb {

constexpr int kScaleBlock = 128;
constexpr float kE4m3Max = 448.f;

struct NormArgs {
    const void* x;
    const void* res;      // null: no residual
    void* sum;            // null: not stored
    const void* w;
    void* y;
    float* scale;         // non-null: e4m3 output
    int64_t N;
    int64_t x_stride, res_stride, sum_stride, y_stride, scale_stride;  // elements between rows
    int C;
    int w_f32;            // weights are fp32 (else x's type)
    float eps;
};

template <typename T>
__device__ __forceinline__ float to_float(T v) {
    return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive elements as fp32; VEC: 16-byte loads (p aligned), else
// element loads of the first n (0..8), the others 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float* v) {
    if (VEC && n == 8) {
        constexpr int kWords = sizeof(T) * 8 / 16;
        uint4 raw[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float(p[i]) : 0.f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float* v) {
    if (VEC && n == 8) {
        constexpr int kWords = sizeof(T) * 8 / 16;
        uint4 raw[kWords];
        T* e = reinterpret_cast<T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_float<T>(v[i]);
    }
}

// Block of any multiple of 32 threads (<= 1024); NV vectors of 8 channels per
// thread: C <= 8 * NV * blockDim.x.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormArgs a) {
    __shared__ float part[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int64_t row = blockIdx.x;
    grid_dep_sync();
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.res ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;

    float h[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + tid) * 8;
        const int n = min(8, a.C - c);
        if (n > 0) {
            load8<T, VEC>(x + c, n, h[j]);
            if (res) {
                float r[8];
                load8<T, VEC>(res + c, n, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[j][i] += r[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[j][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(h[j][i], h[j][i], ss);
    }
    if (a.sum) {
        T* sum = static_cast<T*>(a.sum) + row * a.sum_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + tid) * 8;
            const int n = min(8, a.C - c);
            if (n > 0) store8<T, VEC>(sum + c, n, h[j]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (warps > 1) {
        if (lane == 0) part[warp] = ss;
        __syncthreads();
        ss = lane < warps ? part[lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    const float r = rsqrtf(ss / static_cast<float>(a.C) + a.eps);

#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + tid) * 8;
        const int n = min(8, a.C - c);
        float w[8], y[8];
        if (n > 0) {
            if (a.w_f32) {
                load8<float, VEC>(static_cast<const float*>(a.w) + c, n, w);
            } else {
                load8<T, VEC>(static_cast<const T*>(a.w) + c, n, w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = h[j][i] * r * w[i];
        if (!a.scale) {
            if (n > 0) store8<T, VEC>(static_cast<T*>(a.y) + row * a.y_stride + c, n, y);
            continue;
        }
        // (channels past C: h = w = 0, but r may be inf or NaN)
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, i < n ? fabsf(y[i]) : 0.f);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // A block whose scale would not be a normal fp32 number is all zeros.
        const bool zero = top < kE4m3Max * 1.17549435e-38f;
        const float inv = zero ? 0.f : kE4m3Max / top;
        if (n > 0) {
            if ((lane & 15) == 0) a.scale[row * a.scale_stride + c / kScaleBlock] = zero ? 0.f : top / kE4m3Max;
            uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.y_stride + c;
            uint32_t code[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * p] * inv, y[4 * p + 1] * inv),
                                                             __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * p + 2] * inv, y[4 * p + 3] * inv),
                                                             __NV_SATFINITE, __NV_E4M3);
                code[p] = lo | (hi << 16);
            }
            if (VEC && n == 8) {
                *reinterpret_cast<uint2*>(q) = make_uint2(code[0], code[1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < n) q[i] = static_cast<uint8_t>(code[i >> 2] >> (8 * (i & 3)));
            }
        }
    }
}

}  // namespace vxb
