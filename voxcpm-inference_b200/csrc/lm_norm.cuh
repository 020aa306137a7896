// RMS norm of rows with the residual's addition and an optional 8-bit output.
//
//   h = x (+ residual)                        (fp32; also stored, rounded to x's type)
//   y = h / sqrt(mean(h^2) + eps) * w
//   out = y in x's type, or e4m3 codes with one fp32 scale per row and block
//         of 128 channels: scale = max|y| / 448, code = e4m3(y / scale)
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

// Two consecutive elements as fp32.
template <typename T>
__device__ __forceinline__ float2 pair_of(const T* e) {
    return make_float2(to_float(e[0]), to_float(e[1]));
}
template <>
__device__ __forceinline__ float2 pair_of<__nv_bfloat16>(const __nv_bfloat16* e) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(e);  // a bf16 is an fp32's upper half
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Eight consecutive elements as fp32, those from n on 0.  VEC: 16-byte loads (p
// aligned; n is 8, or at most 0).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float* v) {
    if (VEC) {
        constexpr int kWords = sizeof(T) * 8 / 16;
        uint4 raw[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = n > 0 ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
        const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(v + 2 * i) = pair_of<T>(e + 2 * i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float(p[i]) : 0.f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float* v) {
    if (VEC) {
        constexpr int kWords = sizeof(T) * 8 / 16;
        uint4 raw[kWords];
        T* e = reinterpret_cast<T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
        if (n <= 0) return;
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_float<T>(v[i]);
    }
}

// Block of any multiple of 32 threads (<= 1024); NV vectors of 8 channels per
// thread: C <= 8 * NV * blockDim.x.  VEC: C % 8 == 0 and every row is 16-byte
// aligned.  The kernel was bound by instructions when it tested every element
// and divided each: with packed fp32 arithmetic and one reciprocal per block of
// 128 the 16384 x 4096 bf16 case went from 106 to 73 us in a graph (6.45 TB/s; 80
// us, 5.9 TB/s, a call among others; 72 us at the measured copy rate).
template <typename T, int NV, bool VEC, bool RES, bool Q8>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormArgs a) {
    __shared__ float part[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int64_t row = blockIdx.x;
    grid_dep_sync();
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = RES ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;

    float2 h[NV][4], ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + tid) * 8;
        float v[8];
        load8<T, VEC>(x + c, min(8, a.C - c), v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[j][i] = make_float2(v[2 * i], v[2 * i + 1]);
    }
    if (RES) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + tid) * 8;
            float v[8];
            load8<T, VEC>(res + c, min(8, a.C - c), v);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[j][i].x += v[2 * i], h[j][i].y += v[2 * i + 1];
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = ffma2(h[j][i], h[j][i], ss);
    if (a.sum) {
        T* sum = static_cast<T*>(a.sum) + row * a.sum_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + tid) * 8;
            store8<T, VEC>(sum + c, min(8, a.C - c), reinterpret_cast<const float*>(h[j]));
        }
    }
    // (the weights are here when the sum is)
    float w[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + tid) * 8;
        if (a.w_f32) {
            load8<float, VEC>(static_cast<const float*>(a.w) + c, min(8, a.C - c), w[j]);
        } else {
            load8<T, VEC>(static_cast<const T*>(a.w) + c, min(8, a.C - c), w[j]);
        }
    }
    float all = ss.x + ss.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (warps > 1) {
        if (lane == 0) part[warp] = all;
        __syncthreads();
        all = lane < warps ? part[lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    const float r = rsqrtf(all / static_cast<float>(a.C) + a.eps);
    const float2 rr = make_float2(r, r);

#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + tid) * 8;
        const int n = min(8, a.C - c);
        float2 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = fmul2(fmul2(h[j][i], rr), make_float2(w[j][2 * i], w[j][2 * i + 1]));
        if (!Q8) {
            store8<T, VEC>(static_cast<T*>(a.y) + row * a.y_stride + c, n, reinterpret_cast<const float*>(y));
            continue;
        }
        // (channels past C: h = w = 0, but r may be inf or NaN; the maximum ignores NaN)
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(y[i].x), fabsf(y[i].y)));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // A block whose scale would not be a normal fp32 number is all zeros.
        const bool zero = top < kE4m3Max * 1.17549435e-38f;
        const float s = zero ? 0.f : top * (1.f / kE4m3Max);
        if (n <= 0) continue;
        if ((lane & 15) == 0) a.scale[row * a.scale_stride + c / kScaleBlock] = s;
        // y / s as the product with the reciprocal, itself rounded once by a Newton step: at most one
        // ulp from the quotient (correcting that too, two packed FMAs more, took the case above from
        // 73.1 to 75.2 us).  (s is below 2^126, where __fdividef ends, and an infinite s gives 0.)
        float inv = zero ? 0.f : __fdividef(1.f, s);
        inv = fmaf(fmaf(isinf(s) ? 0.f : -s, inv, 1.f), inv, inv);
        const float2 iv = make_float2(inv, inv);
        uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.y_stride + c;
        uint32_t code[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(fmul2(y[2 * p], iv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(fmul2(y[2 * p + 1], iv), __NV_SATFINITE, __NV_E4M3);
            code[p] = lo | (hi << 16);
        }
        if (VEC) {
            *reinterpret_cast<uint2*>(q) = make_uint2(code[0], code[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) q[i] = static_cast<uint8_t>(code[i >> 2] >> (8 * (i & 3)));
        }
    }
}

}  // namespace vxb
