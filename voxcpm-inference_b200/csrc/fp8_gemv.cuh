// The product of fp8_gemm.cuh for one or two tokens, without tensor cores:
//   y[n][m] = bias[m] + sum_b xs[n][b] ws[m / 128][b] sum_{k in b} x[n][k] w[m][k]
//
// HBM bound on the weights, or, at a few MB, by latency: the tensor path's
// chain (tensor memory, TMA, MMA, a cluster's join) takes 3.5 us before the
// first byte counts.  Here a warp owns kRows outputs: a lane reads 16 codes of
// each of their rows (neighbouring lanes, neighbouring bytes), converts them
// exactly (e4m3 -> f16 -> f32) and adds x * w in fp32; a lane's 16 codes lie in
// one block of 128, so their sum is scaled once.  Lanes are added at the end in
// a fixed order.  Every operand may be what the kernel before wrote while this
// one was already resident, so none is read through the read-only path.
//
// In a graph, against the tensor path: 1 x 1024 -> 4096 2.3 us against 4.5; 1 x
// 4096 -> 4096 5.0 against 6.7; 2 x 1024 -> 4096 2.9 against 4.5.  Longer rows or
// more weights keep the loads of a warp too few: 1 x 8192 -> 8192 19.0 against
// 16.9, and four tokens make its arithmetic count: 4 x 4096 -> 4096 11.6 against
// 6.8.
#pragma once

#include "fp8_gemm.cuh"

namespace vxb {

constexpr int kGemvRows = 2;       // outputs of a warp
constexpr int kGemvThreads = 128;

__device__ __forceinline__ void e4m3x16(uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] >> (16 * h)), __NV_E4M3);
            const float2 p = __half22float2(__half2(r));
            f[4 * i + 2 * h] = p.x;
            f[4 * i + 2 * h + 1] = p.y;
        }
}

// 16 bytes of an operand, in the order of the other volatile instructions (never ahead of
// the wait for the kernel before).
__device__ __forceinline__ uint4 ld_v4(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// NT tokens: args.N == NT.
template <int NT>
__global__ void __launch_bounds__(kGemvThreads) fp8_gemv_kernel(const uint8_t* x, int64_t x_stride, const uint8_t* w,
                                                               int64_t w_stride, const Fp8GemmArgs args) {
    constexpr int RW = kGemvRows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m0 = (blockIdx.x * (kGemvThreads / 32) + warp) * RW;
    grid_dep_sync();
    if (m0 >= args.M) return;
    const uint8_t* wp[RW];
    const float* ws[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) {
        const int m = min(m0 + r, args.M - 1);
        wp[r] = w + m * w_stride;
        ws[r] = args.ws + static_cast<int64_t>(m / 128) * args.kb;
    }
    float acc[RW][NT];
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[r][n] = 0.f;
#pragma unroll 4
    for (int k = lane * 16; k < args.K; k += 512) {
        const int b = k >> 7;
        uint4 wv[RW];
        float sw[RW];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            wv[r] = __ldcs(reinterpret_cast<const uint4*>(wp[r] + k));
            sw[r] = ws[r][b];
        }
        float xf[NT][16], sx[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            e4m3x16(ld_v4(x + n * x_stride + k), xf[n]);
            sx[n] = args.xs[n * args.xs_stride + b];
        }
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float wf[16];
            e4m3x16(wv[r], wf);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float2 p = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                    p = ffma2(make_float2(wf[i], wf[i + 1]), make_float2(xf[n][i], xf[n][i + 1]), p);
                acc[r][n] = fmaf(sx[n] * sw[r], p.x + p.y, acc[r][n]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[r][n] += __shfl_xor_sync(0xffffffffu, acc[r][n], o);
            if (lane == r * NT + n && m0 + r < args.M)
                store_out(args.y, n * args.y_stride + m0 + r, acc[r][n] + (args.bias ? args.bias[m0 + r] : 0.f),
                          args.out_type);
        }
}

}  // namespace vxb
