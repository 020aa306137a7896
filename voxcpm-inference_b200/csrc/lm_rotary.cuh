// Rotary positions: the first R dims of every query and key head are rotated
// in pairs (a, b) by the angle position * inv_freq[i]:
//   a' = (a cos - b sin) * factor, b' = (b cos + a sin) * factor,
// pair i being dims (i, i + R/2) ("half" layout) or (2i, 2i + 1)
// ("interleaved"); dims R.. of a head are copied.  Optionally the rotated keys
// and the values go straight to a paged cache.
//
// The angle is formed in fp64, in turns: position * inv_freq exceeds 2^24
// steps of fp32 in long contexts, where an fp32 product has lost the fraction
// of a turn that the result depends on.  After the nearest whole turn is
// subtracted the rest is rounded to fp32 (error below 2^-25 turns).
//
// HBM bound: q, k, v read and written once.  A block computes its tokens'
// sines and cosines once into shared memory, for all heads; then every thread
// moves 16-byte vectors (VEC elements; element by element where a stride or an
// extent does not allow it).
#pragma once

#include "lm_norm.cuh"

namespace vxb {

constexpr int kRotTokens = 8;    // tokens per block at most
constexpr int kRotMaxR = 256;
constexpr int kRotThreads = 256;

struct HeadsView {               // [N][heads][D], D contiguous
    void* p;
    int64_t token, head;         // strides in elements
};

struct RotaryArgs {
    HeadsView q, q_out, k, k_out, v;  // k.p null: no keys; v.p null: no values
    const int64_t* positions;    // [N]
    const float* inv_freq;       // [R / 2]
    // paged cache (slots non-null): token n's key and value at page slots[n] / page_size,
    // place slots[n] % page_size; a slot outside [0, pages * page_size) is skipped
    const int64_t* slots;
    void* k_cache;
    void* v_cache;
    int64_t cache_slots, page_stride, slot_stride, cache_head;
    int page_size;
    int64_t N;
    int Hq, Hk, D, R;
    int tokens;                  // tokens per block
    float factor;
};

template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
    __shared__ float2 cs[kRotTokens][kRotMaxR / 2];
    __shared__ int64_t slot_off[kRotTokens];  // cache offset of the token, -1 if none
    const int half = a.R / 2;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * a.tokens;
    const int nt = static_cast<int>(min(static_cast<int64_t>(a.tokens), a.N - n0));
    grid_dep_sync();
    for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
        const int t = i / half, f = i - t * half;
        const double turns = static_cast<double>(a.positions[n0 + t]) * static_cast<double>(a.inv_freq[f]) *
                             (1.0 / (2.0 * kPi));
        const float r = static_cast<float>(turns - rint(turns));
        float s, c;
        sincospif(2.f * r, &s, &c);
        cs[t][f] = make_float2(c * a.factor, s * a.factor);
    }
    if (a.slots && threadIdx.x < nt) {
        const int64_t s = a.slots[n0 + threadIdx.x];
        slot_off[threadIdx.x] = s >= 0 && s < a.cache_slots
                                    ? (s / a.page_size) * a.page_stride + (s % a.page_size) * a.slot_stride
                                    : -1;
    }
    __syncthreads();

    // Items of a token: per rotated head the pair items, then the rest of the
    // head; then the values.  A half-layout pair item is two vectors of VEC
    // dims (i.., i + R/2..), an interleaved one a vector of max(VEC, 2) dims.
    constexpr int kStep = INTER ? (VEC > 1 ? VEC : 2) : VEC;
    const int pair_items = INTER ? a.R / kStep : half / kStep;
    const int head_items = pair_items + (a.D - a.R) / VEC;
    const int heads = a.Hq + (a.k.p ? a.Hk : 0);
    const int v_items = a.v.p ? a.D / VEC : 0;
    const int rot_items = heads * head_items;
    const int items = rot_items + a.Hk * v_items;
    for (int w = threadIdx.x; w < nt * items; w += blockDim.x) {
        const int t = w / items;
        int i = w - t * items;
        const int64_t n = n0 + t;
        const T* src;
        T* dst;
        if (i < rot_items) {
            int h = i / head_items;
            i -= h * head_items;
            if (h < a.Hq) {
                src = static_cast<const T*>(a.q.p) + n * a.q.token + h * a.q.head;
                dst = static_cast<T*>(a.q_out.p) + n * a.q_out.token + h * a.q_out.head;
            } else {
                h -= a.Hq;
                src = static_cast<const T*>(a.k.p) + n * a.k.token + h * a.k.head;
                if (a.slots) {
                    if (slot_off[t] < 0) continue;
                    dst = static_cast<T*>(a.k_cache) + slot_off[t] + h * a.cache_head;
                } else {
                    dst = static_cast<T*>(a.k_out.p) + n * a.k_out.token + h * a.k_out.head;
                }
            }
            if (i < pair_items) {
                if (INTER) {
                    T e[kStep], o[kStep];
                    const int d = i * kStep;
                    if (VEC > 1) {
                        *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(src + d);
                    } else {
#pragma unroll
                        for (int j = 0; j < kStep; ++j) e[j] = src[d + j];
                    }
#pragma unroll
                    for (int j = 0; j < kStep / 2; ++j) {
                        const float2 c = cs[t][d / 2 + j];
                        const float x = to_float(e[2 * j]), y = to_float(e[2 * j + 1]);
                        o[2 * j] = from_float<T>(x * c.x - y * c.y);
                        o[2 * j + 1] = from_float<T>(y * c.x + x * c.y);
                    }
                    if (VEC > 1) {
                        *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(o);
                    } else {
#pragma unroll
                        for (int j = 0; j < kStep; ++j) dst[d + j] = o[j];
                    }
                } else {
                    T e[2][VEC], o[2][VEC];
                    const int d = i * VEC;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        if (VEC > 1) {
                            *reinterpret_cast<uint4*>(e[s]) = *reinterpret_cast<const uint4*>(src + d + s * half);
                        } else {
                            e[s][0] = src[d + s * half];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float2 c = cs[t][d + j];
                        const float x = to_float(e[0][j]), y = to_float(e[1][j]);
                        o[0][j] = from_float<T>(x * c.x - y * c.y);
                        o[1][j] = from_float<T>(y * c.x + x * c.y);
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        if (VEC > 1) {
                            *reinterpret_cast<uint4*>(dst + d + s * half) = *reinterpret_cast<const uint4*>(o[s]);
                        } else {
                            dst[d + s * half] = o[s][0];
                        }
                    }
                }
                continue;
            }
            i = i - pair_items;
            src += a.R;
            dst += a.R;
        } else {
            i -= rot_items;
            const int h = i / v_items;
            i -= h * v_items;
            if (slot_off[t] < 0) continue;
            src = static_cast<const T*>(a.v.p) + n * a.v.token + h * a.v.head;
            dst = static_cast<T*>(a.v_cache) + slot_off[t] + h * a.cache_head;
        }
        if (VEC > 1) {
            reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
        } else {
            dst[i] = src[i];
        }
    }
}

}  // namespace vxb
