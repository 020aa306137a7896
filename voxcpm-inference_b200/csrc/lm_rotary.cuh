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
// sines and cosines once into shared memory, for all heads; small blocks (128
// threads, 4 tokens) so that others move data meanwhile (16381 tokens of 32 + 16
// heads of 128: 68 us, 5.9 TB/s, in a graph, 71 us a call among others; 256 threads and 8 tokens with four vectors in
// flight a thread 76 us, with two 69 us, 2 tokens 91 us).  Then every thread
// moves 16-byte vectors (VEC elements; element by element where a stride or an
// extent does not allow it).
#pragma once

#include "lm_norm.cuh"

namespace vxb {

constexpr int kRotTokens = 4;    // tokens per block at most
constexpr int kRotMaxR = 256;
constexpr int kRotThreads = 128;

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

// VEC elements moved at once: 16 bytes, or one element.
template <typename T, int VEC>
struct VecOf {
    using type = uint4;
};
template <typename T>
struct VecOf<T, 1> {
    using type = T;
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

    // Items: (token, head, place in the head).  A half-layout pair item is two
    // vectors of VEC dims (i.. and i + R/2..), an interleaved one a vector of
    // max(VEC, 2) dims, an item of the rest of a head a vector of VEC; a value
    // head is walked alike and only copied.  A thread steps through its items
    // by adding the block's stride in these three digits: no divisions.
    constexpr int kStep = INTER ? (VEC > 1 ? VEC : 2) : VEC;
    constexpr int kLoads = INTER ? (VEC > 1 ? 1 : 2) : 2;  // vectors of an item
    constexpr int kAhead = 2;                              // items whose loads are in flight
    using V = typename VecOf<T, VEC>::type;
    const int pair_items = INTER ? a.R / kStep : half / kStep;
    const int head_items = pair_items + (a.D - a.R) / VEC;
    const int rot_heads = a.Hq + (a.k.p ? a.Hk : 0);
    const int heads = rot_heads + (a.v.p ? a.Hk : 0);
    const int stride_i = blockDim.x % head_items, stride_h = blockDim.x / head_items % heads,
              stride_t = blockDim.x / head_items / heads;
    int i = threadIdx.x % head_items, h = threadIdx.x / head_items % heads, t = threadIdx.x / head_items / heads;
    while (t < nt) {
        V e[kAhead][kLoads];
        T* dst[kAhead];
        int at[kAhead];   // place in the head, -1: nothing to do
        const float2* c[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            at[u] = -1;
            if (t < nt) {
                const int64_t n = n0 + t;
                const T* src;
                if (h < a.Hq) {
                    src = static_cast<const T*>(a.q.p) + n * a.q.token + h * a.q.head;
                    dst[u] = static_cast<T*>(a.q_out.p) + n * a.q_out.token + h * a.q_out.head;
                    at[u] = i;
                } else {
                    const bool key = h < rot_heads;
                    const int hk = h - (key ? a.Hq : rot_heads);
                    const HeadsView& in = key ? a.k : a.v;
                    src = static_cast<const T*>(in.p) + n * in.token + hk * in.head;
                    if (a.slots) {
                        dst[u] = static_cast<T*>(key ? a.k_cache : a.v_cache) + slot_off[t] + hk * a.cache_head;
                        if (slot_off[t] >= 0) at[u] = i;
                    } else {
                        dst[u] = static_cast<T*>(a.k_out.p) + n * a.k_out.token + hk * a.k_out.head;
                        at[u] = i;
                    }
                }
                // where the item lies, and its angles (null: copied)
                const bool pair = i < pair_items;
                const int d = pair ? i * kStep : a.R + (i - pair_items) * VEC;
                src += d;
                dst[u] += d;
                c[u] = pair && h < rot_heads ? &cs[t][INTER ? d / 2 : d] : nullptr;
                if (at[u] >= 0) {
                    at[u] = pair ? 1 : 0;
                    e[u][0] = *reinterpret_cast<const V*>(src);
                    if (kLoads > 1 && pair) e[u][kLoads - 1] = *reinterpret_cast<const V*>(src + (INTER ? 1 : half));
                }
            }
            i += stride_i;
            h += stride_h;
            t += stride_t;
            if (i >= head_items) i -= head_items, ++h;
            if (h >= heads) h -= heads, ++t;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (at[u] < 0) continue;
            if (c[u]) {
                T* v = reinterpret_cast<T*>(e[u]);
                constexpr int kPairs = INTER ? kStep / 2 : VEC;
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    T* x = INTER ? v + 2 * j : v + j;
                    T* y = INTER ? v + 2 * j + 1 : v + VEC + j;
                    const float2 r = c[u][j];
                    const float p = to_float(*x), q = to_float(*y);
                    *x = from_float<T>(p * r.x - q * r.y);
                    *y = from_float<T>(q * r.x + p * r.y);
                }
            }
            *reinterpret_cast<V*>(dst[u]) = e[u][0];
            if (kLoads > 1 && at[u] > 0) *reinterpret_cast<V*>(dst[u] + (INTER ? 1 : half)) = e[u][kLoads - 1];
        }
    }
}

}  // namespace vxb
