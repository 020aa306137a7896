// Attention of long chunks of new tokens over a paged cache, on the
// 5th-generation tensor cores (the same operator as paged_attn.cuh).
//
// A block takes two tiles of 128 query rows (row = token * GT + head of the
// group, as in paged_attn.cuh) and walks the keys in steps of 128:
//   S = Q K^T  (tcgen05.mma kind::f16, 128 x 128, fp32 in TMEM)
//   P = exp2(S * scale * log2(e) - m), rounded to the cache's type, written
//       over S in TMEM (two values a column)
//   O += P V   (A operand from TMEM, fp32 accumulator in TMEM)
// A warpgroup owns a tile's softmax, one row per thread: the maximum and the
// sum need no exchange.  While one tile's softmax runs, the tensor cores work
// on the other tile; the product with V starts on the first 64 keys' weights.
//
// Bound (one B200, 4 chunks of up to 2048 tokens over up to 8192 keys, 32 / 8
// heads of 128: 460 us a call among others, 883 TFLOP/s, 419 to 458 us in a graph
// from rest; 242 us at the measured dense rate): a step
// of both tiles takes about 4100 clocks, the MMAs 2100 and the exponentials of
// the special-function unit 2048 of them; a tile's softmax takes 2200, and its
// hand-over to the MMA warp and back 700.  At heads of more than 64 dims TMEM has
// no room for a third score buffer beside two outputs of 128 columns; at 64 it
// has, 128 columns stay unused (the same chunks, 16 / 2 heads of 64: 204 us, of
// which the MMAs' rate asks 61).
//
// m is the running maximum only loosely: O and the sum are rescaled when the
// maximum has grown by more than 2^8 since the last time (P stays below 2^8,
// exact scaling in the end), so that O is hardly ever read back.
//
// K and V tiles arrive by TMA, one box per page and 64 dims, into a ring of
// 128-byte-swizzled buffers; the group's rows of Q are one box {64 dims, GT
// heads, tokens}.  Boxes past the cache or the head's width read zeros.
// A step in which some row does not see some key ("ragged": the diagonal, a
// window's edge, the end) is masked, and two spare warps clear non-finite
// values out of its V tile, since 0 * inf would reach rows that do not see
// them; if they found any, the epilogue adds them to the rows that do.
#pragma once

#include <cuda.h>

#include "fp8_gemm.cuh"
#include "op_status.cuh"
#include "paged_attn.cuh"

namespace vxb {

constexpr int kCkStep = 128;        // keys per step
constexpr int kCkThreads = 384;     // two softmax warpgroups; TMA, MMA and two clearing warps

template <int DP>
struct ChunkCfg {
    static constexpr int kHalves = DP / 64;
    static constexpr int kQBytes = 2 * 128 * DP * 2;
    static constexpr int kTileBytes = kCkStep * DP * 2;
    static constexpr int kRing = DP > 64 ? 5 : 8;
    static constexpr int kSmemBytes = kQBytes + kRing * kTileBytes + 1024 + 512;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};

// One tcgen05.mma, kind::f16, issued by the lane whose `leader` is set of a warp
// that runs together: in a branch of one lane the operands would have to be
// carried to uniform registers for every instruction (479 us against 462 for the
// case above, before its tiles were ordered).  The matrix descriptors are
// {address >> 4 | leading offset >> 4 << 16, kDescHigh}: 32-bit arithmetic.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride offset 1024, version, 128-byte swizzle

// D[tmem] (+)= A[smem] * B[smem]^T
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint32_t alo, uint32_t blo, uint32_t idesc,
                                        uint32_t accumulate, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n"
        " mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(tmem_d),
        "r"(alo), "r"(blo), "r"(kDescHigh), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t blo, uint32_t idesc,
                                        uint32_t accumulate, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n"
        " mov.b64 b, {%2, %3};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(tmem_d),
        "r"(tmem_a), "r"(blo), "r"(kDescHigh), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// kind::f16 instruction descriptor with A and B of one 16-bit type (format 1
// = bf16, 0 = f16); b_mn: B is MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t make_idesc_16(int M, int N, int b_mn) {
    constexpr uint32_t f = sizeof(T) == 2 && !__is_same(T, __half) ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(b_mn) << 16) |
           (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// The tile of a slot when sequences are taken in the order of their keys, the
// longest first, and a sequence's tiles from its last tokens on: every thread
// ranks one sequence (B <= kCkSort of them) against all others.  `work`: B
// entries of shared memory.  All threads call it.
constexpr int kCkSort = 256;

__device__ __forceinline__ AttnTile find_long_tile(const AttnArgs& a, int64_t slot, int TT, AttnTile* sh, int2* work) {
    const int b = threadIdx.x;
    int2 mine = make_int2(0, 0);  // keys, tiles
    if (b < a.B) {
        const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
        if (lo >= 0 && hi > lo && hi <= a.N) mine = make_int2(a.kv_len[b], (hi - lo + TT - 1) / TT);
        work[b] = mine;
    }
    if (b == 0) sh->b = -1;
    __syncthreads();
    if (mine.y > 0) {
        int64_t base = 0;
        for (int o = 0; o < a.B; ++o) {
            const int2 w = work[o];
            if (w.x > mine.x || (w.x == mine.x && o < b)) base += w.y;
        }
        const int64_t at = slot - base;
        if (at >= 0 && at < mine.y) {
            const int lo = a.cu_q[b];
            const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page_size;
            AttnTile t;
            t.b = b;
            t.tok0 = static_cast<int>(mine.y - 1 - at) * TT;
            t.q0 = lo;
            t.q_len = a.cu_q[b + 1] - lo;
            t.kv_len = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(mine.x), cap)));
            *sh = t;
        }
    }
    fence_proxy_async_smem();  // (`work` lies where TMA writes next)
    __syncthreads();
    return *sh;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kCkThreads, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const AttnArgs a) {
    using Cfg = ChunkCfg<DP>;
    using Mma = MmaType<T>;
    constexpr int R = Cfg::kRing;
    constexpr int H = Cfg::kHalves;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = sq + Cfg::kQBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + R * Cfg::kTileBytes);
    uint64_t* empty = full + R;
    uint64_t* q_bar = empty + R;
    uint64_t* s_full = q_bar + 1;    // [2] scores of a tile ready
    uint64_t* p_full = s_full + 2;   // [2][2] a half of P written
    uint64_t* o_done = p_full + 4;   // [2] O updated
    uint64_t* clear = o_done + 2;    // [R] the slot's tile has been looked at (and cleared)
    uint64_t* end_bar = clear + R;   // every tile has been looked at
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(end_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* poison = abort_flag + 1;
    __shared__ AttnTile sh_tile;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int GT = min(a.G, 128), TT = a.tokens / 2;
    const int gparts = (a.G + GT - 1) / GT;
    // blocks in the order (tiles, the longest first; heads): all heads of a tile run together,
    // and the short tiles fill the end
    const int heads_y = a.Hk * gparts;
    const int64_t slot = blockIdx.x / heads_y;
    const int hy = blockIdx.x % heads_y;
    const int hk = hy / gparts;
    const int g0 = (hy % gparts) * GT;

    if (tid == 0) {
        for (int i = 0; i < R; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
            mbar_init(&clear[i], 2);
        }
        mbar_init(q_bar, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(end_bar, 2);
        *abort_flag = 0;
        *poison = 0;
        fence_barrier_init();
        if (a.pages > 0) {
            prefetch_tmap(&tmap_q);
            prefetch_tmap(&tmap_k);
            prefetch_tmap(&tmap_v);
        }
    }
    grid_dep_wait();
    const AttnTile t = a.B <= kCkSort ? find_long_tile(a, slot, 2 * TT, &sh_tile, reinterpret_cast<int2*>(ring))
                                      : find_tile(a, gridDim.x / heads_y - 1 - slot, 2 * TT, &sh_tile);
    if (t.b < 0) return;
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_launch();  // (the tensor memory is this block's)
    const uint32_t tmem = *tmem_slot;
    // TMEM columns: S (and P) of tile i at 128 i, O of tile i at 256 + 128 i

    const int toks = min(2 * TT, t.q_len - t.tok0);
    const int tiles = toks > TT ? 2 : 1;
    const int heads = min(GT, a.G - g0);
    const int pos0 = t.kv_len - t.q_len + t.tok0;
    const int* table = a.table + t.b * a.table_stride;
    const int key_hi = min(t.kv_len, pos0 + toks);
    const int key_lo = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
    const int step_lo = key_lo / kCkStep;
    const int step_hi = key_hi > key_lo ? (key_hi + kCkStep - 1) / kCkStep : step_lo;
    const int64_t all = step_hi - step_lo;
    const int my_lo = step_lo + static_cast<int>(all * blockIdx.z / a.splits);
    const int my_hi = step_lo + static_cast<int>(all * (blockIdx.z + 1) / a.splits);
    const int steps = my_hi - my_lo;
    // every row of both tiles sees every key of the step (if its pages are there)
    auto even = [&](int step) {
        return step * kCkStep + kCkStep - 1 <= pos0 && (a.window <= 0 || step * kCkStep > pos0 + toks - 1 - a.window);
    };

    if (warp == 8) {
        // -------------------------------------------------- TMA producer --
        if (steps > 0) {
            if (lane == 0) {
                const uint32_t rows = GT * TT;
                mbar_arrive_expect_tx(q_bar, tiles * H * rows * 128);
                for (int i = 0; i < tiles; ++i)
                    for (int h = 0; h < H; ++h)
                        tma_load_3d(sq + (i * H + h) * 16384, &tmap_q, q_bar, h * 64, hk * a.G + g0,
                                    t.q0 + t.tok0 + i * TT);
            }
            const int box = min(a.page_size, kCkStep);   // keys per box
            const int boxes = kCkStep / box;             // 1..8
            bool ok = true;
            for (int i = 0; i < 2 * steps && ok; ++i) {
                const int slot = i % R, step = my_lo + (i >> 1);
                // lane l: box l / H, 64 dims l % H
                const int bx = lane / H, h = lane % H;
                const int j = step * kCkStep + bx * box;
                int pg = -1;
                if (bx < boxes && j < key_hi) pg = table[j >> a.page_shift];
                if (lane == 0) {
                    ok = op_wait(&empty[slot], ((i / R) & 1) ^ 1, abort_flag, kErrWaitEmpty);
                    if (ok) mbar_arrive_expect_tx(&full[slot], Cfg::kTileBytes);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (ok && bx < boxes) {
                    if (pg < 0 || pg >= a.pages) pg = static_cast<int>(a.pages);  // past the cache: zeros
                    tma_load_4d(ring + slot * Cfg::kTileBytes + h * 16384 + bx * box * 128, (i & 1) ? &tmap_v : &tmap_k,
                                &full[slot], h * 64, j & (a.page_size - 1), hk, pg);
                }
                __syncwarp();
            }
        }
        if (*abort_flag) {  // give copies already in flight time to land
            const unsigned long long t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {
            }
        }
    } else if (warp == 9) {
        // ---------------------------------------------------- MMA issuer --
        if (steps > 0) {
            constexpr uint32_t idesc_s = make_idesc_16<T>(128, kCkStep, 0);
            constexpr uint32_t idesc_o = make_idesc_16<T>(128, DP, 1);
            constexpr uint32_t kLow = (16u >> 4) << 16, kLowV = (16384u >> 4) << 16;  // leading offsets
            const uint32_t leader = lane == 0;
            const uint32_t q_addr = smem_u32(sq) >> 4, ring_addr = smem_u32(ring) >> 4;
            auto wait = [&](uint64_t* bar, int parity, int code) {
                return __all_sync(0xffffffffu, op_wait(bar, parity, abort_flag, code)) != 0;
            };
            auto scores = [&](int i, int slot) {  // S_i = Q_i K^T
                const uint32_t qa = kLow | (q_addr + i * (H * 16384 / 16));
                const uint32_t kb = kLow | (ring_addr + slot * (Cfg::kTileBytes / 16));
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) / 16;
                    umma_ss(tmem + i * 128, qa + off, kb + off, idesc_s, kk != 0, leader);
                }
                umma_commit_by(&s_full[i], leader);
            };
            bool ok = wait(q_bar, 0, kErrWaitFull) && wait(&clear[0], 0, kErrWaitFull);
            if (ok) {
                tc_fence_after();
                for (int i = 0; i < tiles; ++i) scores(i, 0);
                umma_commit_by(&empty[0], leader);
            }
            for (int j = 0; j < steps && ok; ++j) {
                const int iv = 2 * j + 1, ik = 2 * j + 2;  // ring items of V_j and K_{j+1}
                ok = wait(&clear[iv % R], (iv / R) & 1, kErrWaitFull);
                if (ok && j + 1 < steps) ok = wait(&clear[ik % R], (ik / R) & 1, kErrWaitFull);
                const uint32_t vb = kLowV | (ring_addr + (iv % R) * (Cfg::kTileBytes / 16));
                for (int i = 0; i < tiles && ok; ++i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // (the product starts on the first half of P)
                        ok = ok && wait(&p_full[2 * i + half], j & 1, kErrWaitAccum);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 4 * half; kk < 4 * half + 4; ++kk)  // 16 keys: 8 TMEM columns of P, 2 KB of V rows
                            umma_ts(tmem + 256 + i * 128, tmem + i * 128 + kk * 8, vb + kk * (2048 / 16), idesc_o,
                                    (j | kk) != 0, leader);
                    }
                    if (!ok) break;
                    umma_commit_by(&o_done[i], leader);
                    if (i == tiles - 1) umma_commit_by(&empty[iv % R], leader);
                    // (in order behind the product that reads P, which these scores overwrite)
                    if (j + 1 < steps) {
                        scores(i, ik % R);
                        if (i == tiles - 1) umma_commit_by(&empty[ik % R], leader);
                    }
                }
            }
            if (!ok) {  // arrives once every issued MMA is done
                umma_commit_by(&o_done[0], leader);
                umma_commit_by(&o_done[1], leader);
            }
        }
        __syncwarp();
    } else if (warp >= 10) {
        // ------------------------------- clearing of ragged steps' V tiles --
        // Every tile passes here on its way from the TMA to the MMA issuer, so
        // that a slot is not filled again before these warps have seen it.
        const int ct = tid - 320;  // 0..63
        bool ok = true;
        for (int i = 0; i < 2 * steps; ++i) {
            const int slot = i % R;
            ok = op_wait(&full[slot], (i / R) & 1, abort_flag, kErrWaitFull);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if ((i & 1) && !even(my_lo + (i >> 1))) {
                uint4* v = reinterpret_cast<uint4*>(ring + slot * Cfg::kTileBytes);
                bool found = false;
#pragma unroll 4
                for (int c = ct; c < Cfg::kTileBytes / 16; c += 64) {
                    uint4 raw = v[c];
                    T* e = reinterpret_cast<T*>(&raw);
                    bool bad = false;
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        if (!isfinite(to_float(e[x]))) {
                            bad = true;
                            e[x] = from_float<T>(0.f);
                        }
                    if (bad) {  // (what lies behind the last key is nobody's)
                        found = found || (my_lo + (i >> 1)) * kCkStep + ((c >> 3) & 127) < key_hi;
                        v[c] = raw;
                    }
                }
                if (found) *poison = 1;
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(&clear[slot]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(end_bar);
    } else {
        // --------------------------------------------- softmax, epilogue --
        const int i = warp >> 2;                 // tile of this warpgroup
        const int q = warp & 3;
        const int r = q * 32 + lane;             // row of the tile
        const int tk = i * TT + r / GT, g = r % GT;
        const bool on = i < tiles && r < GT * TT && tk < toks && g < heads;
        const int pos = on ? pos0 + tk : -1;
        const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
        const uint32_t ts = tmem + i * 128 + lanes, to = tmem + 256 + i * 128 + lanes;
        const bool neg = a.scale_log2 < 0.f;
        const float scale = fabsf(a.scale_log2);
        float m = kNegInf, l = 0.f;              // maximum (of the scores as they are) and sum
        bool ok = true;
        int n = i < tiles ? steps : 0;
        // lane k < 8: is the page of keys 16 k .. 16 k + 15 of the step there?
        auto present = [&](int step) {
            const int j = step * kCkStep + (lane & 7) * 16;
            if (j >= key_hi) return false;
            const int pg = table[j >> a.page_shift];
            return pg >= 0 && pg < a.pages;
        };
        bool here = n > 0 && present(my_lo);
        for (int j = 0; j < n; ++j) {
            const int step = my_lo + j;
            const uint32_t there = __ballot_sync(0xffffffffu, here) & 0xffu;
            here = j + 1 < n && present(step + 1);
            ok = op_wait(&s_full[i], j & 1, abort_flag, kErrWaitAccum);
            ok = __all_sync(0xffffffffu, ok && !*abort_flag);
            if (!ok) break;
            tc_fence_after();
            uint32_t sv[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_async(ts + 32 * c, sv + 32 * c);
            tmem_ld_wait<128>(sv);
            float* s = reinterpret_cast<float*>(sv);
            if (neg) {
#pragma unroll
                for (int c = 0; c < 128; ++c) s[c] = -s[c];
            }
            if (!even(step) || there != 0xffu) {
                const int lo = a.window > 0 ? pos - a.window : -1;  // sees lo < key <= pos
#pragma unroll
                for (int c = 0; c < 128; ++c) {
                    const int key = step * kCkStep + c;
                    if (key > pos || key <= lo || !((there >> (c >> 4)) & 1)) s[c] = kNegInf;
                }
            }
            float t4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < 124; c += 8)
#pragma unroll
                for (int x = 0; x < 4; ++x) t4[x] = fmaxf(t4[x], fmaxf(s[c + x], s[c + 4 + x]));
            const float top = fmaxf(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])),
                                    fmaxf(fmaxf(s[124], s[125]), fmaxf(s[126], s[127])));
            // rescale if some row of the warp has outgrown its m
            const bool grow = m == kNegInf ? top > kNegInf : (top - m) * scale > kAttnLazy;
            if (__any_sync(0xffffffffu, grow)) {
                const float mn = grow ? top : m;
                const float f = m == mn ? 1.f : ex2((m - mn) * scale);  // 0 from an empty start
                m = mn;
                l *= f;
                if (j > 0) {
                    ok = op_wait(&o_done[i], (j - 1) & 1, abort_flag, kErrWaitAccum);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < DP; c += 16) {
                        uint32_t o[16];
                        tmem_ld16_async(to + c, o);
                        tmem_ld_wait<16>(o);
#pragma unroll
                        for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        tmem_st16(to + c, o);
                    }
                }
            }
            const float base = m == kNegInf ? 0.f : m * scale;
            float2 sum = make_float2(0.f, 0.f), sum2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                uint32_t p[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float2 e = ffma2(make_float2(s[c + 2 * x], s[c + 2 * x + 1]), make_float2(scale, scale),
                                           make_float2(-base, -base));
                    const float2 w = make_float2(ex2(e.x), ex2(e.y));
                    if (x & 1) {
                        sum2.x += w.x, sum2.y += w.y;
                    } else {
                        sum.x += w.x, sum.y += w.y;
                    }
                    p[x] = Mma::pack(w.x, w.y);
                }
                tmem_st16(ts + c / 2, p);
                if (c & 32) {  // 64 keys are written: the product with V starts on them
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * i + c / 64]);
                }
            }
            l += (sum.x + sum.y) + (sum2.x + sum2.y);
        }
        if (n > 0 && ok) {
            ok = op_wait(&o_done[i], (n - 1) & 1, abort_flag, kErrWaitAccum);
            ok = ok && op_wait(end_bar, 0, abort_flag, kErrWaitAccum);
            ok = __all_sync(0xffffffffu, ok && !*abort_flag);
            if (ok) tc_fence_after();
        }
        if (ok && i < tiles) {
            const int64_t tok = static_cast<int64_t>(t.q0) + t.tok0 + tk;
            const int head = hk * a.G + g0 + g;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int lo = max(my_lo * kCkStep, a.window > 0 ? max(0, pos - a.window + 1) : 0);
            const int hi = min(my_hi * kCkStep, min(pos + 1, t.kv_len));
            const int64_t row = (blockIdx.z * a.N + tok) * a.Hq + head;
#pragma unroll 1
            for (int c = 0; c < DP; c += 16) {
                uint32_t o[16];
                if (n > 0) {
                    tmem_ld16_async(to + c, o);
                    tmem_ld_wait<16>(o);
                }
                if (on && c < a.D) {
                    float y[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) y[x] = l == 0.f ? 0.f : __uint_as_float(o[x]) * inv;
                    if (*poison) {
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (c + x < a.D) y[x] += attn_poison<T>(a, table, hk, c + x, lo, hi);
                    }
                    T* dst = static_cast<T*>(a.out) + tok * a.o_token + head * a.o_head + c;
                    if (a.splits > 1) {
                        // (D is a multiple of 8: whole vectors, 32-byte rows)
#pragma unroll
                        for (int x = 0; x < 16; x += 8)
                            if (c + x < a.D) store8<float, true>(a.part_o + row * a.D + c + x, 8, y + x);
                    } else if (c + 16 <= a.D && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
                        store8<T, true>(dst, 8, y);
                        store8<T, true>(dst + 8, 8, y + 8);
                    } else {
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (c + x < a.D) dst[x] = from_float<T>(y[x]);
                    }
                }
                __syncwarp();
            }
            if (on && a.splits > 1) a.part_lse[row] = l == 0.f ? kNegInf : (m == kNegInf ? 0.f : m * scale) + log2f(l);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (tid == 0) record_abort(abort_flag);
    if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace vxb
