// Attention of new tokens over a paged cache, few query rows at a time.
//
// For sequence b with q_len new tokens and kv_len cached keys (the new ones
// included), token i stands at position p = kv_len - q_len + i and sees the
// keys j with j <= p and (window > 0) j > p - window:
//   out = sum_j softmax_j(scale * q . k_j) v_j, zeros if it sees none.
// Key j lies in page table[b][j / page_size], place j % page_size.  A table
// entry outside [0, pages) makes its keys unseen.
//
// The G = Hq / Hk query heads that share a key head are rows of one tile
// (row = token * G + head), so a key is read once for all of them: with one
// new token per sequence the kernel reads K and V once and is HBM bound.  A
// block has one tile of 16 * MT rows; a step is 64 * KW keys, of which each
// of 4 warps takes 16 * KW: it keeps its own running maximum, sum and output
// (mma.sync m16n8k16, fp32), so no warp waits for another's softmax, and the
// four are joined once at the end.  The tensor work of a few rows is far below
// the time of its bytes, so the accumulators stay in registers.  A fifth warp feeds a
// ring of kStages steps by TMA, one box per page and 64 dims; it reads the
// table 32 entries ahead, so a step never waits for its page numbers.
//
// With few (sequence, head) pairs the keys are split over blockIdx.z; each
// part leaves its normalised output and log2 of its sum (fp32), and
// attn_join_kernel weighs them.
//
// Measured (one B200, 6.55 TB/s copy rate): one token after 131072 keys, 32 / 8
// heads of 128: 90 us, 5.9 TB/s; 256 tokens after 1 to 2048 keys, 16 / 2 heads of
// 64: 32 us (19.6 us of bytes; 6.0 to 6.5 TB/s from 8 to 20 us after the start,
// then the longest sequences' blocks end).  A sequence far longer than the rest
// of a large batch is not split: 159 of 300 keys and one of 65536, 16 / 2 heads of
// 64, take 395 us, 27 us in two calls.  Steps of 128 keys at 64 dims (39 us
// with 64: the per-step overhead of a warp, not its loads, fills the time), 64 KB
// of ring there so that three blocks share an SM (two with 96 KB: 42 us).
//
// exp(s * scale - max) is computed as exp2 of s * scale * log2(e) - max.  P is
// rounded to the cache's type for the second product (at most half a step,
// 2^-8 of each weight in bf16), the sum is taken of the unrounded weights.
#pragma once

#include <cuda.h>

#include "lm_norm.cuh"
#include "op_status.cuh"

namespace vxb {

constexpr float kAttnLazy = 8.f;   // log2 growth of the maximum that the output is rescaled for
constexpr int kAttnThreads = 160;  // 4 warps of rows x keys, one that loads
constexpr float kNegInf = -INFINITY;

struct AttnArgs {
    const void* q;
    int64_t q_token, q_head;       // strides in elements
    void* out;
    int64_t o_token, o_head;
    const void* k;
    const void* v;
    int64_t page_stride, slot_stride, cache_head;
    const int* table;              // [B][table_stride]
    int64_t table_stride;
    const int* cu_q;               // [B + 1]
    const int* kv_len;             // [B]
    int64_t N;                     // rows of q
    int64_t pages;
    int B, Hq, Hk, G, D;
    int page_size, page_shift;
    int max_pages;                 // entries of a table row
    int window;
    int tokens;                    // tokens of a tile
    float scale_log2;              // softmax scale * log2(e)
    int splits;
    float* part_o;                 // [splits][N * Hq][D]
    float* part_lse;               // [splits][N * Hq], log2 of the sum, -inf if empty
};

template <typename T>
struct MmaType;
template <>
struct MmaType<__half> {
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&h);
    }
};
template <>
struct MmaType<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&h);
    }
};

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* tmap, uint64_t* bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void ldsm_x4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void prefetch_l1(const void* p) {
    asm volatile("prefetch.global.L1 [%0];" ::"l"(p) : "memory");
}

// A tile of query rows: which sequence, its tokens and keys.
struct AttnTile {
    int b;            // -1: nothing to do
    int tok0;         // first token of the tile within the sequence
    int q0;           // the sequence's first row of q
    int q_len, kv_len;
};

// Tile slots of TT tokens are numbered so that sequence b starts at slot
// cu_q[b] / TT + b: the next sequence's start is at least ceil(q_len / TT)
// later, so every tile has a slot and a slot finds its sequence from cu_q
// alone, with no sum over the sequences before it.  With TT = 1 a slot is a
// token.  Lengths out of range (the table's capacity, the rows of q) are cut.
__device__ __forceinline__ bool tile_of(const AttnArgs& a, int b, int64_t slot, int TT, AttnTile* t) {
    const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
    const int kv = a.kv_len[b];
    const int64_t t0 = TT == 1 ? slot - lo : (slot - (lo / TT + b)) * TT;
    if (lo < 0 || hi <= lo || hi > a.N || t0 < 0 || t0 >= hi - lo) return false;
    const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page_size;
    t->b = b;
    t->tok0 = static_cast<int>(t0);
    t->q0 = lo;
    t->q_len = hi - lo;
    t->kv_len = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(kv), cap)));
    return true;
}

// The tile of a slot; all threads call it.  In a batch of single tokens a slot
// is its sequence: one round trip to memory, no search.
__device__ __forceinline__ AttnTile find_tile(const AttnArgs& a, int64_t slot, int TT, AttnTile* sh) {
    AttnTile t;
    t.b = -1;
    if (TT == 1 && slot < a.B && tile_of(a, static_cast<int>(slot), slot, TT, &t)) {
        __syncthreads();
        return t;
    }
    // (the first sequence that claims the slot has it: with row ranges that overlap, which
    // are not sequences, two could)
    if (threadIdx.x == 0) sh->b = INT32_MAX;
    __syncthreads();
    for (int b = threadIdx.x; b < a.B; b += blockDim.x)
        if (tile_of(a, b, slot, TT, &t)) {
            atomicMin(&sh->b, b);
            break;
        }
    __syncthreads();
    const int b = sh->b;
    if (b == INT32_MAX) {
        t.b = -1;
    } else {
        tile_of(a, b, slot, TT, &t);
    }
    return t;
}

template <typename T, int DP, int MT, int KW>
struct AttnCfg {
    static constexpr int kStep = 64 * KW;                      // keys of a step, 16 * KW a warp
    static constexpr int kRows = 16 * MT;
    static constexpr int kHalves = DP / 64;
    static constexpr int kTileBytes = kStep * DP * 2;          // K or V of one step: [half][key][64 dims]
    static constexpr int kStages = (DP > 64 ? 96 : 64) * 1024 / (2 * kTileBytes);
    static constexpr int kQBytes = kRows * DP * 2;
    static constexpr int kSmemBytes = kStages * 2 * kTileBytes + kQBytes + 1024 + 128;
    static constexpr int kJoinLD = DP + 4;
    static constexpr int kJoinBytes = 4 * kRows * kJoinLD * 4 + 4 * kRows * 8;  // reuses the ring
    static_assert(kJoinBytes <= kStages * 2 * kTileBytes, "the joining fits the ring");
};

// Byte offset of 16-byte chunk c of row r in a tile of R rows of 64 * n dims:
// [c / 8][r][c % 8] with the 128-byte swizzle (chunk index XOR row), as TMA
// writes it; ldmatrix reads of 8 rows hit all banks.
template <int R>
__device__ __forceinline__ uint32_t attn_off(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * R * 128 + r * 128 + (((c ^ r) & 7) << 4));
}

// Sum of the non-finite values of v[.., d] over the keys [j0, j1) of sequence
// row `table`: 0 if there are none.
template <typename T>
__device__ float attn_poison(const AttnArgs& a, const int* table, int head, int d, int j0, int j1) {
    float s = 0.f;
    for (int j = j0; j < j1; ++j) {
        const int pg = table[j / a.page_size];
        if (pg < 0 || pg >= a.pages) continue;
        const float v = to_float(static_cast<const T*>(a.v)[pg * a.page_stride + (j % a.page_size) * a.slot_stride +
                                                            head * a.cache_head + d]);
        if (!isfinite(v)) s += v;
    }
    return s;
}

template <typename T, int DP, int MT, int KW>
__global__ void __launch_bounds__(kAttnThreads) attn_rows_kernel(const __grid_constant__ CUtensorMap tmap_k,
                                                                 const __grid_constant__ CUtensorMap tmap_v,
                                                                 const AttnArgs a) {
    using Cfg = AttnCfg<T, DP, MT, KW>;
    constexpr int kStep = Cfg::kStep;
    using Mma = MmaType<T>;
    constexpr int S = Cfg::kStages;
    constexpr int H = Cfg::kHalves;
    constexpr int CH = DP / 8;  // 16-byte chunks of a row
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sq = smem + S * 2 * Cfg::kTileBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(sq + Cfg::kQBytes);
    uint64_t* empty = full + S;
    volatile uint32_t* there = reinterpret_cast<volatile uint32_t*>(empty + S);  // [S] pages of the slot's step
    __shared__ AttnTile sh_tile;
    __shared__ int sh_poison;
    __shared__ int sh_abort;
    volatile int* abort_flag = &sh_abort;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int TT = a.tokens;                                     // of a tile
    const int GT = min(a.G, Cfg::kRows);                         // heads of the group per tile
    const int gparts = (a.G + GT - 1) / GT;                      // tiles a group of heads takes
    const int hk = blockIdx.y / gparts;
    const int g0 = (blockIdx.y % gparts) * GT;
    if (tid == 0) {
        sh_poison = 0;
        sh_abort = 0;
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 4);
        }
        fence_barrier_init();
        if (a.pages > 0) {
            prefetch_tmap(&tmap_k);
            prefetch_tmap(&tmap_v);
        }
    }
    grid_dep_sync();
    if (TT == 1 && warp == 4 && blockIdx.x < a.B && lane < a.max_pages)  // most likely the tile's page numbers
        prefetch_l1(a.table + blockIdx.x * a.table_stride + lane);
    const AttnTile t = find_tile(a, blockIdx.x, TT, &sh_tile);
    if (t.b < 0) return;
    const int toks = min(TT, t.q_len - t.tok0);
    const int heads = min(GT, a.G - g0);
    // row r of the tile: token r / GT, head r % GT
    const int pos0 = t.kv_len - t.q_len + t.tok0;  // position of the tile's first token (may be negative)
    const int* table = a.table + t.b * a.table_stride;

    // keys any row sees, and this part's share of them in whole steps
    const int key_hi = min(t.kv_len, pos0 + toks);
    const int key_lo = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
    const int step_lo = key_lo / kStep;
    const int step_hi = key_hi > key_lo ? (key_hi + kStep - 1) / kStep : step_lo;
    const int64_t steps = step_hi - step_lo;
    const int my_lo = step_lo + static_cast<int>(steps * blockIdx.z / a.splits);
    const int my_hi = step_lo + static_cast<int>(steps * (blockIdx.z + 1) / a.splits);

    if (warp == 4) {
        // -------------------------------------------------- TMA producer --
        const int box = min(a.page_size, kStep), bps = kStep / box;  // keys of a box, boxes of a step
        const int per = 32 / bps;                                           // steps whose boxes 32 lanes know
        auto page = [&](int first) {  // of this lane's box, counted from step `first`
            const int64_t j = static_cast<int64_t>(first) * kStep + lane * box;
            return j < key_hi && first < my_hi ? table[j >> a.page_shift] : -1;
        };
        const int kv = lane & 1, h = (lane >> 1) % H, bx = (lane >> 1) / H;
        int next = page(my_lo);
        bool ok = true;
        for (int first = my_lo; first < my_hi && ok; first += per) {
            const int cur = next;
            next = page(first + per);
            for (int step = first; step < min(first + per, my_hi); ++step) {
                const int i = step - my_lo, slot = i % S;
                int pg = __shfl_sync(0xffffffffu, cur, ((step - first) * bps + bx) & 31);
                ok = op_wait(&empty[slot], ((i / S) & 1) ^ 1, abort_flag, kErrWaitEmpty);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // bit g: keys 16 g .. 16 g + 15 of the step lie in a page
                const uint32_t valid = __ballot_sync(0xffffffffu, bx < bps && pg >= 0 && pg < a.pages);
                const uint32_t groups = __ballot_sync(
                    0xffffffffu, lane < kStep / 16 && ((valid >> ((lane * 16 / box) * H * 2 & 31)) & 1));
                if (lane == 0) {
                    there[slot] = groups;
                    mbar_arrive_expect_tx(&full[slot], 2 * Cfg::kTileBytes);
                }
                __syncwarp();
                if (bx < bps) {
                    if (pg < 0 || pg >= a.pages) pg = static_cast<int>(a.pages);  // past the cache: zeros
                    uint8_t* dst = smem + slot * 2 * Cfg::kTileBytes + kv * Cfg::kTileBytes + h * kStep * 128 +
                                   bx * box * 128;
                    tma_load_4d(dst, kv ? &tmap_v : &tmap_k, &full[slot], h * 64,
                                (step * kStep + bx * box) & (a.page_size - 1), hk, pg);
                }
            }
        }
        if (*abort_flag) {  // give copies already in flight time to land
            const unsigned long long t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {
            }
        }
    } else {
        // queries: rows of the tile (zeros past the tokens and past D)
        for (int i = tid; i < Cfg::kRows * CH; i += 128) {
            const int r = i / CH, c = i % CH;
            const int tk = r / GT, g = r % GT;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (tk < toks && g < heads && c * 8 < a.D)
                v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                    (static_cast<int64_t>(t.q0) + t.tok0 + tk) * a.q_token +
                                                    (hk * a.G + g0 + g) * a.q_head + c * 8);
            *reinterpret_cast<uint4*>(sq + attn_off<Cfg::kRows>(r, c)) = v;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
    }

    float o[MT][DP / 8][4];
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < DP / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
        m[i][0] = m[i][1] = kNegInf;
        l[i][0] = l[i][1] = 0.f;
    }
    // the position of each of this thread's rows (row lane/4 and lane/4 + 8 of each m16)
    int pos[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = i * 16 + h * 8 + (lane >> 2);
            pos[i][h] = r / GT < toks && r % GT < heads ? pos0 + r / GT : -1;
        }
    const int rows = toks * GT;  // of the tile that hold something
    const int pos_min = pos0, pos_max = pos0 + toks - 1;
    bool poison = false;

    // the tile's Q fragments stay in registers where there is room
    constexpr bool kQRegs = MT == 1;
    uint32_t qf[kQRegs ? DP / 16 : 1][4];
    if (kQRegs && warp < 4) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
            ldsm_x4(qf[kQRegs ? k : 0], smem_u32(sq) + attn_off<Cfg::kRows>(lane & 15, 2 * k + (lane >> 4)));
    }
    bool ok = true;
    for (int step = warp < 4 ? my_lo : my_hi; step < my_hi; ++step) {
        const int it = step - my_lo, slot = it % S;
        uint8_t* bk = smem + slot * 2 * Cfg::kTileBytes;
        uint8_t* bv = bk + Cfg::kTileBytes;
        const int j0 = step * kStep + warp * 16 * KW;  // this warp's keys
        // does every row see all of the warp's keys?
        bool whole = j0 + 16 * KW - 1 <= pos_min && (a.window <= 0 || j0 > pos_max - a.window);
        ok = op_wait(&full[slot], (it / S) & 1, abort_flag, kErrWaitFull);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // bit i: key j0 + i lies in no page
        const uint32_t in = there[slot] >> (warp * KW);
        const uint32_t absent = (in & 1 ? 0 : 0xffffu) | (KW > 1 && !(in & 2) ? 0xffff0000u : 0);
        whole = whole && absent == 0;
        if (!whole) {
            // A key that some row does not see has weight 0 there, but 0 * inf is NaN: non-finite
            // values leave the tile and are added at the end to the rows that see them.
            for (int i = lane; i < 16 * KW * CH; i += 32) {
                const int r = warp * 16 * KW + i / CH, c = i % CH;
                uint4* p = reinterpret_cast<uint4*>(bv + attn_off<kStep>(r, c));
                uint4 raw = *p;
                T* e = reinterpret_cast<T*>(&raw);
                bool bad = false;
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (!isfinite(to_float(e[x]))) {
                        bad = true;
                        e[x] = from_float<T>(0.f);
                    }
                if (bad) {
                    poison = poison || step * kStep + r < key_hi;
                    *p = raw;
                }
            }
            fence_proxy_async_smem();  // (before the TMA fills the slot again)
            __syncwarp();
        }

        // S = Q K^T of 16 * MT rows x 16 * KW keys
        float s[MT][2 * KW][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int n = 0; n < 2 * KW; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t qs[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (!kQRegs)
                    ldsm_x4(qs[i], smem_u32(sq) + attn_off<Cfg::kRows>(i * 16 + (lane & 15), 2 * k + (lane >> 4)));
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                uint32_t kb[4];
                // matrices: keys 0-7 and 8-15, each k halves 0-7, 8-15
                ldsm_x4(kb, smem_u32(bk) + attn_off<kStep>((warp * KW + w) * 16 + (lane & 7) + ((lane >> 4) << 3),
                                                           2 * k + ((lane >> 3) & 1)));
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const uint32_t* qa = kQRegs ? qf[kQRegs ? k : 0] : qs[i];
                    Mma::mma(s[i][2 * w], qa, kb[0], kb[1]);
                    Mma::mma(s[i][2 * w + 1], qa, kb[2], kb[3]);
                }
            }
        }
        // Scores in log2 units, hidden ones -inf.  m, the maximum that weights are taken
        // relative to, follows the true one only when that has outgrown it by 2^8.
        bool grow = false;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && rows <= i * 16 + 8) continue;
                float top = kNegInf;
#pragma unroll
                for (int n = 0; n < 2 * KW; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = s[i][n][2 * h + e] * a.scale_log2;
                        if (!whole) {
                            const int kk = n * 8 + (lane & 3) * 2 + e;
                            const int j = j0 + kk;
                            if (j > pos[i][h] || (a.window > 0 && j <= pos[i][h] - a.window) || ((absent >> kk) & 1))
                                v = kNegInf;
                        }
                        s[i][n][2 * h + e] = v;
                        // (a NaN score has to reach the sum: max ignores it)
                        top = fmaxf(top, v);
                    }
                grow = grow || top > m[i][h] + kAttnLazy;
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1 && rows <= i * 16 + 8) continue;
                    float top = kNegInf;
#pragma unroll
                    for (int n = 0; n < 2 * KW; ++n) top = fmaxf(top, fmaxf(s[i][n][2 * h], s[i][n][2 * h + 1]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float old = m[i][h];
                    if (top > old + kAttnLazy) m[i][h] = top;
                    const float corr = m[i][h] == old ? 1.f : ex2(old - m[i][h]);
                    l[i][h] *= corr;
#pragma unroll
                    for (int j = 0; j < DP / 8; ++j) {
                        o[i][j][2 * h] *= corr;
                        o[i][j][2 * h + 1] *= corr;
                    }
                }
        }
        uint32_t pa[MT][KW][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && rows <= i * 16 + 8) {
#pragma unroll
                    for (int w = 0; w < KW; ++w) pa[i][w][1] = pa[i][w][3] = 0;
                    continue;
                }
                const float base = m[i][h] == kNegInf ? 0.f : m[i][h];
#pragma unroll
                for (int n = 0; n < 2 * KW; ++n) {
                    const float p0 = ex2(s[i][n][2 * h] - base), p1 = ex2(s[i][n][2 * h + 1] - base);
                    l[i][h] += p0 + p1;
                    pa[i][n >> 1][2 * (n & 1) + h] = Mma::pack(p0, p1);
                }
            }
        // O += P V
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                uint32_t vb[4];
                // matrices: (keys 0-7, dims 0-7), (keys 8-15, dims 0-7), (keys 0-7, dims 8-15), (8-15, 8-15)
                ldsm_x4_t(vb, smem_u32(bv) + attn_off<kStep>((warp * KW + w) * 16 + (lane & 15), 2 * d + (lane >> 4)));
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    Mma::mma(o[i][2 * d], pa[i][w], vb[0], vb[1]);
                    Mma::mma(o[i][2 * d + 1], pa[i][w], vb[2], vb[3]);
                }
            }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[slot]);
    }
    if (poison) sh_poison = 1;
    __syncthreads();  // every copy has landed and been read: the ring is free
    if (*abort_flag) {
        if (tid == 0) record_abort(abort_flag);
        return;
    }

    // Join the four warps: each leaves its output (rows padded by 4 words: no bank
    // conflicts), maximum and sum; then a thread adds 4 dims of a row.
    constexpr int LD = Cfg::kJoinLD;
    float* jo = reinterpret_cast<float*>(smem);                  // [4][rows][LD]
    float2* jm = reinterpret_cast<float2*>(jo + 4 * Cfg::kRows * LD);  // [rows][4]: maximum, sum
    if (warp < 4) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && rows <= i * 16 + 8) continue;
                const int r = i * 16 + h * 8 + (lane >> 2);
                float sum = l[i][h];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if ((lane & 3) == 0) jm[r * 4 + warp] = make_float2(m[i][h], sum);
#pragma unroll
                for (int j = 0; j < DP / 8; ++j)
                    *reinterpret_cast<float2*>(&jo[(warp * Cfg::kRows + r) * LD + j * 8 + (lane & 3) * 2]) =
                        make_float2(o[i][j][2 * h], o[i][j][2 * h + 1]);
            }
    }
    __syncthreads();
    const bool poisoned = sh_poison != 0;
    for (int i = tid; i < rows * (DP / 4); i += kAttnThreads) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        const int tk = TT == 1 ? 0 : r / GT, g = r - tk * GT;
        if (g >= heads || d >= a.D) continue;
        float2 ml[4];
        float top = kNegInf;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ml[w] = jm[r * 4 + w];
            top = fmaxf(top, ml[w].x);
        }
        const float base = top == kNegInf ? 0.f : top;
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ex2(ml[w].x - base);
            sum += f * ml[w].y;
            const float4 x = *reinterpret_cast<const float4*>(&jo[(w * Cfg::kRows + r) * LD + d]);
            v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
        }
        // (an empty row has sum 0; a NaN score makes the sum NaN)
        const float inv = 1.f / sum;
        float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
        if (sum == 0.f) y[0] = y[1] = y[2] = y[3] = 0.f;
        if (poisoned) {
            const int p = pos0 + tk;
            const int lo = max(my_lo * kStep, a.window > 0 ? max(0, p - a.window + 1) : 0);
            const int hi = min(my_hi * kStep, min(p + 1, t.kv_len));
            for (int x = 0; x < 4; ++x) y[x] += attn_poison<T>(a, table, hk, d + x, lo, hi);
        }
        const int64_t tok = static_cast<int64_t>(t.q0) + t.tok0 + tk;
        const int head = hk * a.G + g0 + g;
        if (a.splits == 1) {
            T* dst = static_cast<T*>(a.out) + tok * a.o_token + head * a.o_head + d;
            uint2 w;
            w.x = Mma::pack(y[0], y[1]);
            w.y = Mma::pack(y[2], y[3]);
            if ((reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
                *reinterpret_cast<uint2*>(dst) = w;
            } else {
                const T* e = reinterpret_cast<const T*>(&w);
                for (int x = 0; x < 4; ++x) dst[x] = e[x];
            }
        } else {
            const int64_t row = (blockIdx.z * a.N + tok) * a.Hq + head;
            *reinterpret_cast<float4*>(a.part_o + row * a.D + d) = make_float4(y[0], y[1], y[2], y[3]);
            if (d == 0) a.part_lse[row] = sum == 0.f ? kNegInf : base + log2f(sum);
        }
    }
}

// out[row] = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max), at most
// kAttnMaxSplits parts.  `warps` (1 or 4) of a block's 4 warps share a row:
// lanes hold the parts' weights, a warp adds every `warps`-th part, 4 dims a
// lane.
constexpr int kAttnMaxSplits = 64;

template <typename T, int kWarps>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a) {
    __shared__ float4 part[4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % kWarps;
    grid_dep_sync();
    const int64_t rows = a.N * a.Hq;
    const int64_t row = min(static_cast<int64_t>(blockIdx.x) * (4 / kWarps) + warp / kWarps, rows - 1);
    const int64_t tok = row / a.Hq;
    const int head = static_cast<int>(row % a.Hq);
    // rows outside every sequence are left as they are
    bool in = false;
    for (int b = lane; b < a.B; b += 32) {
        const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
        in = in || (lo >= 0 && hi <= a.N && tok >= lo && tok < hi);
    }
    float lse[2], w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) lse[i] = lane + 32 * i < a.splits ? a.part_lse[(lane + 32 * i) * rows + row] : kNegInf;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = fmaxf(lse[0], lse[1]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == kNegInf ? 0.f : top;
    // (a NaN part makes every weight's sum NaN, and with it the row)
    w[0] = ex2(lse[0] - base);
    w[1] = ex2(lse[1] - base);
    float sum = w[0] + w[1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // (parts that are empty are not read; one whose weight is only too small for fp32 is, since a
    // non-finite value in it reaches the row all the same)
    const uint32_t some[2] = {__ballot_sync(0xffffffffu, lse[0] != kNegInf), __ballot_sync(0xffffffffu, lse[1] != kNegInf)};
#pragma unroll 4
    for (int s = mine; s < a.splits; s += kWarps) {
        const float f = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
        if (lane * 4 < a.D && ((s < 32 ? some[0] : some[1]) >> (s & 31) & 1)) {
            const float4 o = *reinterpret_cast<const float4*>(a.part_o + (s * rows + row) * a.D + lane * 4);
            v.x = fmaf(f, o.x, v.x), v.y = fmaf(f, o.y, v.y), v.z = fmaf(f, o.z, v.z), v.w = fmaf(f, o.w, v.w);
        }
    }
    in = __any_sync(0xffffffffu, in);
    if (kWarps > 1) {
        part[warp][lane] = v;
        __syncthreads();
        if (warp > 0) return;
        v = part[0][lane];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) {
            const float4 o = part[i][lane];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
    }
    if (!in || lane * 4 >= a.D) return;
    T* dst = static_cast<T*>(a.out) + tok * a.o_token + head * a.o_head + lane * 4;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
    for (int x = 0; x < 4; ++x) dst[x] = from_float<T>(y[x]);
}

}  // namespace vxb
