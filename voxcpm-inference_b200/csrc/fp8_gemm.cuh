// Product of 8-bit (e4m3) matrices with fp32 scales for blocks of 128:
//
//   y[n][m] = bias[m] + sum_b xs[n][b] * ws[m / 128][b] * P_b[n][m],
//   P_b[n][m] = sum_{k in block b} x[n][k] * w[m][k]
//
// A scale changes every 128 k, so the tensor cores cannot accumulate over the
// whole of K: each block's product P_b (four tcgen05.mma of K = 32, kind
// f8f6f4, fp32 accumulator) goes to one of two TMEM buffers, and the epilogue
// warps add it, scaled, to the running sum in their registers (fp32) while the
// next block's product is formed in the other buffer.
//
// Two orientations of the 128-row operand (the TMEM lanes):
//   tokens as rows (many tokens): A = x tile, B = w tile of BN outputs; a
//     thread holds one token, its x scale is the thread's own and the w scale
//     is the same for all of a warpgroup's columns: one FMA per element.
//   weights as rows (few tokens): A = w tile of 128 outputs (one scale block),
//     B = x tile of BN = 16, 32 or 64 tokens; a thread holds one output, the
//     w scale is the same for the tile and the x scales of the columns are
//     kept one per lane and passed around by shuffles.
// With fewer tiles than SMs, K is split over the blocks of a cluster; each
// leaves its partial sums in its own shared memory and all of them add a
// share of the columns over distributed shared memory, in rank order (the
// result does not depend on timing).
//
// Bounds and measurements (one B200).  Few tokens: 4 x 1024 -> 4096 4.6 us, a
// chain of launch, TMA, MMA and join; 1 x 8192 -> 8192 16.9 us, 4.0 TB/s of
// weights.  Many: 8192 x 4096 -> 8192 347 to 353 us a call among others (1570
// TFLOP/s), 293 to 323 us in a graph from rest (1700 to 1880; the MMAs are busy
// 45 % of the time); of 293, 203 us with the scaled additions left out, 177 us with the
// MMAs free-running, and 992 W at 1640 MHz when it runs on (334 us).
//
// Warp roles: warp 0 lane 0 issues TMA loads, warp 1 owns TMEM and issues the
// MMAs, warps 4.. are one or two epilogue warpgroups (warp w reads TMEM lanes
// 32 * (w % 4) ..).
#pragma once

#include <cuda.h>

#include "lm_norm.cuh"
#include "op_status.cuh"

namespace vxb {

enum OutType : int { kOutF32 = 0, kOutF16 = 1, kOutBF16 = 2 };

struct Fp8GemmArgs {
    int64_t N;                 // tokens
    int K, M;                  // inner extent, outputs
    int kb;                    // blocks of 128 k
    int row_tiles;             // tiles along the 128-row operand
    int64_t tiles;             // row_tiles * column tiles
    const float* xs;           // [N][kb], row stride xs_stride
    int64_t xs_stride;
    const float* ws;           // [ceil(M / 128)][kb]
    const float* bias;         // [M] or null
    void* y;                   // [N][M], row stride y_stride
    int64_t y_stride;
    int out_type;
    int split;                 // blocks of a cluster that share a tile's K
    int tma_out;               // the output's rows allow TMA stores
};

// Instruction descriptor, kind::f8f6f4: D fp32, A and B e4m3 (format 0), dense, both K-major.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int M, int N) {
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Issues the load of 16 TMEM columns without waiting for it.
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// Waits for this thread's TMEM loads; the N registers are not used before it.
template <int N>
__device__ __forceinline__ void tmem_ld_wait(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ void cluster_arrive_wait() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t saddr, uint32_t rank) {
    float4 v;
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}\n"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(saddr), "r"(rank)
        : "memory");
    return v;
}

__device__ __forceinline__ void st_cluster_u32(uint32_t saddr, uint32_t rank, uint32_t v) {
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n st.shared::cluster.u32 [a], %2;\n}\n" ::"r"(
                     saddr),
                 "r"(rank), "r"(v)
                 : "memory");
}

constexpr int kMaxSplit = 8;  // blocks of a cluster

template <int BN, bool WROWS>
struct Fp8Cfg {
    static constexpr int kGroups = BN > 64 ? 2 : 1;     // epilogue warpgroups
    static constexpr int kCols = BN / kGroups;          // columns of a warpgroup
    static constexpr int kThreads = 128 + 128 * kGroups;
    static constexpr bool kLarge = BN == 256;           // tiles fill the SMs
    static constexpr bool kSplits = !kLarge;
    static constexpr bool kTmaOut = kLarge;
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = BN * 128;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kOutBytes = kTmaOut ? 4 * kGroups * 4096 : 0;  // output staging, 4 KB a warp
    static constexpr int kStagesFit = (226 * 1024 - 2048 - kOutBytes) / kStageBytes;
    static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
    static constexpr int kBufCols = BN < 32 ? 32 : BN;
    static constexpr int kTmemCols = 2 * kBufCols;
    // split: partial sums over the stages, [BN][128] (weights as rows) or [128][BN + 4] (tokens
    // as rows), so that four outputs next to each other are four neighbouring words
    static constexpr int kRedBytes = 128 * (BN + 4) * 4;
    static __device__ __forceinline__ int red_at(int row, int col) { return WROWS ? col * 128 + row : row * (BN + 4) + col; }
    static constexpr int kSmemBytes = kStages * kStageBytes + kOutBytes + 1024 + 512;
    static_assert(kRedBytes <= kStages * kStageBytes, "partial sums fit the drained stages");
    static_assert(kSmemBytes <= 227 * 1024, "shared memory");
    static_assert(BN % 16 == 0 && BN <= 256, "UMMA N");
    static_assert(!WROWS || kGroups == 1, "weights as rows: at most 64 tokens wide");
};

__device__ __forceinline__ void store_out(void* y, int64_t i, float v, int type) {
    if (type == kOutF32) {
        static_cast<float*>(y)[i] = v;
    } else if (type == kOutF16) {
        static_cast<__half*>(y)[i] = __float2half_rn(v);
    } else {
        static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
    }
}

// NV consecutive outputs of a row from column c, 32 bytes at a time: vectors
// where the address and the row's end allow it.
template <typename T, int NV>
__device__ __forceinline__ void store_cols(T* y, int c, int M, const float* bias, const float* acc) {
    constexpr int kVec = 32 / sizeof(T);  // elements of a 32-byte store (a whole sector of the row)
    const bool fast = (reinterpret_cast<uintptr_t>(y + c) & 31) == 0;
#pragma unroll
    for (int i = 0; i < NV; i += kVec) {
        float v[kVec];
#pragma unroll
        for (int x = 0; x < kVec; ++x) v[x] = acc[i + x] + (bias && c + i + x < M ? bias[c + i + x] : 0.f);
        if (fast && c + i + kVec <= M) {
            uint32_t w[8];
            T* e = reinterpret_cast<T*>(w);
#pragma unroll
            for (int x = 0; x < kVec; ++x) e[x] = from_float<T>(v[x]);
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(y + c + i), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        } else {
#pragma unroll
            for (int x = 0; x < kVec; ++x)
                if (c + i + x < M) y[c + i + x] = from_float<T>(v[x]);
        }
    }
}

// The output through shared memory: a warp's 32 rows x NC columns in boxes of
// 32 rows x 128 bytes (128-byte swizzle), one at a time, by TMA store.
template <typename T, int NC>
__device__ __forceinline__ void store_tile(const void* tmap_y, uint8_t* buf, int lane, int row0, int c0,
                                           const Fp8GemmArgs& args, const float* acc) {
    constexpr int kCols = 128 / sizeof(T);  // columns of a box
    constexpr int kE = 16 / sizeof(T);
#pragma unroll
    for (int b = 0; b < NC; b += kCols) {
        if (lane == 0) bulk_wait_read<0>();  // the buffer's last store has read it
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; ++c) {        // 16-byte chunks of the row
            uint4 w;
            T* e = reinterpret_cast<T*>(&w);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                const int col = b + c * kE + i;
                e[i] = from_float<T>(acc[col] + (args.bias && c0 + col < args.M ? args.bias[c0 + col] : 0.f));
            }
            *reinterpret_cast<uint4*>(buf + lane * 128 + (((c ^ lane) & 7) << 4)) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < args.N && c0 + b < args.M) {
            tma_store_2d(tmap_y, buf, c0 + b, row0);
            bulk_commit();
        }
    }
}

template <int BN, bool WROWS>
__global__ void __launch_bounds__(Fp8Cfg<BN, WROWS>::kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_y, const Fp8GemmArgs args) {
    using Cfg = Fp8Cfg<BN, WROWS>;
    constexpr int S = Cfg::kStages;
    constexpr int NC = Cfg::kCols;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* out = stages + S * Cfg::kStageBytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(out + Cfg::kOutBytes);
    uint64_t* empty_bar = full_bar + S;
    uint64_t* tfull_bar = empty_bar + S;   // product [2] complete
    uint64_t* tempty_bar = tfull_bar + 2;  // product [2] read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int split = Cfg::kSplits ? args.split : 1;
    const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
    // this block's share of the k blocks
    const int kb_lo = static_cast<int>(static_cast<int64_t>(args.kb) * rank / split);
    const int kb_hi = static_cast<int>(static_cast<int64_t>(args.kb) * (rank + 1) / split);
    const int64_t tile0 = blockIdx.x / split;
    const int64_t tile_step = gridDim.x / split;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full_bar[i], 1);
            mbar_init(&empty_bar[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull_bar[i], 1);
            mbar_init(&tempty_bar[i], 4 * Cfg::kGroups);
        }
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    if (warp == 1) tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_dep_sync();

    if (warp == 0) {
        if (lane == 0) {
            // ---------------------------------------------- TMA producer --
            int it = 0;
            for (int64_t tile = tile0; tile < args.tiles && !*abort_flag; tile += tile_step) {
                const int r0 = static_cast<int>(tile % args.row_tiles) * 128;
                const int c0 = static_cast<int>(tile / args.row_tiles) * BN;
                for (int kb = kb_lo; kb < kb_hi; ++kb, ++it) {
                    const int st = it % S;
                    if (!op_wait(&empty_bar[st], ((it / S) & 1) ^ 1, abort_flag, kErrWaitEmpty)) break;
                    uint8_t* dst = stages + st * Cfg::kStageBytes;
                    mbar_arrive_expect_tx(&full_bar[st], Cfg::kStageBytes);
                    tma_load_2d(dst, &tmap_a, &full_bar[st], kb * 128, r0);
                    tma_load_2d(dst + Cfg::kABytes, &tmap_b, &full_bar[st], kb * 128, c0);
                }
            }
            if (*abort_flag) {  // give copies already in flight time to land
                const unsigned long long t0 = globaltimer_ns();
                while (globaltimer_ns() - t0 < 1000000ull) {
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            // ----------------------------------------------- MMA issuer --
            constexpr uint32_t idesc = make_idesc_e4m3(128, BN);
            int it = 0;
            bool ok = true;
            for (int64_t tile = tile0; tile < args.tiles && ok; tile += tile_step) {
                for (int kb = kb_lo; kb < kb_hi; ++kb, ++it) {
                    const int st = it % S, buf = it & 1;
                    if (!op_wait(&full_bar[st], (it / S) & 1, abort_flag, kErrWaitFull) ||
                        !op_wait(&tempty_bar[buf], ((it >> 1) & 1) ^ 1, abort_flag, kErrWaitAccum)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(stages + st * Cfg::kStageBytes);
                    const uint32_t b_addr = a_addr + Cfg::kABytes;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)  // K = 32 bytes per instruction inside the 128-byte rows
                        umma_f8(tmem_base + buf * Cfg::kBufCols, make_sdesc(a_addr + kk * 32, 16, 1024),
                                make_sdesc(b_addr + kk * 32, 16, 1024), idesc, kk != 0);
                    umma_commit(&empty_bar[st]);
                    umma_commit(&tfull_bar[buf]);
                }
            }
            if (!ok) {  // completes once every issued MMA is done: TMEM and the stages are idle after it
                umma_commit(&tfull_bar[0]);
                umma_commit(&tfull_bar[1]);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------------------------------------------- epilogue --
        const int eg = (warp - 4) >> 2;
        const int q = warp & 3;
        const int row = q * 32 + lane;
        const uint32_t t_row = tmem_base + eg * NC + (static_cast<uint32_t>(q * 32) << 16);
        int it = 0;
        for (int64_t tile = tile0; tile < args.tiles; tile += tile_step) {
            const int r = static_cast<int>(tile % args.row_tiles) * 128 + row;   // A row of this thread
            const int c0 = static_cast<int>(tile / args.row_tiles) * BN + eg * NC;  // first column of this group
            // scales: `own` of the thread's row, `col` of the columns (tokens as rows: one for
            // all of them; weights as rows: lane l keeps columns l and l + 32)
            const float *own_p, *col_p, *col_p2 = nullptr;
            if (WROWS) {
                own_p = args.ws + static_cast<int64_t>(r / 128) * args.kb;
                col_p = c0 + lane < args.N && lane < BN ? args.xs + (c0 + lane) * args.xs_stride : nullptr;
                col_p2 = BN > 32 && c0 + 32 + lane < args.N ? args.xs + (c0 + 32 + lane) * args.xs_stride : nullptr;
            } else {
                own_p = r < args.N ? args.xs + r * args.xs_stride : nullptr;
                col_p = c0 < args.M ? args.ws + static_cast<int64_t>(c0 / 128) * args.kb : nullptr;
            }
            float acc[NC];
#pragma unroll
            for (int i = 0; i < NC; ++i) acc[i] = 0.f;
            // (no read-only loads here: the kernel before, still running when this one starts, may
            // have written any operand)
            auto load = [](const float* p, int kb) { return p ? p[kb] : 0.f; };
            float own = 0.f, col = 0.f, col2 = 0.f;
            if (kb_lo < kb_hi) own = load(own_p, kb_lo), col = load(col_p, kb_lo), col2 = load(col_p2, kb_lo);
            bool ok = true;
            for (int kb = kb_lo; kb < kb_hi; ++kb, ++it) {
                const int buf = it & 1;
                float own_n = 0.f, col_n = 0.f, col2_n = 0.f;
                if (kb + 1 < kb_hi) {  // the next block's scales
                    own_n = load(own_p, kb + 1);
                    col_n = load(col_p, kb + 1);
                    col2_n = load(col_p2, kb + 1);
                }
                ok = op_wait(&tfull_bar[buf], (it >> 1) & 1, abort_flag, kErrWaitAccum);
                ok = __all_sync(0xffffffffu, ok && !*abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t t = t_row + buf * Cfg::kBufCols;
                constexpr int CH = NC < 32 ? NC : 32;  // columns in flight
                const float s = own * col;
#pragma unroll
                for (int c = 0; c < NC; c += CH) {
                    uint32_t v[CH];
#pragma unroll
                    for (int i = 0; i < CH; i += 16) tmem_ld16_async(t + c + i, v + i);
                    tmem_ld_wait<CH>(v);
#pragma unroll
                    for (int i = 0; i < CH; i += 2) {
                        float2 sc = make_float2(s, s);
                        if (WROWS) {
                            const float from = c + i < 32 ? col : col2;
                            sc.x = own * __shfl_sync(0xffffffffu, from, (c + i) & 31);
                            sc.y = own * __shfl_sync(0xffffffffu, from, (c + i + 1) & 31);
                        }
                        const float2 p = make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                        const float2 o = ffma2(sc, p, make_float2(acc[c + i], acc[c + i + 1]));
                        acc[c + i] = o.x;
                        acc[c + i + 1] = o.y;
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&tempty_bar[buf]);
                own = own_n;
                col = col_n;
                col2 = col2_n;
            }
            if (!ok) break;
            if (Cfg::kSplits && split > 1) {
                // partial sums over the drained stages (one tile per cluster)
                float* red = reinterpret_cast<float*>(stages);
#pragma unroll
                for (int i = 0; i < NC; ++i) red[Cfg::red_at(row, eg * NC + i)] = acc[i];
                break;
            }
            if (WROWS) {
                const float b = args.bias && r < args.M ? args.bias[r] : 0.f;
#pragma unroll
                for (int i = 0; i < NC; ++i)
                    if (r < args.M && c0 + i < args.N)
                        store_out(args.y, (c0 + i) * args.y_stride + r, acc[i] + b, args.out_type);
            } else if (Cfg::kTmaOut && args.tma_out) {
                uint8_t* buf = out + (warp - 4) * 4096;
                const int row0 = r - lane;
                if (args.out_type == kOutF32) {
                    store_tile<float, NC>(&tmap_y, buf, lane, row0, c0, args, acc);
                } else if (args.out_type == kOutF16) {
                    store_tile<__half, NC>(&tmap_y, buf, lane, row0, c0, args, acc);
                } else {
                    store_tile<__nv_bfloat16, NC>(&tmap_y, buf, lane, row0, c0, args, acc);
                }
            } else if (r < args.N) {
                const int64_t at = r * args.y_stride;
                if (args.out_type == kOutF32) {
                    store_cols<float, NC>(static_cast<float*>(args.y) + at, c0, args.M, args.bias, acc);
                } else if (args.out_type == kOutF16) {
                    store_cols<__half, NC>(static_cast<__half*>(args.y) + at, c0, args.M, args.bias, acc);
                } else {
                    store_cols<__nv_bfloat16, NC>(static_cast<__nv_bfloat16*>(args.y) + at, c0, args.M, args.bias, acc);
                }
            }
        }
    }

    if (Cfg::kTmaOut && args.tma_out && warp >= 4 && lane == 0) bulk_wait_all();  // stores done before the staging goes
    if (Cfg::kSplits && split > 1) {
        __syncwarp();
        if (*abort_flag && lane == 0)  // a rank that gave up takes the others with it
            for (int p = 0; p < split; ++p)
                st_cluster_u32(smem_u32(const_cast<const int*>(abort_flag)), p, *abort_flag);
        __syncwarp();
        cluster_arrive_wait();  // every rank's partial sums are written, or every rank's flag is set
        if (!*abort_flag && tile0 < args.tiles) {
            const int r0 = static_cast<int>(tile0 % args.row_tiles) * 128;
            const int64_t c0 = tile0 / args.row_tiles * BN;
            const uint32_t red = smem_u32(stages);
            // rank's share of the tile, four outputs of a row at a time
            constexpr int kQuads = WROWS ? 32 : BN / 4;  // of a row of outputs
            for (int i = rank * static_cast<int>(blockDim.x) + threadIdx.x; i < BN * 32; i += split * blockDim.x) {
                const int c = WROWS ? i / kQuads : i % kQuads * 4, rr = WROWS ? i % kQuads * 4 : i / kQuads;
                const int64_t n = WROWS ? c0 + c : r0 + rr;
                const int64_t m = WROWS ? r0 + rr : c0 + c;
                if (n >= args.N || m >= args.M) continue;
                float4 part[kMaxSplit];
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p)
                    part[p] = p < split ? ld_cluster_f32x4(red + Cfg::red_at(rr, c) * 4, p) : make_float4(0.f, 0.f, 0.f, 0.f);
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p)
                    v[0] += part[p].x, v[1] += part[p].y, v[2] += part[p].z, v[3] += part[p].w;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (m + x < args.M)
                        store_out(args.y, n * args.y_stride + m + x, v[x] + (args.bias ? args.bias[m + x] : 0.f),
                                  args.out_type);
            }
        }
        __syncwarp();
        cluster_arrive_wait();  // no rank leaves while its shared memory is read
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) record_abort(abort_flag);
    if (warp == 1) tmem_dealloc(tmem_base, Cfg::kTmemCols);
}

}  // namespace vxb
