// Language-model operators of the C ABI: RMS norm with 8-bit output, 8-bit
// block-scaled product, rotary positions into a paged cache, attention over
// a paged cache.  Arguments are checked before any CUDA call; every entry
// point only enqueues work on `stream`.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>
#include <utility>

#include "chunk_attn.cuh"
#include "fp8_gemm.cuh"
#include "fp8_gemv.cuh"
#include "host.h"
#include "lm_norm.cuh"
#include "lm_rotary.cuh"
#include "paged_attn.cuh"
#include "vxb.h"

using namespace vxb;

namespace {

constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024;  // rows addressed by 32-bit tile coordinates

int bad(const char* op, const char* what) {
    return fail(VXB_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int elem_size(int type) { return type == VXB_TYPE_F32 ? 4 : 2; }

bool is_float(int type) { return type == VXB_TYPE_F32 || type == VXB_TYPE_F16 || type == VXB_TYPE_BF16; }

// An output's rows of `width` elements along axes of (extent, stride): does each have memory of
// its own?  (As axes nest, the next one has to step over the whole of those inside it.)
struct Axis {
    int64_t extent, stride;
};
bool rows_apart(int64_t width, Axis a, Axis b, Axis c = {1, 0}) {
    const auto step = [](const Axis& x) {  // (an axis of one element has any stride)
        return x.extent < 2 ? static_cast<__int128>(0) : x.stride < 0 ? -static_cast<__int128>(x.stride) : x.stride;
    };
    if (step(b) < step(a)) std::swap(a, b);
    if (step(c) < step(b)) std::swap(b, c);
    if (step(b) < step(a)) std::swap(a, b);
    __int128 span = width;
    for (const Axis& x : {a, b, c}) {
        if (x.extent < 2) continue;
        if (step(x) < span) return false;
        span += step(x) * (x.extent - 1);
    }
    return true;
}

int this_device(int* dev) {
    CUDA_TRY(cudaGetDevice(dev));
    return VXB_OK;
}

// No C++ exception leaves the C ABI.
template <typename F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return VXB_ERR_OUT_OF_MEMORY;
    } catch (...) {
        return VXB_ERR_BACKEND;
    }
}

// ---------------------------------------------------------------- rms norm --

template <typename T, int NV, bool VEC>
cudaError_t launch_norm_v(const NormArgs& a, int threads, cudaStream_t st) {
    const dim3 g(static_cast<unsigned>(a.N)), b(threads);
    if (a.scale)
        return a.res ? launch_pdl(rms_norm_kernel<T, NV, VEC, true, true>, g, b, 0, st, a)
                     : launch_pdl(rms_norm_kernel<T, NV, VEC, false, true>, g, b, 0, st, a);
    return a.res ? launch_pdl(rms_norm_kernel<T, NV, VEC, true, false>, g, b, 0, st, a)
                 : launch_pdl(rms_norm_kernel<T, NV, VEC, false, false>, g, b, 0, st, a);
}

template <typename T>
cudaError_t launch_norm(const NormArgs& a, bool vec, cudaStream_t st) {
    const int vecs = (a.C + 7) / 8;
    const auto threads = [&](int nv) { return std::max(32, (vecs + 32 * nv - 1) / (32 * nv) * 32); };
    if (!vec) {  // strides or widths that do not allow 16-byte vectors
        if (threads(2) <= 1024) return launch_norm_v<T, 2, false>(a, threads(2), st);
        return launch_norm_v<T, 4, false>(a, threads(4), st);
    }
    if (threads(1) <= 256) return launch_norm_v<T, 1, true>(a, threads(1), st);
    if (threads(2) <= 1024) return launch_norm_v<T, 2, true>(a, threads(2), st);
    return launch_norm_v<T, 4, true>(a, threads(4), st);
}

}  // namespace

extern "C" int vxb_rms_norm(int type, int64_t N, int C, const void* x, int64_t x_stride, const void* residual,
                            int64_t residual_stride, void* sum, int64_t sum_stride, int w_type, const void* w,
                            float eps, int y_type, void* y, int64_t y_stride, float* y_scale, int64_t scale_stride,
                            void* stream) {
    const char* op = "rms_norm";
    return guarded([&]() -> int {
        if (!is_float(type)) return bad(op, "x must be f32, f16 or bf16");
        if (w_type != type && w_type != VXB_TYPE_F32) return bad(op, "the weight must be of x's type or f32");
        if (y_type != type && y_type != VXB_TYPE_E4M3) return bad(op, "the output must be of x's type or e4m3");
        if (N < 0 || N > kMaxRows) return bad(op, "bad row count");
        if (C < 1 || C > 32768) return bad(op, "width must be 1..32768");
        if (!(eps >= 0.f) || std::isinf(eps)) return bad(op, "eps must be finite and not negative");
        const bool q8 = y_type == VXB_TYPE_E4M3;
        if (N == 0) return VXB_OK;
        if (!x || !w || !y) return bad(op, "null argument");
        if (q8 != (y_scale != nullptr)) return bad(op, "e4m3 output takes a scale, other outputs none");
        if (x_stride < C || y_stride < C || (residual && residual_stride < C) || (sum && sum_stride < C) ||
            (q8 && scale_stride < (C + kScaleBlock - 1) / kScaleBlock))
            return bad(op, "a row stride is smaller than the row");
        const int es = elem_size(type);
        if (!aligned(x, es) || !aligned(residual, es) || !aligned(sum, es) || !aligned(w, elem_size(w_type)) ||
            !aligned(y, q8 ? 1 : es) || !aligned(y_scale, 4))
            return bad(op, "a pointer is not aligned to its element");
        NormArgs a{x,  residual, sum, w,        y,        y_scale,      N, x_stride, residual_stride, sum_stride,
                   y_stride, scale_stride, C, w_type == VXB_TYPE_F32 && type != VXB_TYPE_F32, eps};
        const bool vec = C % 8 == 0 && aligned(x, 16) && aligned(w, 16) && aligned(y, q8 ? 8 : 16) && aligned(residual, 16) &&
                         aligned(sum, 16) && x_stride % 8 == 0 && y_stride % 8 == 0 &&
                         (!residual || residual_stride % 8 == 0) && (!sum || sum_stride % 8 == 0);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        CUDA_TRY(type == VXB_TYPE_F32   ? launch_norm<float>(a, vec, st)
                 : type == VXB_TYPE_F16 ? launch_norm<__half>(a, vec, st)
                                        : launch_norm<__nv_bfloat16>(a, vec, st));
        return VXB_OK;
    });
}

// ------------------------------------------------------------------ rotary --

namespace {

template <typename T, int VEC>
cudaError_t launch_rotary(const RotaryArgs& a, bool inter, cudaStream_t st) {
    const dim3 g(static_cast<unsigned>((a.N + a.tokens - 1) / a.tokens)), b(kRotThreads);
    return inter ? launch_pdl(rotary_kernel<T, VEC, true>, g, b, 0, st, a)
                 : launch_pdl(rotary_kernel<T, VEC, false>, g, b, 0, st, a);
}

bool head_vec(const void* p, int64_t token, int64_t head, int vec) {
    return !p || (aligned(p, 16) && token % vec == 0 && head % vec == 0);
}

int run_rotary(const char* op, int type, RotaryArgs a, int interleaved, void* stream) {
    if (!is_float(type)) return bad(op, "the type must be f32, f16 or bf16");
    if (a.N < 0 || a.N > kMaxRows) return bad(op, "bad token count");
    if (a.Hq < 1 || a.Hk < 0 || a.Hq > 65535 || a.Hk > 65535) return bad(op, "bad head count");
    if (a.D < 1 || a.D > 1024) return bad(op, "head width must be 1..1024");
    if (a.R < 2 || a.R % 2 || a.R > a.D || a.R > kRotMaxR)
        return bad(op, "the rotated part must be even, at most the head and at most 256");
    if (std::isnan(a.factor) || std::isinf(a.factor)) return bad(op, "the factor must be finite");
    if (a.N == 0) return VXB_OK;
    if (!a.q.p || !a.q_out.p || !a.positions || !a.inv_freq) return bad(op, "null argument");
    const int es = elem_size(type);
    for (const void* p : {static_cast<const void*>(a.q.p), static_cast<const void*>(a.q_out.p),
                          static_cast<const void*>(a.k.p), static_cast<const void*>(a.k_out.p),
                          static_cast<const void*>(a.v.p), static_cast<const void*>(a.k_cache),
                          static_cast<const void*>(a.v_cache)})
        if (!aligned(p, es)) return bad(op, "a pointer is not aligned to its element");
    if (!aligned(a.positions, 8) || !aligned(a.slots, 8) || !aligned(a.inv_freq, 4))
        return bad(op, "positions, slots or frequencies are not aligned to their elements");
    if (!rows_apart(a.D, {a.N, a.q_out.token}, {a.Hq, a.q_out.head}) ||
        (a.k_out.p && !rows_apart(a.D, {a.N, a.k_out.token}, {a.Hk, a.k_out.head})) ||
        (a.k_cache && a.cache_slots > 0 &&
         !rows_apart(a.D, {a.cache_slots / a.page_size, a.page_stride}, {a.page_size, a.slot_stride},
                     {a.Hk, a.cache_head})))
        return bad(op, "heads of an output overlap");
    const int vec = 16 / es;
    const bool v = a.D % vec == 0 && a.R % (2 * vec) == 0 && head_vec(a.q.p, a.q.token, a.q.head, vec) &&
                   head_vec(a.q_out.p, a.q_out.token, a.q_out.head, vec) &&
                   head_vec(a.k.p, a.k.token, a.k.head, vec) &&
                   head_vec(a.k_out.p, a.k_out.token, a.k_out.head, vec) &&
                   head_vec(a.v.p, a.v.token, a.v.head, vec) &&
                   head_vec(a.k_cache, a.page_stride, a.slot_stride, vec) &&
                   head_vec(a.v_cache, a.page_stride, a.cache_head, vec);
    int dev = 0, rc = this_device(&dev);
    if (rc) return rc;
    a.tokens = static_cast<int>(std::min<int64_t>(kRotTokens, std::max<int64_t>(1, a.N / (4 * num_sms(dev)))));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == VXB_TYPE_F32) {
        CUDA_TRY(v ? (launch_rotary<float, 4>(a, interleaved, st)) : (launch_rotary<float, 1>(a, interleaved, st)));
    } else if (type == VXB_TYPE_F16) {
        CUDA_TRY(v ? (launch_rotary<__half, 8>(a, interleaved, st)) : (launch_rotary<__half, 1>(a, interleaved, st)));
    } else {
        CUDA_TRY(v ? (launch_rotary<__nv_bfloat16, 8>(a, interleaved, st))
                   : (launch_rotary<__nv_bfloat16, 1>(a, interleaved, st)));
    }
    return VXB_OK;
}

}  // namespace

extern "C" int vxb_rotary(int type, int64_t N, int Hq, int Hk, int D, int R, int interleaved, float factor,
                          const int64_t* positions, const float* inv_freq, const void* q, int64_t q_token,
                          int64_t q_head, void* q_out, int64_t qo_token, int64_t qo_head, const void* k,
                          int64_t k_token, int64_t k_head, void* k_out, int64_t ko_token, int64_t ko_head,
                          void* stream) {
    return guarded([&]() -> int {
        if ((k != nullptr) != (k_out != nullptr)) return bad("rotary", "keys and their output come together");
        if (k && Hk < 1 && N > 0) return bad("rotary", "bad head count");
        RotaryArgs a{};
        a.q = {const_cast<void*>(q), q_token, q_head};
        a.q_out = {q_out, qo_token, qo_head};
        a.k = {const_cast<void*>(k), k_token, k_head};
        a.k_out = {k_out, ko_token, ko_head};
        a.positions = positions;
        a.inv_freq = inv_freq;
        a.page_size = 1;
        a.N = N, a.Hq = Hq, a.Hk = Hk, a.D = D, a.R = R, a.factor = factor;
        return run_rotary("rotary", type, a, interleaved, stream);
    });
}

extern "C" int vxb_rotary_append(int type, int64_t N, int Hq, int Hk, int D, int R, int interleaved, float factor,
                                 const int64_t* positions, const int64_t* slots, const float* inv_freq,
                                 const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t qo_token,
                                 int64_t qo_head, const void* k, int64_t k_token, int64_t k_head, const void* v,
                                 int64_t v_token, int64_t v_head, void* k_cache, void* v_cache, int64_t pages,
                                 int page_size, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
                                 void* stream) {
    const char* op = "rotary_append";
    return guarded([&]() -> int {
        if (pages < 0 || page_size < 1 || pages > (int64_t(1) << 40) / page_size) return bad(op, "bad cache extents");
        if (Hk < 1) return bad(op, "bad head count");
        if (N > 0 && (!k || !v || !slots || !k_cache || !v_cache)) return bad(op, "null argument");
        RotaryArgs a{};
        a.q = {const_cast<void*>(q), q_token, q_head};
        a.q_out = {q_out, qo_token, qo_head};
        a.k = {const_cast<void*>(k), k_token, k_head};
        a.v = {const_cast<void*>(v), v_token, v_head};
        a.positions = positions;
        a.inv_freq = inv_freq;
        a.slots = slots;
        a.k_cache = k_cache;
        a.v_cache = v_cache;
        a.cache_slots = pages * page_size;
        a.page_stride = page_stride, a.slot_stride = slot_stride, a.cache_head = head_stride;
        a.page_size = page_size;
        a.N = N, a.Hq = Hq, a.Hk = Hk, a.D = D, a.R = R, a.factor = factor;
        return run_rotary(op, type, a, interleaved, stream);
    });
}

// ------------------------------------------------------------- fp8 product --

namespace {

// e4m3 matrix [rows][K] (row pitch in bytes), boxes of 128 k x box_rows.
int make_tmap_e4m3(CUtensorMap* m, const void* base, uint64_t K, uint64_t rows, uint64_t pitch, uint32_t box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(VXB_ERR_BACKEND, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {K, rows};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t box[2] = {128, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VXB_ERR_BACKEND, "cuTensorMapEncodeTiled (e4m3) failed: " + std::to_string(r));
    return VXB_OK;
}

// Output [rows][cols] (row pitch in bytes), boxes of 128 bytes x 32 rows.
int make_tmap_out(CUtensorMap* m, void* base, int type, uint64_t cols, uint64_t rows, uint64_t pitch) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(VXB_ERR_BACKEND, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t box[2] = {type == kOutF32 ? 32u : 64u, 32};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(m, type == kOutF32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : type == kOutF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                     2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VXB_ERR_BACKEND, "cuTensorMapEncodeTiled (output) failed: " + std::to_string(r));
    return VXB_OK;
}

struct Fp8Operands {
    const void *x, *w;
    int64_t x_stride, w_stride;
};

template <int BN, bool WROWS>
int launch_fp8(const Fp8Operands& o, Fp8GemmArgs a, int dev, cudaStream_t st) {
    using Cfg = Fp8Cfg<BN, WROWS>;
    static std::atomic<bool> attr[64];
    int rc = allow_smem(fp8_gemm_kernel<BN, WROWS>, Cfg::kSmemBytes, attr, dev);
    if (rc) return rc;
    const int64_t rows = WROWS ? a.M : a.N, cols = WROWS ? a.N : a.M;
    a.row_tiles = static_cast<int>((rows + 127) / 128);
    a.tiles = a.row_tiles * ((cols + BN - 1) / BN);
    // fewer tiles than SMs: K is shared by the blocks of a cluster, each with two k blocks at least
    const int sms = num_sms(dev);
    a.split = 1;
    while (Cfg::kSplits && a.split < kMaxSplit && a.tiles * a.split * 2 <= sms && a.kb >= a.split * 4) a.split *= 2;
    CUtensorMap tx, tw, ty = {};
    if (Cfg::kTmaOut) {
        const int es = a.out_type == kOutF32 ? 4 : 2;
        a.tma_out = aligned(a.y, 16) && a.y_stride * es % 16 == 0;
        if (a.tma_out && (rc = make_tmap_out(&ty, a.y, a.out_type, a.M, a.N, a.y_stride * es))) return rc;
    }
    if ((rc = make_tmap_e4m3(&tx, o.x, a.K, a.N, o.x_stride, WROWS ? BN : 128))) return rc;
    if ((rc = make_tmap_e4m3(&tw, o.w, a.K, a.M, o.w_stride, WROWS ? 128 : BN))) return rc;
    const int64_t grid = a.split > 1 ? a.tiles * a.split : std::min<int64_t>(a.tiles, sms);
    CUDA_TRY(launch_pdl_cluster(fp8_gemm_kernel<BN, WROWS>, dim3(static_cast<unsigned>(grid)), dim3(Cfg::kThreads),
                                a.split, Cfg::kSmemBytes, st, WROWS ? tw : tx, WROWS ? tx : tw, ty, a));
    return VXB_OK;
}

template <int NT>
int launch_fp8_gemv(const Fp8Operands& o, const Fp8GemmArgs& a, cudaStream_t st) {
    constexpr int rows = kGemvRows * kGemvThreads / 32;
    CUDA_TRY(launch_pdl(fp8_gemv_kernel<NT>, dim3((a.M + rows - 1) / rows), dim3(kGemvThreads), 0, st,
                        static_cast<const uint8_t*>(o.x), o.x_stride, static_cast<const uint8_t*>(o.w), o.w_stride, a));
    return VXB_OK;
}

}  // namespace

extern "C" int vxb_fp8_product(int64_t N, int K, int M, const void* x, int64_t x_stride, const float* x_scale,
                               int64_t x_scale_stride, const void* w, int64_t w_stride, const float* w_scale,
                               const float* bias, int y_type, void* y, int64_t y_stride, void* stream) {
    const char* op = "fp8_product";
    return guarded([&]() -> int {
        if (N < 0 || N > kMaxRows) return bad(op, "bad row count");
        if (K < 16 || K % 16 || K > (1 << 24)) return bad(op, "K must be a multiple of 16");
        if (M < 1 || M > (1 << 30)) return bad(op, "bad output width");
        if (!is_float(y_type)) return bad(op, "the output must be f32, f16 or bf16");
        if (N == 0) return VXB_OK;
        if (!x || !x_scale || !w || !w_scale || !y) return bad(op, "null argument");
        const int kb = (K + kScaleBlock - 1) / kScaleBlock;
        if (x_stride < K || w_stride < K || y_stride < M || x_scale_stride < kb)
            return bad(op, "a row stride is smaller than the row");
        if (!aligned(x, 16) || !aligned(w, 16) || x_stride % 16 || w_stride % 16)
            return bad(op, "TMA operand needs 16-byte aligned base and row pitch");
        if (!aligned(x_scale, 4) || !aligned(w_scale, 4) || !aligned(bias, 4) || !aligned(y, elem_size(y_type)))
            return bad(op, "a pointer is not aligned to its element");
        int dev = 0, rc = this_device(&dev);
        if (rc) return rc;
        Fp8GemmArgs a{};
        a.N = N, a.K = K, a.M = M, a.kb = kb;
        a.xs = x_scale, a.xs_stride = x_scale_stride, a.ws = w_scale, a.bias = bias;
        a.y = y, a.y_stride = y_stride;
        a.out_type = y_type == VXB_TYPE_F32 ? kOutF32 : y_type == VXB_TYPE_F16 ? kOutF16 : kOutBF16;
        const Fp8Operands o{x, w, x_stride, w_stride};
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        // Few tokens: weights as rows, so that a tile's 128 rows are all in use and the tokens
        // set its width.  So too where there are more tokens but few tiles of 128 x 128
        // (256 x 1024 -> 64: 4.2 us against 5.9; 77 x 1536 -> 1001: 5.5 against 6.5; with 32
        // such tiles the other way round, 128 x 4096 -> 4096: 13.6 against 9.8): 64 tokens wide
        // if that fills the SMs with K split, else 32.  256 outputs wide where that fills them.
        const int sms = num_sms(dev);
        const int64_t rows = (int64_t(M) + 127) / 128;
        // One or two tokens and a few MB of weights in rows of at most 4096: no tensor cores, no
        // chain of set-up (measurements beside the kernel).
        if (N == 1 && K <= 4096 && int64_t(K) * M <= (1 << 24)) return launch_fp8_gemv<1>(o, a, st);
        if (N == 2 && K <= 2048 && int64_t(K) * M <= (1 << 23)) return launch_fp8_gemv<2>(o, a, st);
        if (N <= 16) return launch_fp8<16, true>(o, a, dev, st);
        if (N <= 32) return launch_fp8<32, true>(o, a, dev, st);
        if (N <= 64) return launch_fp8<64, true>(o, a, dev, st);
        if ((N + 127) / 128 * rows <= 16) {
            const int64_t most = (N + 63) / 64 * rows * std::min(kMaxSplit, std::max(1, kb / 2));
            if (most * 5 >= sms * 4) return launch_fp8<64, true>(o, a, dev, st);
            return launch_fp8<32, true>(o, a, dev, st);
        }
        if ((N + 127) / 128 * ((M + 255) / 256) >= sms) return launch_fp8<256, false>(o, a, dev, st);
        return launch_fp8<128, false>(o, a, dev, st);
    });
}

// --------------------------------------------------------- paged attention --

namespace {

constexpr int kAttnMaxD = 128;

// Which kernel a call takes and into how many parts its keys are split; a
// function of the extents alone, so that the workspace is known beforehand.
struct AttnPlan {
    bool chunk;    // tensor-core kernel for chunks
    int rows;      // else: rows of a tile
    int tokens;    // tokens of a tile
    int64_t slots; // tile slots over the tokens
    int groups;    // tiles that a group of heads takes
    int splits;
};

AttnPlan attn_plan(int64_t N, int B, int Hq, int Hk, int max_pages, int page_size, int sms) {
    const int G = Hq / Hk;
    const int64_t keys = int64_t(max_pages) * page_size;
    AttnPlan p{};
    p.chunk = N * G > int64_t(B) * 64;
    p.rows = p.chunk ? 128 : N * G > int64_t(B) * 16 ? 32 : 16;
    const int GT = std::min(G, p.rows);
    // tokens of a tile; single tokens (no more of them than sequences) get a tile each
    p.tokens = p.chunk ? 2 * (128 / GT) : N <= B ? 1 : std::max(1, p.rows / G);
    p.slots = p.tokens == 1 ? N : N / p.tokens + B;
    p.groups = (G + GT - 1) / GT;
    // as many parts as fill the device (two blocks per SM, one of the chunk kernel), each of 256
    // keys (512) at least
    const int64_t blocks = std::max<int64_t>(1, p.slots * Hk * p.groups);
    const int64_t want = (p.chunk ? sms : 2 * int64_t(sms)) / blocks;
    p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, keys / (p.chunk ? 512 : 256), kAttnMaxSplits})));
    return p;
}

int make_tmap_16(CUtensorMap* m, bool bf16, const void* base, int rank, const cuuint64_t* dims,
                 const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(VXB_ERR_BACKEND, "cuTensorMapEncodeTiled unavailable");
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                     const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VXB_ERR_BACKEND, "cuTensorMapEncodeTiled (16 bit) failed: " + std::to_string(r));
    return VXB_OK;
}

// A cache [pages][page_size][Hk][D]: boxes of 64 dims and min(page_size, keys) keys of one head.
int make_tmap_cache(CUtensorMap* m, bool bf16, const void* base, const AttnArgs& a, int keys) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.page_size),
                                static_cast<cuuint64_t>(a.Hk), static_cast<cuuint64_t>(a.pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.slot_stride) * 2, static_cast<cuuint64_t>(a.cache_head) * 2,
                                   static_cast<cuuint64_t>(a.page_stride) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(std::min(a.page_size, keys)), 1, 1};
    return make_tmap_16(m, bf16, base, 4, dims, strides, box);
}

template <typename T>
int launch_join(const AttnArgs& a, cudaStream_t st) {
    // a block per row, or a warp where there are rows enough for the device
    const int64_t rows = a.N * a.Hq;
    if (rows < 2048) {
        CUDA_TRY(launch_pdl(attn_join_kernel<T, 4>, dim3(static_cast<unsigned>(rows)), dim3(128), 0, st, a));
    } else {
        CUDA_TRY(launch_pdl(attn_join_kernel<T, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, st, a));
    }
    return VXB_OK;
}

template <typename T, int DP>
int launch_chunk(const AttnArgs& a, const AttnPlan& p, int dev, cudaStream_t st) {
    using Cfg = ChunkCfg<DP>;
    constexpr bool bf = !std::is_same<T, __half>::value;
    static std::atomic<bool> attr[64];
    int rc = allow_smem(attn_chunk_kernel<T, DP>, Cfg::kSmemBytes, attr, dev);
    if (rc) return rc;
    CUtensorMap tq = {}, tk = {}, tv = {};
    if (a.pages > 0) {
        const cuuint32_t GT = std::min(a.G, 128);
        const cuuint64_t qd[3] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.Hq),
                                  static_cast<cuuint64_t>(a.N)};
        const cuuint64_t qs[2] = {static_cast<cuuint64_t>(a.q_head) * 2, static_cast<cuuint64_t>(a.q_token) * 2};
        const cuuint32_t qb[3] = {64, GT, 128 / GT};
        if ((rc = make_tmap_16(&tq, bf, a.q, 3, qd, qs, qb))) return rc;
        if ((rc = make_tmap_cache(&tk, bf, a.k, a, kCkStep)) || (rc = make_tmap_cache(&tv, bf, a.v, a, kCkStep)))
            return rc;
    }
    const dim3 g(static_cast<unsigned>(p.slots * a.Hk * p.groups), 1, static_cast<unsigned>(p.splits));
    CUDA_TRY(launch_pdl(attn_chunk_kernel<T, DP>, g, dim3(kCkThreads), Cfg::kSmemBytes, st, tq, tk, tv, a));
    return a.splits > 1 ? launch_join<T>(a, st) : VXB_OK;
}

template <typename T, int DP, int MT, int KW>
int launch_rows(const AttnArgs& a, const AttnPlan& p, int dev, cudaStream_t st) {
    using Cfg = AttnCfg<T, DP, MT, KW>;
    static std::atomic<bool> attr[64];
    int rc = allow_smem(attn_rows_kernel<T, DP, MT, KW>, Cfg::kSmemBytes, attr, dev);
    if (rc) return rc;
    const dim3 g(static_cast<unsigned>(p.slots), static_cast<unsigned>(a.Hk * p.groups), static_cast<unsigned>(p.splits));
    constexpr bool bf = !std::is_same<T, __half>::value;
    CUtensorMap tk = {}, tv = {};
    if (a.pages > 0 && ((rc = make_tmap_cache(&tk, bf, a.k, a, Cfg::kStep)) ||
                        (rc = make_tmap_cache(&tv, bf, a.v, a, Cfg::kStep))))
        return rc;
    CUDA_TRY(launch_pdl(attn_rows_kernel<T, DP, MT, KW>, g, dim3(kAttnThreads), Cfg::kSmemBytes, st, tk, tv, a));
    return a.splits > 1 ? launch_join<T>(a, st) : VXB_OK;
}

template <typename T>
int launch_attn(const AttnArgs& a, const AttnPlan& p, int dev, cudaStream_t st) {
    if (p.chunk) return a.D <= 64 ? launch_chunk<T, 64>(a, p, dev, st) : launch_chunk<T, 128>(a, p, dev, st);
    if (a.D <= 64) return p.rows == 16 ? launch_rows<T, 64, 1, 2>(a, p, dev, st) : launch_rows<T, 64, 2, 2>(a, p, dev, st);
    return p.rows == 16 ? launch_rows<T, 128, 1, 1>(a, p, dev, st) : launch_rows<T, 128, 2, 1>(a, p, dev, st);
}

int check_attn(const char* op, int64_t N, int B, int Hq, int Hk, int D, int max_pages, int page_size) {
    // (positions and windows are 32-bit differences of these)
    if (N < 0 || N > (1 << 30) || B < 0 || B > (1 << 24)) return bad(op, "bad token or sequence count");
    if (Hk < 1 || Hq < 1 || Hq % Hk || Hq > 4096) return bad(op, "query heads must be a multiple of key heads");
    if (D < 8 || D % 8 || D > kAttnMaxD) return bad(op, "head width must be a multiple of 8, 8..128");
    if (page_size < 16 || (page_size & (page_size - 1)) || page_size > (1 << 20))
        return bad(op, "page size must be a power of two, 16 at least");
    if (max_pages < 0 || int64_t(max_pages) * page_size >= (int64_t(1) << 30))
        return bad(op, "a table row must cover less than 2^30 keys");
    return VXB_OK;
}

}  // namespace

extern "C" int64_t vxb_paged_attention_workspace(int64_t N, int B, int Hq, int Hk, int D, int max_pages,
                                                 int page_size) {
    return guarded([&]() -> int { return check_attn("paged_attention", N, B, Hq, Hk, D, max_pages, page_size); })
               ? -1
               : [&]() -> int64_t {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return -1;
        const int splits = attn_plan(N, B, Hq, Hk, max_pages, page_size, num_sms(dev)).splits;
        return splits > 1 ? int64_t(splits) * N * Hq * (D + 1) * 4 : 0;
    }();
}

extern "C" int vxb_paged_attention(int type, int64_t N, int B, int Hq, int Hk, int D, const void* q, int64_t q_token,
                                   int64_t q_head, const void* k_cache, const void* v_cache, int64_t pages,
                                   int page_size, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
                                   const int32_t* block_table, int64_t table_stride, int max_pages,
                                   const int32_t* cu_q, const int32_t* kv_len, float scale, int window, void* out,
                                   int64_t o_token, int64_t o_head, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
    const char* op = "paged_attention";
    return guarded([&]() -> int {
        int rc = check_attn(op, N, B, Hq, Hk, D, max_pages, page_size);
        if (rc) return rc;
        if (type != VXB_TYPE_F16 && type != VXB_TYPE_BF16) return bad(op, "the type must be f16 or bf16");
        if (pages < 0 || pages >= (int64_t(1) << 31)) return bad(op, "bad page count");
        if (window < 0) return bad(op, "the window must not be negative");
        if (std::isnan(scale) || std::isinf(scale * 1.4426950408889634f))  // (in log2 units)
            return bad(op, "the scale must be finite and below 2.3e38");
        if (N == 0 || B == 0) return VXB_OK;
        if (!q || !out || !cu_q || !kv_len) return bad(op, "null argument");
        if (max_pages > 0 && (!block_table || (pages > 0 && (!k_cache || !v_cache))))
            return bad(op, "null argument");
        if (max_pages > 0 && B > 1 && table_stride < max_pages) return bad(op, "a table row overlaps the next");
        if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || q_token % 8 || q_head % 8 ||
            page_stride % 8 || slot_stride % 8 || head_stride % 8)
            return bad(op, "queries and cache need 16-byte aligned bases and strides");
        constexpr int64_t far = int64_t(1) << 38;  // a tensor map's strides are below 2^40 bytes
        if (q_token < 0 || q_head < 0 || page_stride < 0 || slot_stride < 0 || head_stride < 0 || q_token > far ||
            q_head > far || page_stride > far || slot_stride > far || head_stride > far)
            return bad(op, "strides of queries and cache must not be negative or beyond 2^38");
        if (!aligned(out, 2) || !aligned(block_table, 4) || !aligned(cu_q, 4) || !aligned(kv_len, 4))
            return bad(op, "a pointer is not aligned to its element");
        if (!rows_apart(D, {N, o_token}, {Hq, o_head})) return bad(op, "heads of the output overlap");
        int dev = 0;
        if ((rc = this_device(&dev))) return rc;
        AttnArgs a{};
        a.q = q, a.q_token = q_token, a.q_head = q_head;
        a.out = out, a.o_token = o_token, a.o_head = o_head;
        a.k = k_cache, a.v = v_cache;
        a.page_stride = page_stride, a.slot_stride = slot_stride, a.cache_head = head_stride;
        a.table = block_table, a.table_stride = table_stride, a.cu_q = cu_q, a.kv_len = kv_len;
        a.N = N, a.pages = pages, a.B = B, a.Hq = Hq, a.Hk = Hk, a.G = Hq / Hk, a.D = D;
        // (a cache without pages: no key is seen, nothing is loaded)
        a.page_size = page_size, a.max_pages = pages ? max_pages : 0;
        a.window = window < int64_t(max_pages) * page_size ? window : 0;  // (as wide as the table: none)
        while ((1 << a.page_shift) < page_size) ++a.page_shift;
        // (a scale of 0 weighs every key alike; the smallest normal number does too, and keeps
        // a masked score, -inf, times it -inf)
        a.scale_log2 = scale == 0.f ? 1.17549435e-38f : scale * 1.4426950408889634f;
        const AttnPlan p = attn_plan(N, B, Hq, Hk, max_pages, page_size, num_sms(dev));
        a.splits = p.splits;
        a.tokens = p.tokens;
        if (a.splits > 1) {
            const int64_t need = int64_t(a.splits) * N * Hq * (D + 1) * 4;
            if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
                return bad(op, "the workspace is smaller than vxb_paged_attention_workspace says, or not 16-byte aligned");
            a.part_o = static_cast<float*>(workspace);
            a.part_lse = a.part_o + int64_t(a.splits) * N * Hq * D;
        }
        if (p.slots * Hk * p.groups >= (int64_t(1) << 31)) return bad(op, "too many tokens for one call");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        return type == VXB_TYPE_F16 ? launch_attn<__half>(a, p, dev, st)
                                    : launch_attn<__nv_bfloat16>(a, p, dev, st);
    });
}

// ------------------------------------------------------------ failed waits --

extern "C" int vxb_operators_sync(int timeout_ms, void* stream) {
    return guarded([&]() -> int {
        if (timeout_ms < 0) return bad("operators_sync", "the timeout must not be negative");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        int code = 0;
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        CUDA_TRY(cudaStreamIsCapturing(st, &capture));
        if (capture != cudaStreamCaptureStatusNone) return bad("operators_sync", "the stream is being captured");
        if (int rc = wait_stream(st, timeout_ms)) return rc;
        CUDA_TRY(cudaMemcpyFromSymbolAsync(&code, g_op_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
        CUDA_TRY(cudaStreamSynchronize(st));
        if (!code) return VXB_OK;
        const int none = 0;
        CUDA_TRY(cudaMemcpyToSymbolAsync(g_op_status, &none, sizeof(int), 0, cudaMemcpyHostToDevice, st));
        CUDA_TRY(cudaStreamSynchronize(st));
        return fail(VXB_ERR_DEVICE_STATUS, "a language-model operator's bounded wait failed (code " +
                                               std::to_string(code) + "): its output is not valid");
    });
}

extern "C" int vxb_debug_operators_wait_probe(int limit_us, void* stream) {
    return guarded([&]() -> int {
        if (limit_us < 1 || limit_us > 2000000) return bad("operators_wait_probe", "bad limit");
        op_wait_probe_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<unsigned long long>(limit_us) *
                                                                              1000ull);
        CUDA_TRY(cudaGetLastError());
        return VXB_OK;
    });
}
