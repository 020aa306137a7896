// Python entry points of the language-model operators (module _vxb_native):
// they take torch tensors, check them and call the C ABI of libvxb.
//
// These calls run for every token of a stream, next to kernels of 2 to 10 us,
// and cost 10 to 15 us of interpreted checks and foreign-function conversions
// when they were written in Python; here they cost the launch.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <string>

#include "vxb.h"

namespace {

PyObject* g_error = nullptr;  // vxb.VxbError

struct Refused {
    int code;
    std::string what;
};

[[noreturn]] void refuse(const std::string& what) { throw Refused{VXB_ERR_INVALID_ARGUMENT, what}; }

constexpr int kInt32 = -32, kInt64 = -64, kUint8 = -8;

int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return VXB_TYPE_F32;
        case at::kHalf: return VXB_TYPE_F16;
        case at::kBFloat16: return VXB_TYPE_BF16;
        case at::kFloat8_e4m3fn: return VXB_TYPE_E4M3;
        case at::kInt: return kInt32;
        case at::kLong: return kInt64;
        case at::kByte: return kUint8;
        default: return -1;
    }
}

std::string shape_text(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

// The positional arguments of one call; the tensors seen so far share a device.
struct Call {
    const char* op;
    PyObject* const* args;
    int device = -2;

    bool given(int i) const { return args[i] != Py_None; }

    const at::Tensor& tensor(int i, const char* what) {
        if (!THPVariable_Check(args[i])) refuse(std::string(op) + ": " + what + " must be a tensor");
        return THPVariable_Unpack(args[i]);
    }
    // (device checked last, so that a tensor of the wrong form is named first)
    void on_device(const at::Tensor& t) {
        const int d = t.is_cuda() ? t.get_device() : -1;
        if (d < 0 || (device >= 0 && d != device)) refuse(std::string(op) + ": tensors must be on one CUDA device");
        if (t.requires_grad() && c10::GradMode::is_enabled())
            refuse(std::string(op) + ": there is no backward pass, but a tensor asks for a gradient (torch.no_grad())");
        device = d;
    }
    // Outputs that the call has written: autograd refuses what it saved of them before.
    static void wrote(std::initializer_list<const at::Tensor*> outputs) {
        for (const at::Tensor* t : outputs)
            if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
    // Checks rank, type and that the last axis is contiguous.
    const at::Tensor& of(int i, const char* what, size_t rank, int type) {
        const at::Tensor& t = tensor(i, what);
        if (static_cast<size_t>(t.dim()) != rank)
            refuse(std::string(op) + ": " + what + ": expected " + std::to_string(rank) + " axes, got " +
                   shape_text(t.sizes()));
        if (type_of(t) != type) refuse(std::string(op) + ": " + what + ": wrong type");
        if (t.is_neg()) refuse(std::string(op) + ": " + what + ": a lazily negated view (resolve_neg it)");
        if (t.size(rank - 1) > 1 && t.stride(rank - 1) != 1)
            refuse(std::string(op) + ": " + what + ": the last axis must be contiguous");
        return t;
    }
    const at::Tensor& of(int i, const char* what, std::initializer_list<int64_t> shape, int type) {
        const at::Tensor& t = of(i, what, shape.size(), type);
        if (t.sizes() != at::IntArrayRef(shape))
            refuse(std::string(op) + ": " + what + ": expected shape " + shape_text(at::IntArrayRef(shape)) + ", got " +
                   shape_text(t.sizes()));
        return t;
    }
    double number(int i, const char* what) {
        const double v = PyFloat_AsDouble(args[i]);
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse(std::string(op) + ": " + what + " must be a number");
        }
        return v;
    }
    bool truth(int i, const char* what) {
        const int v = PyObject_IsTrue(args[i]);
        if (v < 0) {
            PyErr_Clear();
            refuse(std::string(op) + ": " + what + " must be true or false");
        }
        return v != 0;
    }
    long integer(int i, const char* what) {
        int over = 0;
        const long v = PyLong_AsLongAndOverflow(args[i], &over);
        if (over || (v == -1 && PyErr_Occurred()) || v > INT32_MAX || v < INT32_MIN) {
            PyErr_Clear();
            refuse(std::string(op) + ": " + what + " must be an integer");
        }
        return v;
    }
};

// Runs the call on the tensors' device and on the stream that was asked for:
// None (the device's current one), a handle or an object with cuda_stream.
struct OnDevice {
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = nullptr;
    bool own_stream = false;

    OnDevice(Call& c, PyObject* s) {
        if (c.device < 0) refuse(std::string(c.op) + ": tensors must be on one CUDA device");
        if (c10::cuda::current_device() != c.device) guard.set_index(c.device);
        uintptr_t h = 0;
        if (s == Py_None) {
            h = reinterpret_cast<uintptr_t>(c10::cuda::getCurrentCUDAStream(c.device).stream());
        } else {
            PyObject* held = nullptr;
            if (!PyLong_Check(s)) s = held = PyObject_GetAttrString(s, "cuda_stream");
            const unsigned long long v = s ? PyLong_AsUnsignedLongLong(s) : 0;
            Py_XDECREF(held);
            if (PyErr_Occurred()) {
                PyErr_Clear();
                refuse(std::string(c.op) + ": stream must be a CUDA stream or its handle");
            }
            h = static_cast<uintptr_t>(v);
            own_stream = true;
        }
        stream = reinterpret_cast<void*>(h ? h : 1);  // 1: the legacy default stream by name (NULL means another)
    }
};

int64_t row_stride(const at::Tensor& t, int64_t rows, int64_t width) { return rows > 1 ? t.stride(0) : width; }

void check(int rc) {
    if (rc != VXB_OK) throw Refused{rc, vxb_last_error()};
}

void* ptr(const at::Tensor& t) { return t.data_ptr(); }

// x, weight, y, y_scale, residual, sum_out, eps, stream
void rms_norm(Call& c) {
    const at::Tensor& x = c.tensor(0, "x");
    const int type = type_of(x);
    c.of(0, "x", 2, type);
    const int64_t N = x.size(0), C = x.size(1);
    const at::Tensor& w = c.tensor(1, "weight");
    c.of(1, "weight", {C}, type_of(w));
    const at::Tensor& y = c.tensor(2, "y");
    c.of(2, "y", {N, C}, type_of(y));
    const int64_t kb = (C + 127) / 128;
    const at::Tensor* s = c.given(3) ? &c.of(3, "y_scale", {N, kb}, VXB_TYPE_F32) : nullptr;
    const at::Tensor* r = c.given(4) ? &c.of(4, "residual", {N, C}, type) : nullptr;
    const at::Tensor* h = c.given(5) ? &c.of(5, "sum_out", {N, C}, type) : nullptr;
    for (const at::Tensor* t : {&x, &w, &y, s, r, h})
        if (t) c.on_device(*t);
    if (C > INT32_MAX) refuse("rms_norm: width must be 1..32768");
    const float eps = static_cast<float>(c.number(6, "eps"));
    OnDevice d(c, c.args[7]);
    check(vxb_rms_norm(type, N, static_cast<int>(C), ptr(x), row_stride(x, N, C), r ? ptr(*r) : nullptr,
                       r ? row_stride(*r, N, C) : 0, h ? ptr(*h) : nullptr, h ? row_stride(*h, N, C) : 0, type_of(w),
                       ptr(w), eps, type_of(y), ptr(y), row_stride(y, N, C), s ? static_cast<float*>(ptr(*s)) : nullptr,
                       s ? row_stride(*s, N, kb) : 0, d.stream));
    c.wrote({&y, s, h});
}

// x, x_scale, w, w_scale, y, bias, stream
void fp8_product(Call& c) {
    const at::Tensor& x = c.of(0, "x", 2, VXB_TYPE_E4M3);
    const at::Tensor& w = c.of(2, "w", 2, VXB_TYPE_E4M3);
    const int64_t N = x.size(0), K = x.size(1), M = w.size(0), kb = (K + 127) / 128;
    c.of(2, "w", {M, K}, VXB_TYPE_E4M3);
    const at::Tensor& xs = c.of(1, "x_scale", {N, kb}, VXB_TYPE_F32);
    const at::Tensor& ws = c.of(3, "w_scale", {(M + 127) / 128, kb}, VXB_TYPE_F32);
    const at::Tensor& y = c.tensor(4, "y");
    c.of(4, "y", {N, M}, type_of(y));
    if (!ws.is_contiguous()) refuse("fp8_product: w_scale must be contiguous");
    const at::Tensor* b = c.given(5) ? &c.of(5, "bias", {M}, VXB_TYPE_F32) : nullptr;
    for (const at::Tensor* t : {&x, &xs, &w, &ws, &y, b})
        if (t) c.on_device(*t);
    if (K > INT32_MAX || M > INT32_MAX) refuse("fp8_product: bad extents");
    const int64_t pitch = (K + 15) / 16 * 16;  // of a single row
    OnDevice d(c, c.args[6]);
    check(vxb_fp8_product(N, static_cast<int>(K), static_cast<int>(M), ptr(x), row_stride(x, N, pitch),
                          static_cast<const float*>(ptr(xs)), row_stride(xs, N, kb), ptr(w), row_stride(w, M, pitch),
                          static_cast<const float*>(ptr(ws)), b ? static_cast<const float*>(ptr(*b)) : nullptr,
                          type_of(y), ptr(y), row_stride(y, N, M), d.stream));
    c.wrote({&y});
}

// Strides of [N][heads][D]; an axis of one element has whatever stride fits.
struct Heads {
    void* p = nullptr;
    int64_t token = 0, head = 0;
    Heads() = default;
    explicit Heads(const at::Tensor& t)
        : p(ptr(t)),
          token(t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2)),
          head(t.size(1) > 1 ? t.stride(1) : t.size(2)) {}
};

int checked_int(const char* op, int64_t v) {
    if (v > INT32_MAX) refuse(std::string(op) + ": an extent is too large");
    return static_cast<int>(v);
}

// q, positions, inv_freq, q_out, k, k_out, interleaved, factor, stream
void rotary(Call& c) {
    const at::Tensor& q = c.tensor(0, "q");
    const int type = type_of(q);
    c.of(0, "q", 3, type);
    const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2);
    const at::Tensor& pos = c.of(1, "positions", {N}, kInt64);
    const at::Tensor& f = c.of(2, "inv_freq", 1, VXB_TYPE_F32);
    const at::Tensor& qo = c.of(3, "q_out", {N, Hq, D}, type);
    if (c.given(4) != c.given(5)) refuse("rotary: k and k_out come together");
    const at::Tensor* k = c.given(4) ? &c.of(4, "k", 3, type) : nullptr;
    const int64_t Hk = k ? k->size(1) : 0;
    const at::Tensor* ko = nullptr;
    if (k) {
        c.of(4, "k", {N, Hk, D}, type);
        ko = &c.of(5, "k_out", {N, Hk, D}, type);
    }
    for (const at::Tensor* t : {&q, &pos, &f, &qo, k, ko})
        if (t) c.on_device(*t);
    const int inter = c.truth(6, "interleaved");
    const float factor = static_cast<float>(c.number(7, "factor"));
    const Heads hq(q), hqo(qo), hk = k ? Heads(*k) : Heads(), hko = ko ? Heads(*ko) : Heads();
    OnDevice d(c, c.args[8]);
    check(vxb_rotary(type, N, checked_int(c.op, Hq), checked_int(c.op, Hk), checked_int(c.op, D),
                     checked_int(c.op, 2 * f.size(0)), inter, factor, static_cast<const int64_t*>(ptr(pos)),
                     static_cast<const float*>(ptr(f)), hq.p, hq.token, hq.head, hqo.p, hqo.token, hqo.head, hk.p,
                     hk.token, hk.head, hko.p, hko.token, hko.head, d.stream));
    c.wrote({&qo, ko});
}

// The two caches of one shape and one set of strides.
struct Cache {
    const at::Tensor *k, *v;
    int64_t pages, page, page_stride, slot_stride, head_stride;
    Cache(Call& c, int ik, int iv, int64_t Hk, int64_t D, int type) {
        const at::Tensor& kc = c.of(ik, "k_cache", 4, type);
        if (kc.size(2) != Hk || kc.size(3) != D)
            refuse(std::string(c.op) + ": k_cache: expected [.., .., " + std::to_string(Hk) + ", " + std::to_string(D) +
                   "], got " + shape_text(kc.sizes()));
        const at::Tensor& vc = c.of(iv, "v_cache", 4, type);
        if (vc.sizes() != kc.sizes()) refuse(std::string(c.op) + ": k_cache and v_cache must have one shape");
        for (int i = 0; i < 3; ++i)
            if (kc.size(i) > 1 && kc.stride(i) != vc.stride(i))
                refuse(std::string(c.op) + ": k_cache and v_cache must have one set of strides");
        k = &kc, v = &vc;
        pages = kc.size(0), page = kc.size(1);
        head_stride = Hk > 1 ? kc.stride(2) : D;
        slot_stride = page > 1 ? kc.stride(1) : Hk * D;
        page_stride = pages > 1 ? kc.stride(0) : page * Hk * D;
    }
};

// q, k, v, positions, slots, inv_freq, q_out, k_cache, v_cache, interleaved, factor, stream
void rotary_append(Call& c) {
    const at::Tensor& q = c.tensor(0, "q");
    const int type = type_of(q);
    c.of(0, "q", 3, type);
    const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2);
    const int64_t Hk = c.of(1, "k", 3, type).size(1);
    const at::Tensor& k = c.of(1, "k", {N, Hk, D}, type);
    const at::Tensor& v = c.of(2, "v", {N, Hk, D}, type);
    const at::Tensor& pos = c.of(3, "positions", {N}, kInt64);
    const at::Tensor& slots = c.of(4, "slots", {N}, kInt64);
    const at::Tensor& f = c.of(5, "inv_freq", 1, VXB_TYPE_F32);
    const at::Tensor& qo = c.of(6, "q_out", {N, Hq, D}, type);
    const Cache m(c, 7, 8, Hk, D, type);
    for (const at::Tensor* t : {&q, &k, &v, &pos, &slots, &f, &qo, m.k, m.v}) c.on_device(*t);
    const int inter = c.truth(9, "interleaved");
    const float factor = static_cast<float>(c.number(10, "factor"));
    const Heads hq(q), hqo(qo), hk(k), hv(v);
    OnDevice d(c, c.args[11]);
    check(vxb_rotary_append(type, N, checked_int(c.op, Hq), checked_int(c.op, Hk), checked_int(c.op, D),
                            checked_int(c.op, 2 * f.size(0)), inter, factor, static_cast<const int64_t*>(ptr(pos)),
                            static_cast<const int64_t*>(ptr(slots)), static_cast<const float*>(ptr(f)), hq.p, hq.token,
                            hq.head, hqo.p, hqo.token, hqo.head, hk.p, hk.token, hk.head, hv.p, hv.token, hv.head,
                            ptr(*m.k), ptr(*m.v), m.pages, checked_int(c.op, m.page), m.page_stride, m.slot_stride,
                            m.head_stride, d.stream));
    c.wrote({&qo, m.k, m.v});
}

// q, k_cache, v_cache, block_table, cu_q, kv_len, out, scale, window, workspace, stream
void paged_attention(Call& c) {
    const at::Tensor& q = c.tensor(0, "q");
    const int type = type_of(q);
    c.of(0, "q", 3, type);
    const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2);
    const int64_t Hk = c.of(1, "k_cache", 4, type).size(2);
    const Cache m(c, 1, 2, Hk, D, type);
    const at::Tensor& table = c.of(3, "block_table", 2, kInt32);
    const int64_t B = table.size(0), max_pages = table.size(1);
    const at::Tensor& cu = c.of(4, "cu_q", {B + 1}, kInt32);
    const at::Tensor& kv = c.of(5, "kv_len", {B}, kInt32);
    const at::Tensor& out = c.of(6, "out", {N, Hq, D}, type);
    const at::Tensor* ws = c.given(9) ? &c.of(9, "workspace", 1, kUint8) : nullptr;
    for (const at::Tensor* t : {&q, m.k, m.v, &table, &cu, &kv, &out, ws})
        if (t) c.on_device(*t);
    const double scale = c.given(7) ? c.number(7, "scale") : 1.0 / std::sqrt(static_cast<double>(D));
    const int window = static_cast<int>(c.integer(8, "window"));
    const int b = checked_int(c.op, B), hq = checked_int(c.op, Hq), hk = checked_int(c.op, Hk),
              dd = checked_int(c.op, D), mp = checked_int(c.op, max_pages), pg = checked_int(c.op, m.page);
    OnDevice d(c, c.args[10]);
    at::Tensor mine;
    if (!ws) {
        const int64_t need = vxb_paged_attention_workspace(N, b, hq, hk, dd, mp, pg);
        if (need < 0) refuse(vxb_last_error());
        if (need > 0) {  // memory of the stream that uses it
            c10::cuda::OptionalCUDAStreamGuard on;
            if (d.own_stream)
                on.reset_stream(d.stream == reinterpret_cast<void*>(1)
                                    ? c10::cuda::getDefaultCUDAStream(c.device)
                                    : c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(d.stream), c.device));
            mine = at::empty({need}, q.options().dtype(at::kByte));
            ws = &mine;
        }
    }
    const Heads h(q), ho(out);
    check(vxb_paged_attention(type, N, b, hq, hk, dd, h.p, h.token, h.head, ptr(*m.k), ptr(*m.v), m.pages, pg,
                              m.page_stride, m.slot_stride, m.head_stride, static_cast<const int32_t*>(ptr(table)),
                              B > 1 ? table.stride(0) : max_pages, mp, static_cast<const int32_t*>(ptr(cu)),
                              static_cast<const int32_t*>(ptr(kv)), static_cast<float>(scale), window, ho.p, ho.token,
                              ho.head, ws ? ptr(*ws) : nullptr, ws ? ws->numel() : 0, d.stream));
    c.wrote({&out, mine.defined() ? nullptr : ws});
}

template <void (*F)(Call&), int kArgs>
PyObject* entry(const char* op, PyObject* const* args, Py_ssize_t n) {
    if (n != kArgs) {
        PyErr_Format(PyExc_TypeError, "%s takes %d arguments", op, kArgs);
        return nullptr;
    }
    int code = VXB_ERR_BACKEND;
    std::string what;
    try {
        Call c{op, args};
        F(c);
        Py_RETURN_NONE;
    } catch (const Refused& r) {
        code = r.code;
        what = r.what;
    } catch (const std::exception& e) {
        what = e.what();
    } catch (...) {
        what = "unknown error";
    }
    PyObject* err = g_error ? PyObject_CallFunction(g_error, "is", code, what.c_str()) : nullptr;
    if (err) {
        PyErr_SetObject(g_error, err);
        Py_DECREF(err);
    } else if (!PyErr_Occurred()) {
        PyErr_SetString(PyExc_RuntimeError, what.c_str());
    }
    return nullptr;
}

#define VXB_ENTRY(name, n)                                                              \
    PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t count) {           \
        return entry<name, n>(#name, args, count);                                      \
    }
VXB_ENTRY(rms_norm, 8)
VXB_ENTRY(fp8_product, 7)
VXB_ENTRY(rotary, 9)
VXB_ENTRY(rotary_append, 12)
VXB_ENTRY(paged_attention, 11)

PyObject* py_set_error(PyObject*, PyObject* cls) {
    Py_XINCREF(cls);
    Py_XSETREF(g_error, cls);
    Py_RETURN_NONE;
}

#define VXB_METHOD(name) \
    {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {VXB_METHOD(rms_norm), VXB_METHOD(fp8_product), VXB_METHOD(rotary), VXB_METHOD(rotary_append),
                          VXB_METHOD(paged_attention), {"set_error", py_set_error, METH_O, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_vxb_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__vxb_native() { return PyModule_Create(&kModule); }
