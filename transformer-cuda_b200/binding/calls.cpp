// Python entry of the calls that a program makes once per layer and token, where the arithmetic is over in some ten
// microseconds: checks the tensors, allocates outputs and scratch from torch's allocator and makes the C call
// (include/b200attn.h, include/b200loss.h), in a few microseconds instead of the thirty that the same steps take in Python
// (a packed training pass over three short sequences: 50 us of host time for 20 us of GPU time). ops.py and loss_ops.py
// hold the documented functions; every check of an argument that concerns a tensor is here, every check of sizes behind
// the C entry.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cstdarg>
#include <cstdio>
#include <string>

#include "b200attn.h"
#include "b200loss.h"

namespace {

PyObject *g_attn_error = nullptr, *g_loss_error = nullptr;  // classes taking (code, message)

// Thrown once the Python error is set.
struct PyFailed {};

[[noreturn]] void raise_code(PyObject* cls, int code, const char* text) {
    PyObject* e = PyObject_CallFunction(cls, "is", code, text);
    if (e) {
        PyErr_SetObject(cls, e);
        Py_DECREF(e);
    }
    throw PyFailed{};
}
// Refusals of the attention calls carry the library's error class, those of the loss calls are ValueErrors.
enum class Kind { kAttn, kLoss };
[[noreturn]] void refuse(Kind kind, const char* fmt, ...) {
    char text[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    if (kind == Kind::kAttn) raise_code(g_attn_error, B200ATTN_ERR_INVALID_ARGUMENT, text);
    PyErr_SetString(PyExc_ValueError, text);
    throw PyFailed{};
}
void check_attn(int rc) {
    if (rc != 0) raise_code(g_attn_error, rc, b200attn_last_error());
}
void check_loss(int rc) {
    if (rc != 0) raise_code(g_loss_error, rc, b200loss_last_error());
}

std::string shape_text(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

const at::Tensor& tensor(PyObject* o, Kind kind, const char* name) {
    if (!THPVariable_Check(o)) refuse(kind, "%s: expected a CUDA tensor", name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse(kind, "%s: expected a CUDA tensor", name);
    return t;
}
const at::Tensor& on_device(PyObject* o, Kind kind, const char* name, at::Device device) {
    const at::Tensor& t = tensor(o, kind, name);
    if (t.device() != device) refuse(kind, "%s: is on %s, expected %s", name, t.device().str().c_str(), device.str().c_str());
    return t;
}
// A contiguous tensor of `numel` elements.
void* vector(PyObject* o, Kind kind, const char* name, at::ScalarType type, int64_t numel, at::Device device) {
    const at::Tensor& t = on_device(o, kind, name, device);
    if (t.scalar_type() != type || t.numel() != numel || !t.is_contiguous())
        refuse(kind, "%s: expected a contiguous %s tensor of %lld elements, got %s %s", name, c10::toString(type), (long long)numel,
               c10::toString(t.scalar_type()), shape_text(t).c_str());
    return t.data_ptr();
}
// Row stride of a BF16 tensor (rows, heads, d) whose heads are contiguous; rows may be any distance apart.
int64_t head_rows(const at::Tensor& t, const char* name) {
    if (t.scalar_type() != at::kBFloat16 || t.dim() != 3)
        refuse(Kind::kAttn, "%s: expected a BF16 tensor (rows, heads, d), got %s %s", name, c10::toString(t.scalar_type()), shape_text(t).c_str());
    const int64_t rows = t.size(0), heads = t.size(1), d = t.size(2);
    if (rows && heads && ((d > 1 && t.stride(2) != 1) || (heads > 1 && t.stride(1) != d)))
        refuse(Kind::kAttn, "%s: heads must be contiguous (strides %lld, %lld, %lld)", name, (long long)t.stride(0), (long long)t.stride(1), (long long)t.stride(2));
    return rows > 1 ? t.stride(0) : heads * d;
}
int64_t head_rows_like(PyObject* o, const char* name, const at::Tensor& like, void** ptr) {
    const at::Tensor& t = on_device(o, Kind::kAttn, name, like.device());
    const int64_t stride = head_rows(t, name);
    if (t.sizes() != like.sizes()) refuse(Kind::kAttn, "%s: has shape %s, expected %s", name, shape_text(t).c_str(), shape_text(like).c_str());
    *ptr = t.data_ptr();
    return stride;
}
int to_int(int64_t x, Kind kind, const char* name) {
    if (x > 0x7fffffff) refuse(kind, "%s: %lld is too large", name, (long long)x);
    return int(x);
}
float to_float(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw PyFailed{};
    return float(x);
}
void need_args(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
        throw PyFailed{};
    }
}
at::Tensor empty(c10::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));  // torch.empty without its dispatch
}
at::Tensor zeros(c10::IntArrayRef sizes, at::ScalarType type, at::Device device) { return at::zeros(sizes, at::TensorOptions(type).device(device)); }
// Scratch of one call from torch's allocator: ordered with the stream, its own in every captured graph.
at::Tensor scratch(int64_t bytes, at::Device device) { return empty({bytes > 16 ? bytes : 16}, at::kByte, device); }

// A new reference to `o`, and to a Python tensor around `t`.
THPObjectPtr own(PyObject* o) {
    Py_INCREF(o);
    return THPObjectPtr(o);
}
THPObjectPtr wrap(at::Tensor t) {
    THPObjectPtr o(THPVariable_Wrap(std::move(t)));
    if (!o) throw PyFailed{};
    return o;
}
template <typename... P>
PyObject* tuple_of(P&&... items) {
    THPObjectPtr t(PyTuple_New(sizeof...(items)));
    if (!t) throw PyFailed{};
    Py_ssize_t i = 0;
    (PyTuple_SET_ITEM(t.get(), i++, items.release()), ...);
    return t.release();
}
// The tuple of what `make` returns, or the Python error.
template <typename F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const PyFailed&) {
        return nullptr;
    } catch (...) {  // torch's own errors (out of memory among them) in its own classes
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

// ---------------------------------------------------------------- packed attention
struct Ragged {
    const at::Tensor *q, *k, *v;
    void* offsets;
    int total, n, H, Hkv, d;
    int64_t sq, skv;
};
Ragged ragged_args(PyObject* q_, PyObject* k_, PyObject* v_, PyObject* offsets_) {
    Ragged a;
    a.q = &tensor(q_, Kind::kAttn, "q");
    const at::Device device = a.q->device();
    a.sq = head_rows(*a.q, "q");
    a.k = &on_device(k_, Kind::kAttn, "k", device);
    a.skv = head_rows(*a.k, "k");
    a.total = to_int(a.q->size(0), Kind::kAttn, "rows of q"), a.H = to_int(a.q->size(1), Kind::kAttn, "heads of q"), a.d = to_int(a.q->size(2), Kind::kAttn, "d");
    a.Hkv = to_int(a.k->size(1), Kind::kAttn, "heads of k");
    if (a.k->size(0) != a.total || a.k->size(2) != a.d || a.Hkv == 0 || a.H % a.Hkv != 0)
        refuse(Kind::kAttn, "k: expected (%d, a divisor of %d, %d), got %s", a.total, a.H, a.d, shape_text(*a.k).c_str());
    void* unused;
    if (head_rows_like(v_, "v", *a.k, &unused) != a.skv) refuse(Kind::kAttn, "k and v must have the same row stride");
    a.v = &THPVariable_Unpack(v_);
    const at::Tensor& o = on_device(offsets_, Kind::kAttn, "offsets", device);
    if (o.dim() != 1 || o.numel() < 1) refuse(Kind::kAttn, "offsets: expected n + 1 row numbers");
    a.n = to_int(o.numel() - 1, Kind::kAttn, "sequences");
    a.offsets = vector(offsets_, Kind::kAttn, "offsets", at::kInt, o.numel(), device);
    return a;
}

// q, k, v, offsets, scale, out or None, lse or None -> (out, lse)
PyObject* ragged_forward(PyObject*, PyObject* const* p, Py_ssize_t np) {
    return guarded([&]() -> PyObject* {
        need_args(np, 7);
        const Ragged a = ragged_args(p[0], p[1], p[2], p[3]);
        const float scale = to_float(p[4]);
        const at::Device device = a.q->device();
        const c10::cuda::CUDAGuard guard(device);
        THPObjectPtr out = p[5] == Py_None ? wrap(zeros(a.q->sizes(), at::kBFloat16, device)) : own(p[5]);
        THPObjectPtr lse = p[6] == Py_None ? wrap(zeros({a.H, a.total}, at::kFloat, device)) : own(p[6]);
        void* out_ptr;
        const int64_t so = head_rows_like(out, "out", *a.q, &out_ptr);
        float* lse_ptr = static_cast<float*>(vector(lse, Kind::kAttn, "lse", at::kFloat, (int64_t)a.H * a.total, device));
        const long long bytes = b200attn_ragged_workspace_bytes(a.total, a.n, a.H, a.Hkv, a.d, 0);
        const at::Tensor ws = scratch(bytes, device);
        check_attn(b200attn_fwd_bf16_ragged(a.q->data_ptr(), a.k->data_ptr(), a.v->data_ptr(), static_cast<int*>(a.offsets), out_ptr, lse_ptr,
                                            ws.data_ptr(), bytes, a.total, a.n, a.H, a.Hkv, a.d, a.sq, a.skv, so, scale,
                                            c10::cuda::getCurrentCUDAStream(device.index()).stream()));
        return tuple_of(out, lse);
    });
}

// q, k, v, out, dout, lse, offsets, scale, dq or None, dk or None, dv or None -> (dq, dk, dv)
PyObject* ragged_backward(PyObject*, PyObject* const* p, Py_ssize_t np) {
    return guarded([&]() -> PyObject* {
        need_args(np, 11);
        const Ragged a = ragged_args(p[0], p[1], p[2], p[6]);
        const float scale = to_float(p[7]);
        const at::Device device = a.q->device();
        const c10::cuda::CUDAGuard guard(device);
        void *out_ptr, *dout_ptr, *dq_ptr, *dk_ptr, *dv_ptr;
        const int64_t so = head_rows_like(p[3], "out", *a.q, &out_ptr), sdo = head_rows_like(p[4], "dout", *a.q, &dout_ptr);
        float* lse_ptr = static_cast<float*>(vector(p[5], Kind::kAttn, "lse", at::kFloat, (int64_t)a.H * a.total, device));
        THPObjectPtr dq = p[8] == Py_None ? wrap(zeros(a.q->sizes(), at::kBFloat16, device)) : own(p[8]);
        THPObjectPtr dk = p[9] == Py_None ? wrap(zeros(a.k->sizes(), at::kBFloat16, device)) : own(p[9]);
        THPObjectPtr dv = p[10] == Py_None ? wrap(zeros(a.k->sizes(), at::kBFloat16, device)) : own(p[10]);
        const int64_t sdq = head_rows_like(dq, "dq", *a.q, &dq_ptr), sdk = head_rows_like(dk, "dk", *a.k, &dk_ptr);
        if (head_rows_like(dv, "dv", *a.k, &dv_ptr) != sdk) refuse(Kind::kAttn, "dk and dv must have the same row stride");
        const long long bytes = b200attn_ragged_workspace_bytes(a.total, a.n, a.H, a.Hkv, a.d, 1);
        const at::Tensor ws = scratch(bytes, device);
        check_attn(b200attn_bwd_bf16_ragged(a.q->data_ptr(), a.k->data_ptr(), a.v->data_ptr(), out_ptr, dout_ptr, lse_ptr,
                                            static_cast<int*>(a.offsets), dq_ptr, dk_ptr, dv_ptr, ws.data_ptr(), bytes, a.total, a.n, a.H,
                                            a.Hkv, a.d, a.sq, a.skv, so, sdo, sdq, sdk, scale,
                                            c10::cuda::getCurrentCUDAStream(device.index()).stream()));
        return tuple_of(dq, dk, dv);
    });
}

// ---------------------------------------------------------------- one token per sequence
// q, k_cache, v_cache, lengths, scale, out or None, lse or None -> (out, lse)
PyObject* decode(PyObject*, PyObject* const* p, Py_ssize_t np) {
    return guarded([&]() -> PyObject* {
        need_args(np, 7);
        const at::Tensor& q = tensor(p[0], Kind::kAttn, "q");
        const at::Device device = q.device();
        const int64_t sq = head_rows(q, "q");
        const int B = to_int(q.size(0), Kind::kAttn, "sequences"), H = to_int(q.size(1), Kind::kAttn, "heads"), d = to_int(q.size(2), Kind::kAttn, "d");
        const at::Tensor* cache[2];
        int64_t strides[2][3];
        for (int i = 0; i < 2; ++i) {
            const char* name = i ? "v_cache" : "k_cache";
            const at::Tensor& t = on_device(p[1 + i], Kind::kAttn, name, device);
            cache[i] = &t;
            if (t.scalar_type() != at::kBFloat16 || t.dim() != 4)
                refuse(Kind::kAttn, "%s: expected a BF16 tensor (B, T, Hkv, d), got %s %s", name, c10::toString(t.scalar_type()), shape_text(t).c_str());
            if (t.size(0) != B || t.size(3) != d || t.size(2) == 0 || H % t.size(2) != 0 || t.sizes() != cache[0]->sizes())
                refuse(Kind::kAttn, "%s: expected (%d, T, a divisor of %d, %d), the same for both, got %s", name, B, H, d, shape_text(t).c_str());
            if (t.numel() && t.stride(3) != 1) refuse(Kind::kAttn, "%s: the last dimension must be contiguous", name);
            for (int x = 0; x < 3; ++x) strides[i][x] = t.size(x) > 1 ? t.stride(x) : 0;  // one element: no stride to keep
        }
        const int T = to_int(cache[0]->size(1), Kind::kAttn, "T"), Hkv = int(cache[0]->size(2));
        const float scale = to_float(p[4]);
        int* lengths = static_cast<int*>(vector(p[3], Kind::kAttn, "lengths", at::kInt, B, device));
        const c10::cuda::CUDAGuard guard(device);
        THPObjectPtr out = p[5] == Py_None ? wrap(empty({B, H, d}, at::kBFloat16, device)) : own(p[5]);
        THPObjectPtr lse = p[6] == Py_None ? wrap(empty({B, H}, at::kFloat, device)) : own(p[6]);
        void* out_ptr = vector(out, Kind::kAttn, "out", at::kBFloat16, (int64_t)B * H * d, device);
        float* lse_ptr = static_cast<float*>(vector(lse, Kind::kAttn, "lse", at::kFloat, (int64_t)B * H, device));
        const long long bytes = b200attn_decode_workspace_bytes(B, T, H, Hkv, d);
        at::Tensor ws;
        if (bytes) ws = scratch(bytes, device);
        check_attn(b200attn_decode_bf16(q.data_ptr(), cache[0]->data_ptr(), cache[1]->data_ptr(), lengths, out_ptr, lse_ptr,
                                        bytes ? ws.data_ptr() : nullptr, bytes, B, T, H, Hkv, d, sq, strides[0][0], strides[0][1], strides[0][2],
                                        strides[1][0], strides[1][1], strides[1][2], scale,
                                        c10::cuda::getCurrentCUDAStream(device.index()).stream()));
        return tuple_of(out, lse);
    });
}

// ---------------------------------------------------------------- token log-probabilities
struct Rows {
    int rows, V, dtype;
    int64_t stride;
};
// FP32 or BF16 rows (..., V): contiguous elements, one stride from row to row.
Rows rows_of(const at::Tensor& t, const char* name) {
    const bool f32 = t.scalar_type() == at::kFloat;
    if ((!f32 && t.scalar_type() != at::kBFloat16) || t.dim() < 1 || t.size(-1) < 1)
        refuse(Kind::kLoss, "%s must be a CUDA float32 or bfloat16 tensor of shape (..., V), is %s %s", name, c10::toString(t.scalar_type()), shape_text(t).c_str());
    const int64_t V = t.size(-1);
    int64_t rows = 1, stride = -1, next = -1;  // next: the stride that the dimension in front has to have
    bool regular = t.stride(-1) == 1 || V == 1;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
        rows *= t.size(i);
        if (t.size(i) == 1) continue;
        if (stride < 0) stride = t.stride(i);
        else regular = regular && t.stride(i) == next;
        next = t.stride(i) * t.size(i);
    }
    if (stride < 0) stride = V;
    if (rows && (!regular || stride < V)) refuse(Kind::kLoss, "%s must consist of contiguous rows at one row stride", name);
    return Rows{to_int(rows, Kind::kLoss, "rows"), to_int(V, Kind::kLoss, "V"), f32 ? B200LOSS_F32 : B200LOSS_BF16, rows ? stride : V};
}

// logits, targets, temperature, top -> (logprobs, entropy, stats, top_logprobs or None, top_tokens or None)
PyObject* token_logprobs(PyObject*, PyObject* const* p, Py_ssize_t np) {
    return guarded([&]() -> PyObject* {
        need_args(np, 4);
        const at::Tensor& x = tensor(p[0], Kind::kLoss, "logits");
        const Rows r = rows_of(x, "logits");
        const at::Device device = x.device();
        int* targets = static_cast<int*>(vector(p[1], Kind::kLoss, "targets", at::kInt, r.rows, device));
        const float temperature = to_float(p[2]);
        const long top = PyLong_AsLong(p[3]);
        if (top == -1 && PyErr_Occurred()) throw PyFailed{};
        if (top < 0 || top > 32 || top > r.V) refuse(Kind::kLoss, "top must be between 0 and min(32, V), got %ld", top);
        const c10::cuda::CUDAGuard guard(device);
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end() - 1);
        at::Tensor logprobs = empty(shape, at::kFloat, device), entropy = empty(shape, at::kFloat, device), top_logprobs, top_tokens;
        shape.push_back(2);
        at::Tensor stats = empty(shape, at::kFloat, device);
        if (top) {
            shape.back() = top;
            top_logprobs = empty(shape, at::kFloat, device), top_tokens = empty(shape, at::kInt, device);
        }
        check_loss(b200loss_token_logprobs(x.data_ptr(), r.dtype, r.stride, targets, r.rows, r.V, temperature, static_cast<float*>(logprobs.data_ptr()),
                                           static_cast<float*>(entropy.data_ptr()), static_cast<float*>(stats.data_ptr()), int(top),
                                           top ? static_cast<float*>(top_logprobs.data_ptr()) : nullptr, top ? static_cast<int*>(top_tokens.data_ptr()) : nullptr,
                                           c10::cuda::getCurrentCUDAStream(device.index()).stream()));
        return tuple_of(wrap(std::move(logprobs)), wrap(std::move(entropy)), wrap(std::move(stats)),
                        top ? wrap(std::move(top_logprobs)) : own(Py_None), top ? wrap(std::move(top_tokens)) : own(Py_None));
    });
}

// logits, targets, entropy, stats, grad_logprobs, grad_entropy or None, temperature, dlogits or None -> dlogits
PyObject* token_logprobs_backward(PyObject*, PyObject* const* p, Py_ssize_t np) {
    return guarded([&]() -> PyObject* {
        need_args(np, 8);
        const at::Tensor& x = tensor(p[0], Kind::kLoss, "logits");
        const Rows r = rows_of(x, "logits");
        const at::Device device = x.device();
        int* targets = static_cast<int*>(vector(p[1], Kind::kLoss, "targets", at::kInt, r.rows, device));
        const float* entropy = static_cast<float*>(vector(p[2], Kind::kLoss, "result.entropy", at::kFloat, r.rows, device));
        const float* stats = static_cast<float*>(vector(p[3], Kind::kLoss, "result.stats", at::kFloat, 2ll * r.rows, device));
        const float* g = static_cast<float*>(vector(p[4], Kind::kLoss, "grad_logprobs", at::kFloat, r.rows, device));
        const float* ge = p[5] == Py_None ? nullptr : static_cast<float*>(vector(p[5], Kind::kLoss, "grad_entropy", at::kFloat, r.rows, device));
        const float temperature = to_float(p[6]);
        const c10::cuda::CUDAGuard guard(device);
        THPObjectPtr result;
        int64_t d_stride = r.V;
        if (p[7] == Py_None) {
            result = wrap(empty(x.sizes(), x.scalar_type(), device));
        } else {
            const at::Tensor& d = on_device(p[7], Kind::kLoss, "dlogits", device);
            if (d.scalar_type() != x.scalar_type() || d.sizes() != x.sizes()) refuse(Kind::kLoss, "dlogits must have the logits' shape and type");
            d_stride = rows_of(d, "dlogits").stride;
            if (d.data_ptr() == x.data_ptr() && d_stride != r.stride) refuse(Kind::kLoss, "dlogits in the logits' place must have the logits' row stride");
            result = own(p[7]);
        }
        check_loss(b200loss_token_logprobs_backward(x.data_ptr(), r.dtype, r.stride, targets, entropy, stats, g, ge, r.rows, r.V, temperature,
                                                    THPVariable_Unpack(result.get()).data_ptr(), d_stride,
                                                    c10::cuda::getCurrentCUDAStream(device.index()).stream()));
        return result.release();
    });
}

// The error classes: B200AttnError, B200LossError.
PyObject* set_errors(PyObject*, PyObject* const* p, Py_ssize_t np) {
    return guarded([&]() -> PyObject* {
        need_args(np, 2);
        for (int i = 0; i < 2; ++i) {
            PyObject*& slot = i ? g_loss_error : g_attn_error;
            Py_XDECREF(slot);
            slot = own(p[i]).release();
        }
        return own(Py_None).release();
    });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(set_errors), METHOD(ragged_forward), METHOD(ragged_backward), METHOD(decode), METHOD(token_logprobs),
                         METHOD(token_logprobs_backward), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b200calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__b200calls(void) { return PyModule_Create(&module); }
