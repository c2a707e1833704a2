// g4q_torch.cpp -- the Python side of the attention calls (helios_b200/attention.py) as a CPython module.
//
// A decoded token's attention calls take 2 to 9 us on the GPU, less than the interpreter needs to check the tensors,
// describe them with ctypes structures and make the outputs (11 to 13 us a call; 5 to 7 with this module). It checks
// dtype, device, shape, strides and overlap of torch tensors, allocates outputs and calls the C ABI of libg4q
// (include/g4q.h) through the entry points that the ctypes binding loaded, so there is one library and one set of
// checks behind both. Errors of the C ABI are raised by the binding's own function.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>
#include <string>

#include "g4q.h"

namespace {

decltype(&g4q_qk_norm_rope) fn_qk_norm_rope = nullptr;
decltype(&g4q_kv_append) fn_kv_append = nullptr;
decltype(&g4q_paged_attention) fn_paged_attention = nullptr;
PyObject* raise_status = nullptr;    // (status, entry point): raises

struct Refused {
    std::string message;
};

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused{std::string(name) + " must be a torch tensor"};
    return THPVariable_Unpack(o);
}

// The C view of a [tokens, heads, head_dim] tensor (any strides that keep 16-byte chunks whole).
G4qHeadRows head_rows(const at::Tensor& t, int64_t head_dim, int64_t device, const char* name, bool output = false) {
    if (t.scalar_type() != at::kBFloat16 || !t.is_cuda() || t.get_device() != device)
        throw Refused{std::string(name) + " must be a bfloat16 CUDA tensor on cuda:" + std::to_string(device)};
    if (t.dim() != 3 || t.size(2) != head_dim)
        throw Refused{std::string(name) + " must be [tokens, heads, " + std::to_string(head_dim) + "] (got " + shape_of(t) + ")"};
    const int64_t st = t.stride(0), sd = t.stride(2);
    int64_t sh = t.stride(1);
    void* data = t.data_ptr();
    if (sd != 1 || ((st | sh) & 7) != 0 || (reinterpret_cast<uintptr_t>(data) & 15u) != 0)
        throw Refused{std::string(name) + ": the last dimension must be contiguous, strides multiples of 8 and data 16-byte aligned"};
    if (t.size(1) == 1) sh = std::max(sh, head_dim);
    if (output && (sh < head_dim || (t.size(0) > 1 && st < head_dim))) throw Refused{std::string(name) + ": its rows overlap"};
    if (t.size(1) > 65536) throw Refused{std::string(name) + ": too many heads"};
    return {static_cast<uint16_t*>(data), st, sh, (int32_t)t.size(1)};
}

// The output for t's shape: the caller's, or a new contiguous tensor.
at::Tensor output(const at::Tensor& t, PyObject* out, int64_t head_dim, int64_t device, const char* name, G4qHeadRows& rows) {
    at::Tensor o;
    if (out == Py_None) {
        o = at::empty(t.sizes(), t.options());
    } else {
        o = tensor(out, name);
        if (o.sizes() != t.sizes()) throw Refused{std::string(name) + " must be shaped " + shape_of(t)};
    }
    rows = head_rows(o, head_dim, device, name, true);
    return o;
}

const uint16_t* norm_weight(PyObject* o, int64_t head_dim, int64_t device, const char* name) {
    if (o == Py_None) return nullptr;
    const at::Tensor& w = tensor(o, name);
    if (w.scalar_type() != at::kBFloat16 || !w.is_cuda() || w.get_device() != device || w.dim() != 1 || w.size(0) != head_dim ||
        !w.is_contiguous())
        throw Refused{std::string(name) + " must be a contiguous bf16 tensor of shape (" + std::to_string(head_dim) + ",) on cuda:" +
                      std::to_string(device)};
    return static_cast<const uint16_t*>(w.data_ptr());
}

// Numbers of the calling convention; a Python error stays set for the caller to see.
struct Args {
    PyObject* const* a;
    long long integer(int i) const { return PyLong_AsLongLong(a[i]); }
    void* pointer(int i) const { return PyLong_AsVoidPtr(a[i]); }
    double real(int i) const { return PyFloat_AsDouble(a[i]); }
};

template <typename F>
PyObject* guarded(const char* name, Py_ssize_t got, Py_ssize_t want, F&& body) {
    HANDLE_TH_ERRORS
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (got %zd)", name, want, got);
        return nullptr;
    }
    if (raise_status == nullptr) {
        PyErr_SetString(PyExc_RuntimeError, "the library's entry points are not bound");
        return nullptr;
    }
    try {
        return body();
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.message.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// Runs a C ABI call without the interpreter lock; true when it succeeded, else an exception is set.
template <typename F>
bool call(const char* name, F&& f) {
    G4qStatus s;
    Py_BEGIN_ALLOW_THREADS
    s = f();
    Py_END_ALLOW_THREADS
    if (s == G4Q_OK) return true;
    PyObject* r = PyObject_CallFunction(raise_status, "is", (int)s, name);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, name);
    return false;
}

// (handle, head_dim, device, stream, q, k, positions, q_weight, k_weight, eps, q_out, k_out) -> (q_out, k_out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded("qk_norm_rope", n, 12, [&]() -> PyObject* {
        const Args a{args};
        auto* rope = static_cast<G4qRope*>(a.pointer(0));
        const int64_t d = a.integer(1), dev = a.integer(2);
        void* stream = a.pointer(3);
        const double eps = a.real(9);
        if (PyErr_Occurred()) return nullptr;
        const at::Tensor &q = tensor(args[4], "q"), &k = tensor(args[5], "k"), &pos = tensor(args[6], "positions");
        const G4qHeadRows cq = head_rows(q, d, dev, "q"), ck = head_rows(k, d, dev, "k");
        const int64_t m = q.size(0);
        if (k.size(0) != m) throw Refused{"q and k must have the same number of tokens"};
        if (pos.scalar_type() != at::kInt || !pos.is_cuda() || pos.get_device() != dev || pos.dim() != 1 || pos.size(0) != m ||
            (m > 1 && pos.stride(0) != 1))
            throw Refused{"positions must be a contiguous int32 tensor on cuda:" + std::to_string(dev) + " with one entry per token"};
        const uint16_t *wq = norm_weight(args[7], d, dev, "q_weight"), *wk = norm_weight(args[8], d, dev, "k_weight");
        G4qHeadRows coq, cok;
        const at::Tensor oq = output(q, args[10], d, dev, "q_out", coq), ok = output(k, args[11], d, dev, "k_out", cok);
        const auto* p = static_cast<const int32_t*>(pos.data_ptr());
        if (!call("g4q_qk_norm_rope", [&] { return fn_qk_norm_rope(rope, &cq, &ck, m, p, wq, wk, (float)eps, &coq, &cok, stream); }))
            return nullptr;
        PyObject* r = PyTuple_New(2);
        if (r == nullptr) return nullptr;
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(oq));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(ok));
        return r;
    });
}

// (handle, head_dim, device, stream, q or None, k, v, cache, batch, q_weight, k_weight, eps, flags, q_out) -> q_out or None
PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded("kv_append", n, 14, [&]() -> PyObject* {
        const Args a{args};
        auto* rope = static_cast<G4qRope*>(a.pointer(0));
        const int64_t d = a.integer(1), dev = a.integer(2);
        void* stream = a.pointer(3);
        const auto* cache = static_cast<const G4qPagedCache*>(a.pointer(7));
        const auto* batch = static_cast<const G4qPagedBatch*>(a.pointer(8));
        const double eps = a.real(11);
        const auto flags = (uint32_t)a.integer(12);
        if (PyErr_Occurred()) return nullptr;
        const at::Tensor &k = tensor(args[5], "k"), &v = tensor(args[6], "v");
        const G4qHeadRows ck = head_rows(k, d, dev, "k"), cv = head_rows(v, d, dev, "v");
        const int64_t m = k.size(0);
        const bool has_q = args[4] != Py_None;
        if (v.size(0) != m || (has_q && tensor(args[4], "q").dim() == 3 && tensor(args[4], "q").size(0) != m))
            throw Refused{"q, k and v must have the same number of tokens"};
        G4qHeadRows cq, co;
        at::Tensor o;
        if (has_q) {
            const at::Tensor& q = tensor(args[4], "q");
            cq = head_rows(q, d, dev, "q");
            o = output(q, args[13], d, dev, "q_out", co);
        } else if (args[13] != Py_None) {
            throw Refused{"q_out without q"};
        }
        const uint16_t *wq = norm_weight(args[9], d, dev, "q_weight"), *wk = norm_weight(args[10], d, dev, "k_weight");
        if (!call("g4q_kv_append", [&] {
                return fn_kv_append(rope, has_q ? &cq : nullptr, &ck, &cv, m, wq, wk, (float)eps, flags, has_q ? &co : nullptr, cache,
                                    batch, stream);
            }))
            return nullptr;
        if (!has_q) Py_RETURN_NONE;
        return THPVariable_Wrap(o);
    });
}

// (handle, head_dim, device, stream, q, cache, batch, scale, window, out) -> out
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded("paged_attention", n, 10, [&]() -> PyObject* {
        const Args a{args};
        auto* attn = static_cast<G4qAttn*>(a.pointer(0));
        const int64_t d = a.integer(1), dev = a.integer(2);
        void* stream = a.pointer(3);
        const auto* cache = static_cast<const G4qPagedCache*>(a.pointer(5));
        const auto* batch = static_cast<const G4qPagedBatch*>(a.pointer(6));
        const double scale = a.real(7);
        const long long window = a.integer(8);
        if (PyErr_Occurred()) return nullptr;
        if (window < 0 || window > 0x7FFFFFFFll) throw Refused{"window must be >= 0 (0: none) and below 2^31"};
        const at::Tensor& q = tensor(args[4], "q");
        const G4qHeadRows cq = head_rows(q, d, dev, "q");
        G4qHeadRows co;
        const at::Tensor o = output(q, args[9], d, dev, "out", co);
        if (!call("g4q_paged_attention",
                  [&] { return fn_paged_attention(attn, &cq, q.size(0), cache, batch, (float)scale, (int32_t)window, &co, stream); }))
            return nullptr;
        return THPVariable_Wrap(o);
    });
}

// (address of g4q_qk_norm_rope, of g4q_kv_append, of g4q_paged_attention, raise_status)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4 || !PyCallable_Check(args[3])) {
        PyErr_SetString(PyExc_TypeError, "bind takes three addresses and a function");
        return nullptr;
    }
    void* p[3];
    for (int i = 0; i < 3; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    fn_qk_norm_rope = reinterpret_cast<decltype(fn_qk_norm_rope)>(p[0]);
    fn_kv_append = reinterpret_cast<decltype(fn_kv_append)>(p[1]);
    fn_paged_attention = reinterpret_cast<decltype(fn_paged_attention)>(p[2]);
    Py_INCREF(args[3]);
    Py_XDECREF(raise_status);
    raise_status = args[3];
    Py_RETURN_NONE;
}

template <PyObject* (*kF)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(kF)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<qk_norm_rope>("qk_norm_rope"), method<kv_append>("kv_append"),
                         method<paged_attention>("paged_attention"), method<bind>("bind"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_g4q_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__g4q_torch(void) { return PyModule_Create(&module); }
