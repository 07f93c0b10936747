// The cache operators' call path from Python (module q4rdna._kv_torch): reads the
// torch tensors, checks them and calls the C ABI.  The same calls through ctypes
// cost 20 to 35 us of host time, several times the kernels of a decode step.
//
// Every function runs with the cache's device current, on that device's current
// stream, and allocates there.  Argument errors raise ValueError; a status of the
// library goes to the package's check(), which raises its own error.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "q4rdna.h"

namespace {

// What KVCache and KVBatch keep for a call (q4rdna/__init__.py holds the same structures)
struct CacheRec {
    q4rdna_kv_cache desc;
    int device;  // -1: not a CUDA device
};
struct BatchRec {
    q4rdna_kv_batch desc;
    int pages;  // entries of a page table row
    int limit;  // the user's max_length, 0: none
    int device;
};

PyObject *g_check = nullptr;

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python error is set

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) throw Refused(std::string("kv cache operators: ") + name + " is a tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.requires_grad() && c10::GradMode::is_enabled())
        throw Refused(std::string("kv cache operators have no gradients: ") + name + " requires one (not under torch.no_grad())");
    // (torch.no_grad does not turn forward mode off)
    if (t._fw_grad(0).defined())
        throw Refused(std::string("kv cache operators have no gradients: ") + name + " carries a tangent");
    return t;
}
bool given(PyObject *o) { return o != Py_None; }

template <class Rec>
const Rec &record(PyObject *o) {
    const void *p = PyLong_AsVoidPtr(o);
    if (p == nullptr) {
        if (PyErr_Occurred()) throw Raised();
        throw Refused("kv cache operators: no cache or batch");
    }
    return *static_cast<const Rec *>(p);
}
long integer(PyObject *o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    if (v < INT_MIN || v > INT_MAX) throw Refused("kv cache operators: a number is beyond 32 bits");
    return v;
}
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return (float)v;
}

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return Q4RDNA_F32;
        case at::kHalf: return Q4RDNA_F16;
        case at::kBFloat16: return Q4RDNA_BF16;
        default: throw Refused("kv cache operators take float32, float16 or bfloat16");
    }
}

void on_device(const at::Tensor &t, const CacheRec &c, const char *name) {
    if (!t.is_cuda() || t.get_device() != c.device)
        throw Refused(std::string("kv cache operators: ") + name + " is a CUDA tensor on the cache's device");
}

struct Rows {
    int heads;
    int64_t stride;
};
// [rows, heads, head_dim] or [rows, heads * head_dim], the heads of a row contiguous;
// heads 0: any number; like: the same type and number of rows
Rows rows_of(const at::Tensor &x, int heads, const CacheRec &c, const at::Tensor *like, const char *name) {
    const int64_t D = c.desc.head_dim;
    const auto size = x.sizes(), stride = x.strides();
    int64_t n = 0;
    bool ok = false;
    if (size.size() == 3) {
        n = size[1];
        ok = size[2] == D && stride[2] == 1 && (stride[1] == D || n == 1);
    } else if (size.size() == 2) {
        n = size[1] / D;
        ok = size[1] % D == 0 && stride[1] == 1;
    }
    if (!ok || (heads != 0 && n != heads) || n > INT_MAX)
        throw Refused(std::string("kv cache operators: ") + name + " is [rows, heads, " + std::to_string(D) +
                      "], the heads of a row contiguous" + (heads ? ", " + std::to_string(heads) + " heads" : ""));
    if (size[0] > INT_MAX) throw Refused("kv cache operators: too many rows");
    if (like != nullptr && (x.scalar_type() != like->scalar_type() || size[0] != like->size(0)))
        throw Refused(std::string("kv cache operators: ") + name + " has another type or number of rows");
    on_device(x, c, name);
    return {(int)n, size[0] > 1 ? stride[0] : n * D};
}

// A contiguous vector of n elements, or null
const void *vector_of(PyObject *o, at::ScalarType type, int64_t n, const CacheRec &c, const char *name) {
    if (!given(o)) return nullptr;
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != type || !t.is_contiguous() || t.numel() != n)
        throw Refused(std::string("kv cache operators: ") + name + " is a contiguous " + c10::toString(type) + " tensor of " +
                      std::to_string(n));
    on_device(t, c, name);
    return t.data_ptr();
}

q4rdna_kv_batch batch_for(const BatchRec &b, const CacheRec &c) {
    const int64_t room = (int64_t)b.pages * c.desc.page_tokens;
    if (b.limit > room)
        throw Refused("kv batch: max_length " + std::to_string(b.limit) + " is more than the page table's " +
                      std::to_string(room) + " tokens");
    if (b.device != c.device) throw Refused("kv cache operators: the batch is on another device than the cache");
    q4rdna_kv_batch d = b.desc;
    d.max_length = b.limit > 0 ? b.limit : (int)std::min<int64_t>(room, 1 << 30);
    return d;
}

void check(q4rdna_status st, const char *what) {
    if (st == Q4RDNA_OK) return;
    PyObject *r = PyObject_CallFunction(g_check, "is", (int)st, what);
    Py_XDECREF(r);
    if (r != nullptr) PyErr_SetString(PyExc_RuntimeError, what);
    throw Raised();
}

// Runs f and turns C++ exceptions into Python ones
template <class F>
PyObject *guarded(F f) {
    try {
        return f();
    } catch (const Raised &) {
    } catch (const Refused &e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// append(cache, batch, k, v, q, q_out, inv_freq, rotary_dim, rope, positions, q_norm, k_norm, norm_eps)
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 13) throw Refused("append takes 13 arguments");
        const CacheRec &c = record<CacheRec>(a[0]);
        const q4rdna_kv_batch b = batch_for(record<BatchRec>(a[1]), c);
        const at::Tensor &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
        q4rdna_kv_append_args g{};
        g.type = type_of(k.scalar_type());
        g.k_stride = rows_of(k, c.desc.kv_heads, c, nullptr, "k").stride;
        g.v_stride = rows_of(v, c.desc.kv_heads, c, &k, "v").stride;
        g.tokens = (int)k.size(0);
        g.k = k.data_ptr();
        g.v = v.data_ptr();
        g.rotary_dim = (int)integer(a[7]);
        g.rope = (int)integer(a[8]);
        const int64_t D = c.desc.head_dim;
        g.inv_freq = (const float *)vector_of(a[6], at::kFloat, (g.rotary_dim ? g.rotary_dim : D) / 2, c, "inv_freq");
        g.positions = (const int32_t *)vector_of(a[9], at::kInt, g.tokens, c, "positions");
        g.q_norm = (const float *)vector_of(a[10], at::kFloat, D, c, "q_norm");
        g.k_norm = (const float *)vector_of(a[11], at::kFloat, D, c, "k_norm");
        g.norm_eps = real(a[12]);
        const c10::cuda::CUDAGuard on((c10::DeviceIndex)c.device);
        at::Tensor out;
        if (given(a[4])) {
            const at::Tensor &q = tensor(a[4], "q");
            const Rows r = rows_of(q, 0, c, &k, "q");
            out = given(a[5]) ? tensor(a[5], "q_out") : at::empty(q.sizes(), q.options().requires_grad(false));
            g.q_out_stride = rows_of(out, r.heads, c, &k, "q_out").stride;
            g.heads = r.heads;
            g.q_stride = r.stride;
            g.q = q.data_ptr();
            g.q_out = out.data_ptr();
        } else if (given(a[5])) {
            throw Refused("kv_append: q_out without q");
        }
        check(q4rdna_kv_append(&c.desc, &b, &g, c10::cuda::getCurrentCUDAStream().stream()), "kv_append");
        if (!out.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(out);
    });
}

// attention(cache, batch, q, scale, window, out)
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 6) throw Refused("attention takes 6 arguments");
        const CacheRec &c = record<CacheRec>(a[0]);
        const q4rdna_kv_batch b = batch_for(record<BatchRec>(a[1]), c);
        const at::Tensor &q = tensor(a[2], "q");
        q4rdna_kv_attention_args g{};
        g.type = type_of(q.scalar_type());
        const Rows r = rows_of(q, 0, c, nullptr, "q");
        g.scale = real(a[3]);
        g.window = (int)integer(a[4]);
        const c10::cuda::CUDAGuard on((c10::DeviceIndex)c.device);
        at::Tensor out = given(a[5]) ? tensor(a[5], "out") : at::empty(q.sizes(), q.options().requires_grad(false));
        g.out_stride = rows_of(out, r.heads, c, &q, "out").stride;
        g.tokens = (int)q.size(0);
        g.heads = r.heads;
        g.q = q.data_ptr();
        g.out = out.data_ptr();
        g.q_stride = r.stride;
        const size_t bytes = q4rdna_kv_attention_workspace_bytes(&c.desc, &b, &g);
        // a workspace of its own for each call: calls on different streams and captured
        // graphs (whose pool it then belongs to) share nothing
        at::Tensor ws;
        if (bytes > 0) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte).requires_grad(false));
        check(q4rdna_kv_attention(&c.desc, &b, &g, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                                  c10::cuda::getCurrentCUDAStream().stream()),
              "kv_attention");
        return THPVariable_Wrap(out);
    });
}

// dequant(cache, pages, dtype)
PyObject *dequant(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 3) throw Refused("dequant takes 3 arguments");
        const CacheRec &c = record<CacheRec>(a[0]);
        const at::Tensor &pages = tensor(a[1], "pages");
        if (pages.numel() > INT_MAX) throw Refused("kv_dequant: too many pages");
        const void *list = vector_of(a[1], at::kInt, pages.numel(), c, "pages");
        if (!THPDtype_Check(a[2])) throw Refused("kv_dequant: dtype is a torch.dtype");
        const at::ScalarType type = reinterpret_cast<THPDtype *>(a[2])->scalar_type;
        const int t = type_of(type);
        const c10::cuda::CUDAGuard on((c10::DeviceIndex)c.device);
        const auto options = pages.options().dtype(type);
        const std::array<int64_t, 4> size{pages.numel(), c.desc.kv_heads, c.desc.page_tokens, c.desc.head_dim};
        const at::Tensor k = at::empty(size, options), v = at::empty(size, options);
        check(q4rdna_kv_dequant(&c.desc, (const int32_t *)list, (int)pages.numel(), t, k.data_ptr(), v.data_ptr(),
                                c10::cuda::getCurrentCUDAStream().stream()),
              "kv_dequant");
        return Py_BuildValue("NN", THPVariable_Wrap(k), THPVariable_Wrap(v));
    });
}

PyObject *set_check(PyObject *, PyObject *f) {
    Py_INCREF(f);
    Py_XDECREF(g_check);
    g_check = f;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
    {"dequant", (PyCFunction)(void (*)(void))dequant, METH_FASTCALL, nullptr},
    {"set_check", set_check, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_kv_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_torch(void) {
    PyObject *m = PyModule_Create(&module_def);
    // the package compares it with the torch that it runs under
    if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
