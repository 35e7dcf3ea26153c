// Python's fast way to the operators in 8 bits: arguments are checked and packed here, from torch's tensors as they lie in memory, instead of attribute by attribute in Python (64 x 1024 rows through
// et_skip_rmsnorm: 6.1 us a call from Python before). A function returns the C ABI's status, or -1 where the arguments are not what it takes: then the caller's checks in Python, which name what is
// wrong, see them again. The C ABI is called by address: which library it is in is the caller's choice.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <algorithm>
#include <climits>
#include "../../include/et_b200.h"

namespace {

struct Entries {
    int (*skip_rmsnorm)(const et_skip_rmsnorm_args*);
    int (*quantise_rows)(const et_quantise_rows_args*);
    int (*fp8_linear)(const et_fp8_linear_args*);
    int (*cache_write)(const et_kv_cache_args*);
    int (*cache_read)(const et_kv_cache_args*);
    int (*attention_tree)(const et_attention_tree_args*);
} entries = {};

// What a call's tensors have in common, and whether all have been what they should be.
struct Call {
    int device = -1;
    void* stream = nullptr;
    bool ok = true;

    // stream: a number, or None for the current one
    explicit Call(PyObject* given) {
        device = c10::cuda::current_device();
        if (given == Py_None) {
            stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        } else {
            stream = PyLong_AsVoidPtr(given);
            if (PyErr_Occurred()) refuse();
        }
    }
    void refuse() {
        PyErr_Clear();
        ok = false;
    }
    const at::Tensor* tensor(PyObject* o) {
        if (!THPVariable_Check(o)) {
            ok = false;
            return nullptr;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.defined() || !t.is_cuda() || t.device().index() != device || t.layout() != c10::kStrided) {
            ok = false;
            return nullptr;
        }
        return &t;
    }
    static bool is(const at::Tensor& t, at::ScalarType a, at::ScalarType b) { return t.scalar_type() == a || t.scalar_type() == b; }
    // Rows with neighbouring elements: their address, and their pitch. None: nothing.
    void* rows(PyObject* o, at::ScalarType a, at::ScalarType b, int64_t n, int64_t width, int& pitch) {
        pitch = 0;
        if (o == Py_None) return nullptr;
        const at::Tensor* const t = tensor(o);
        if (!t || !is(*t, a, b) || t->dim() != 2 || t->size(0) != n || t->size(1) != width || (width > 1 && t->stride(1) != 1 && t->numel() > 0)) {
            ok = false;
            return nullptr;
        }
        const int64_t p = n > 1 ? t->stride(0) : width;
        if (p < 0 || p > INT_MAX) ok = false;
        pitch = (int)p;
        return t->data_ptr();
    }
    // A contiguous array of n elements (below 0: of any number). None: nothing.
    void* array(PyObject* o, at::ScalarType type, int64_t n) {
        if (o == Py_None) return nullptr;
        const at::Tensor* const t = tensor(o);
        if (!t || t->scalar_type() != type || t->dim() != 1 || (n >= 0 && t->size(0) != n) || !t->is_contiguous()) {
            ok = false;
            return nullptr;
        }
        return t->data_ptr();
    }
    float* scales(PyObject* o, int64_t n, int64_t width) {
        if (o == Py_None) return nullptr;
        const at::Tensor* const t = tensor(o);
        if (!t || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != (width + 127) / 128 || t->size(1) != n || !t->is_contiguous()) {
            ok = false;
            return nullptr;
        }
        return static_cast<float*>(t->data_ptr());
    }
    // (rows, columns) of a matrix of halves or bytes, 0 and 0 where it is none
    bool shape(PyObject* o, int64_t& n, int64_t& width) {
        const at::Tensor* const t = tensor(o);
        if (!t || t->dim() != 2) return ok = false;
        n = t->size(0);
        width = t->size(1);
        if (n > INT_MAX || width > INT_MAX) ok = false;
        return ok;
    }
    // codes int8 [pages, 2, heads, page, head_dim] and scales
    bool cache(PyObject* codes, PyObject* scales, const at::Tensor*& c, const at::Tensor*& s) {
        c = tensor(codes);
        s = tensor(scales);
        if (!ok || c->scalar_type() != at::kChar || s->scalar_type() != at::kFloat || c->dim() != 5 || s->dim() != 4 || c->size(1) != 2 || !c->is_contiguous() || !s->is_contiguous()) return ok = false;
        for (int i = 0; i < 4; ++i)
            if (c->size(i) != s->size(i) || c->size(i) > INT_MAX) ok = false;
        return ok = ok && c->size(4) <= INT_MAX;
    }
    int number(PyObject* o) {
        const long v = PyLong_AsLong(o);
        if ((v == -1 && PyErr_Occurred()) || v < INT_MIN || v > INT_MAX) refuse();
        return (int)v;
    }
    float real(PyObject* o) {
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) refuse();
        return (float)v;
    }
};

// Calls the C ABI without Python's lock: a launch waits where the device's queue is full, for as long as what is queued takes.
template <typename Args>
PyObject* run(int (*entry)(const Args*), const Args& a) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = entry(&a);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

constexpr int64_t kMostKeys = 0x7ff00000;   // that et_attention_tree takes
constexpr at::ScalarType kE4m3 = at::ScalarType::Float8_e4m3fn;
PyObject* unsuitable() { return PyLong_FromLong(-1); }

// (out, x, skip, gamma, residual, scales, eps, stream)
PyObject* skip_rmsnorm(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 8 || !entries.skip_rmsnorm) return unsuitable();
    Call c(o[7]);
    int64_t rows, width;
    if (!c.shape(o[1], rows, width)) return unsuitable();
    et_skip_rmsnorm_args a = {};
    a.x = c.rows(o[1], at::kHalf, at::kHalf, rows, width, a.x_pitch);
    a.skip = c.rows(o[2], at::kHalf, at::kHalf, rows, width, a.skip_pitch);
    a.gamma = c.array(o[3], at::kHalf, width);
    a.residual = c.rows(o[4], at::kHalf, at::kHalf, rows, width, a.residual_pitch);
    a.scales = c.scales(o[5], rows, width);
    a.out = o[5] == Py_None ? c.rows(o[0], at::kHalf, at::kHalf, rows, width, a.out_pitch) : c.rows(o[0], kE4m3, at::kByte, rows, width, a.out_pitch);
    a.eps = c.real(o[6]);
    a.stream = c.stream;
    a.rows = (int)rows;
    a.width = (int)width;
    return c.ok ? run(entries.skip_rmsnorm, a) : unsuitable();
}

// (out, scales, x, stream)
PyObject* quantise_rows(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 4 || !entries.quantise_rows) return unsuitable();
    Call c(o[3]);
    int64_t rows, width;
    if (!c.shape(o[2], rows, width)) return unsuitable();
    et_quantise_rows_args a = {};
    a.x = c.rows(o[2], at::kHalf, at::kHalf, rows, width, a.x_pitch);
    a.out = c.rows(o[0], kE4m3, at::kByte, rows, width, a.out_pitch);
    a.scales = c.scales(o[1], rows, width);
    a.stream = c.stream;
    a.rows = (int)rows;
    a.width = (int)width;
    return c.ok ? run(entries.quantise_rows, a) : unsuitable();
}

// (weight, in_feat, out_feat, gelu, out, x, x_scales, stream)
PyObject* fp8_linear(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 8 || !entries.fp8_linear) return unsuitable();
    Call c(o[7]);
    int64_t tokens, width;
    if (!c.shape(o[5], tokens, width)) return unsuitable();
    et_fp8_linear_args a = {};
    const int in_feat = c.number(o[1]), out_feat = c.number(o[2]);
    a.weight = static_cast<const et_fp8_weight*>(PyLong_AsVoidPtr(o[0]));
    if (PyErr_Occurred()) c.refuse();
    a.x = c.rows(o[5], kE4m3, at::kByte, tokens, in_feat, a.x_pitch);
    a.y = c.rows(o[4], at::kHalf, at::kHalf, tokens, out_feat, a.y_pitch);
    a.x_scales = c.scales(o[6], tokens, in_feat);
    a.stream = c.stream;
    a.tokens = (int)tokens;
    a.gelu = c.number(o[3]);
    return c.ok ? run(entries.fp8_linear, a) : unsuitable();
}

// (write, codes, scales, k, v, slots, stream)
PyObject* kv_cache(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 7 || !entries.cache_write || !entries.cache_read) return unsuitable();
    Call c(o[6]);
    const at::Tensor *codes, *scales;
    int64_t tokens, width;
    if (!c.cache(o[1], o[2], codes, scales) || !c.shape(o[3], tokens, width)) return unsuitable();
    et_kv_cache_args a = {};
    a.codes = codes->data_ptr();
    a.scales = static_cast<float*>(scales->data_ptr());
    a.pages = (int)codes->size(0);
    a.heads = (int)codes->size(2);
    a.page = (int)codes->size(3);
    a.head_dim = (int)codes->size(4);
    a.k = c.rows(o[3], at::kHalf, at::kHalf, tokens, (int64_t)a.heads * a.head_dim, a.k_pitch);
    a.v = c.rows(o[4], at::kHalf, at::kHalf, tokens, (int64_t)a.heads * a.head_dim, a.v_pitch);
    a.slots = static_cast<const int*>(c.array(o[5], at::kInt, tokens));
    a.stream = c.stream;
    a.tokens = (int)tokens;
    const bool write = o[0] == Py_True;
    return c.ok ? run(write ? entries.cache_write : entries.cache_read, a) : unsuitable();
}

// (out, q, codes, scales, table, k_lens, tree, cu_seqlens, max_q_len, max_k_len, scale, stream)
PyObject* attention_tree(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 12 || !entries.attention_tree) return unsuitable();
    Call c(o[11]);
    const at::Tensor *codes, *scales;
    int64_t tokens, width, batch, most;
    if (!c.cache(o[2], o[3], codes, scales) || !c.shape(o[1], tokens, width) || !c.shape(o[4], batch, most)) return unsuitable();
    const int64_t head_dim = codes->size(4), heads = codes->size(2), page = codes->size(3);
    const at::Tensor* const table = c.tensor(o[4]);
    if (head_dim < 1 || heads < 1 || width % head_dim || table->scalar_type() != at::kInt || !table->is_contiguous() || o[5] == Py_None) return unsuitable();
    et_attention_tree_args a = {};
    a.q = c.rows(o[1], at::kHalf, at::kHalf, tokens, width, a.q_pitch);
    a.out = c.rows(o[0], at::kHalf, at::kHalf, tokens, width, a.out_pitch);
    a.codes = codes->data_ptr();
    a.scales = static_cast<const float*>(scales->data_ptr());
    a.table = static_cast<const int*>(table->data_ptr());
    a.k_lens = static_cast<const int*>(c.array(o[5], at::kInt, batch));
    a.tree = static_cast<const int64_t*>(c.array(o[6], at::kLong, tokens));
    a.cu_seqlens = static_cast<const int*>(c.array(o[7], at::kInt, batch + 1));
    a.stream = c.stream;
    a.nhead = (int)(width / head_dim);
    a.nhead_kv = (int)heads;
    a.head_dim = (int)head_dim;
    a.batch = (int)batch;
    a.q_tokens = (int)tokens;
    a.pages = (int)codes->size(0);
    a.page = (int)page;
    a.table_width = (int)most;
    a.max_q_len = c.number(o[8]);
    a.max_k_len = c.number(o[9]);
    if (a.max_q_len == 0) a.max_q_len = o[7] == Py_None ? 1 : 64;
    if (a.max_k_len == 0) a.max_k_len = (int)std::min<int64_t>(most * page, kMostKeys);
    a.scale = c.real(o[10]);
    return c.ok ? run(entries.attention_tree, a) : unsuitable();
}

// Addresses of the C ABI's functions, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
    void* at[6];
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "six addresses expected");
        return nullptr;
    }
    for (int i = 0; i < 6; ++i) {
        at[i] = PyLong_AsVoidPtr(o[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    entries.skip_rmsnorm = reinterpret_cast<decltype(entries.skip_rmsnorm)>(at[0]);
    entries.quantise_rows = reinterpret_cast<decltype(entries.quantise_rows)>(at[1]);
    entries.fp8_linear = reinterpret_cast<decltype(entries.fp8_linear)>(at[2]);
    entries.cache_write = reinterpret_cast<decltype(entries.cache_write)>(at[3]);
    entries.cache_read = reinterpret_cast<decltype(entries.cache_read)>(at[4]);
    entries.attention_tree = reinterpret_cast<decltype(entries.attention_tree)>(at[5]);
    Py_RETURN_NONE;
}

// C++ exceptions of torch do not leave through Python's C interface.
template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* o, Py_ssize_t n) {
    try {
        return kFunction(self, o, n);
    } catch (...) {
        PyErr_Clear();
        return unsuitable();
    }
}
template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
constexpr PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<kFunction>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<skip_rmsnorm>("skip_rmsnorm"), method<quantise_rows>("quantise_rows"), method<fp8_linear>("fp8_linear"), method<kv_cache>("kv_cache"),
                         method<attention_tree>("attention_tree"), method<bind>("bind"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
