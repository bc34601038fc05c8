// The per-call path of the torch launchers (drinkme_amd/radix_ops.py) and of
// the key/value cache's operators (drinkme_amd/kv_ops.py) as a CPython
// extension: one call checks the activation, allocates the output
// with torch and launches through the C ABI. What bounds a decode step's
// small calls is the host: through ctypes and Python's own checks a call of
// one Linear took 10.1 us on the host for a 5.5 us kernel (k_proj of 1024 x
// 4096, M = 1), a grouped attention block 33.6 us for 20.6 us of kernels.
//
// Every function takes the plain case alone (dense contiguous GPU tensors of
// the types, shapes and device the launcher was built for, and a descriptor
// whose buffers are still its runtime dict's) and returns None for anything
// else, having launched nothing: the caller's general path then copies,
// rebuilds its descriptor or raises.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "dmx_kv.h"
#include "dmx_radix.h"

namespace {

constexpr int kMaxRows = 8, kMaxGroup = 16;

// A dense strided tensor of the GPU that no torch wrapper (functorch, a
// dispatch subclass, a lazy negation) stands in front of.
bool plain(const at::Tensor& t) {
    using K = c10::DispatchKey;
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage() &&
           !t.key_set().has_any(c10::DispatchKeySet({K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Functionalize,
                                                     K::Python, K::Negative, K::Conjugate, K::ZeroTensor})) &&
           t.is_contiguous();
}

// The tensor of an exact torch.Tensor or Parameter, null for anything else.
const at::Tensor* exact(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

int code(at::ScalarType t) { return t == at::kBFloat16 ? DMX_BF16 : t == at::kFloat ? DMX_F32 : -1; }

// Rows of x [..., C], 0 where x is not a plain [..., C] of 1..8 rows on
// device `index` in a type that the kernels take.
uint32_t rows_of(const at::Tensor* x, int64_t C, int64_t index) {
    if (!x || !plain(*x) || x->get_device() != index || code(x->scalar_type()) < 0) return 0;
    if (x->dim() == 0 || C <= 0 || x->size(-1) != C) return 0;
    const int64_t m = x->numel() / C;
    return m >= 1 && m <= kMaxRows ? (uint32_t)m : 0;
}

// Whether `o` (None or a bias of R elements) is taken; its address and type.
bool bias_of(PyObject* o, int64_t R, int64_t index, const void*& at, int& dtype) {
    at = nullptr;
    dtype = 0;
    if (o == Py_None) return true;
    const at::Tensor* b = exact(o);
    if (!b || !plain(*b) || b->get_device() != index || b->numel() != R || code(b->scalar_type()) < 0) return false;
    at = b->const_data_ptr();
    dtype = code(b->scalar_type());
    return true;
}

// Whether the descriptor's buffers are those in the runtime dict p.
PyObject* g_keys[4];  // "rx_data", "rx_offsets", "rx_palette", "rx_schedule"
bool current(const dmx_radix_tensor* t, PyObject* p) {
    const void* held[4] = {t->data, t->offsets, t->palette, t->schedule};
    if (!PyDict_Check(p)) return false;
    for (int i = 0; i < 4; ++i) {
        PyObject* o = PyDict_GetItem(p, g_keys[i]);  // borrowed
        const at::Tensor* b = o && o != Py_None ? exact(o) : nullptr;
        if (!b ? i != 3 || (o && o != Py_None) : !plain(*b)) return false;
        const void* at = b && b->numel() ? b->const_data_ptr() : nullptr;
        if (at != held[i]) return false;
    }
    return true;
}

at::ScalarType dtype_of(PyObject* o) {
    return THPDtype_Check(o) ? reinterpret_cast<THPDtype*>(o)->scalar_type : at::ScalarType::Undefined;
}

at::Tensor output(const at::Tensor& x, int64_t R, at::ScalarType dtype) {
    c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = R;
    return at::empty(sizes, at::TensorOptions().device(x.device()).dtype(dtype));
}

PyObject* launch_failed(const char* what, const char* err) {
    PyErr_SetString(PyExc_RuntimeError, (std::string(what) + ": " + err).c_str());
    return nullptr;
}

bool modes_off() { return !at::impl::torch_function_mode_enabled(); }

// rows(descriptor address, p, x, bias, out dtype, R, C, device index, stream)
PyObject* rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) return launch_failed("rows", "nine arguments");
    const auto* t = static_cast<const dmx_radix_tensor*>(PyLong_AsVoidPtr(a[0]));
    const at::Tensor* x = exact(a[2]);
    const at::ScalarType od = dtype_of(a[4]);
    const int64_t R = PyLong_AsLongLong(a[5]), C = PyLong_AsLongLong(a[6]), index = PyLong_AsLongLong(a[7]);
    void* stream = PyLong_AsVoidPtr(a[8]);
    if (PyErr_Occurred()) return nullptr;
    const uint32_t m = rows_of(x, C, index);
    const void* bias;
    int bd;
    if (!t || !m || code(od) < 0 || !modes_off() || !bias_of(a[3], R, index, bias, bd) || !current(t, a[1]))
        Py_RETURN_NONE;
    at::Tensor out;
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        out = output(*x, R, od);
        st = dmx_radix_gemv(t, x->const_data_ptr(), code(x->scalar_type()), m, bias, bd, out.mutable_data_ptr(), code(od),
                            stream, err, sizeof err);
    }
    return st ? launch_failed("dmx_radix_gemv", err) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// group(descriptor table address, [p, ...], x, bias table address, bias dtype
// code, out dtype, (R, ...), C, device index, stream)
PyObject* group(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !PyList_Check(a[1]) || !PyTuple_Check(a[6])) return launch_failed("group", "ten arguments");
    const auto* const* ts = static_cast<const dmx_radix_tensor* const*>(PyLong_AsVoidPtr(a[0]));
    const Py_ssize_t k = PyTuple_GET_SIZE(a[6]);
    const at::Tensor* x = exact(a[2]);
    const void* const* bias = static_cast<const void* const*>(PyLong_AsVoidPtr(a[3]));
    const long bd = PyLong_AsLong(a[4]);
    const at::ScalarType od = dtype_of(a[5]);
    const int64_t C = PyLong_AsLongLong(a[7]), index = PyLong_AsLongLong(a[8]);
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    const uint32_t m = rows_of(x, C, index);
    if (!ts || !m || code(od) < 0 || !modes_off() || k < 1 || k > kMaxGroup || PyList_GET_SIZE(a[1]) != k) Py_RETURN_NONE;
    int64_t R[kMaxGroup];
    for (Py_ssize_t i = 0; i < k; ++i) {
        if (!current(ts[i], PyList_GET_ITEM(a[1], i))) Py_RETURN_NONE;
        R[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(a[6], i));
    }
    if (PyErr_Occurred()) return nullptr;
    at::Tensor outs[kMaxGroup];
    void* at_out[kMaxGroup];
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        for (Py_ssize_t i = 0; i < k; ++i) {
            outs[i] = output(*x, R[i], od);
            at_out[i] = outs[i].mutable_data_ptr();
        }
        st = dmx_radix_gemv_group(ts, (uint32_t)k, x->const_data_ptr(), code(x->scalar_type()), m, bias, (int)bd, at_out,
                                  code(od), stream, err, sizeof err);
    }
    if (st) return launch_failed("dmx_radix_gemv_group", err);
    PyObject* list = PyList_New(k);
    if (!list) return nullptr;
    for (Py_ssize_t i = 0; i < k; ++i) {
        PyObject* o = THPVariable_Wrap(std::move(outs[i]));
        if (!o) {
            Py_DECREF(list);
            return nullptr;
        }
        PyList_SET_ITEM(list, i, o);
    }
    return list;
    END_HANDLE_TH_ERRORS
}

// narrow(w, x, bias, stream): x [..., C] against the raw bf16 w [R, C], in x's dtype
PyObject* narrow(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) return launch_failed("narrow", "four arguments");
    const at::Tensor *w = exact(a[0]), *x = exact(a[1]);
    void* stream = PyLong_AsVoidPtr(a[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!w || !plain(*w) || w->dim() != 2 || w->scalar_type() != at::kBFloat16 || !modes_off()) Py_RETURN_NONE;
    const int64_t R = w->size(0), C = w->size(1), index = w->get_device();
    const uint32_t m = rows_of(x, C, index);
    const void* bias;
    int bd;
    if (!m || R < 1 || R >= (1ll << 31) || C >= (1ll << 32) || !bias_of(a[2], R, index, bias, bd)) Py_RETURN_NONE;
    at::Tensor out;
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        const int xd = code(x->scalar_type());
        out = output(*x, R, x->scalar_type());
        st = dmx_gemv_narrow(static_cast<const uint16_t*>(w->const_data_ptr()), (uint32_t)R, (uint32_t)C,
                             x->const_data_ptr(), xd, m, bias, bd, out.mutable_data_ptr(), xd, stream, err, sizeof err);
    }
    return st ? launch_failed("dmx_gemv_narrow", err) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------- the key/value cache's operators --
//
// As above: the plain case or None. Plain here: tensors of the types, shapes
// and device that kv_ops documents, activations with adjacent channels, nothing
// that asks for a gradient. The tensors' device is made current for the launch:
// the null stream is the current device's, and so is a kernel's LDS limit.

constexpr int64_t kMost = 1ll << 30;

// A whole number; -1 for one that 64 bits do not hold.
int64_t whole(PyObject* o) {
    int over;
    const int64_t n = PyLong_AsLongLongAndOverflow(o, &over);
    return over ? -1 : n;
}

// Whether x asks for a gradient, or carries a tangent.
bool wants(const at::Tensor& x) {
    return (x.requires_grad() && at::GradMode::is_enabled()) ||
           (x._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
}

// A dense tensor of `dtype` and `dims` dimensions on device `index`.
const at::Tensor* dense(PyObject* o, at::ScalarType dtype, int64_t dims, int64_t index) {
    const at::Tensor* t = exact(o);
    return t && plain(*t) && t->scalar_type() == dtype && t->dim() == dims && t->get_device() == index ? t : nullptr;
}

// x [tokens, heads, dim], any strides but for adjacent channels.
bool rows_at(PyObject* o, const at::Tensor*& x, dmx_rows& r) {
    using K = c10::DispatchKey;
    x = exact(o);
    if (!x || !x->defined() || !x->is_cuda() || x->layout() != at::kStrided || !x->has_storage() || x->dim() != 3 ||
        x->key_set().has_any(c10::DispatchKeySet({K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Functionalize,
                                                  K::Python, K::Negative, K::Conjugate, K::ZeroTensor})))
        return false;
    if (code(x->scalar_type()) < 0 || x->stride(2) != 1 || x->size(0) >= kMost || x->size(1) >= kMost ||
        wants(*x))
        return false;
    r = {const_cast<void*>(x->const_data_ptr()), x->stride(0), x->stride(1), (uint32_t)x->size(1)};
    return true;
}

bool like(const at::Tensor& a, const at::Tensor& b) {
    return a.scalar_type() == b.scalar_type() && a.get_device() == b.get_device() && a.size(0) == b.size(0) &&
           a.size(2) == b.size(2);
}

dmx_rows dense_rows(const at::Tensor& t) {
    return {t.mutable_data_ptr(), t.size(1) * t.size(2), t.size(2), (uint32_t)t.size(1)};
}

bool table_of(PyObject* o, long layout, int64_t dim, int64_t index, dmx_rotary_table& r) {
    const at::Tensor* t = dense(o, at::kFloat, 3, index);
    if (!t || t->size(2) != 2 || 2 * t->size(1) > dim || t->size(0) >= kMost || wants(*t) ||
        reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16)
        return false;
    r = {static_cast<const float*>(t->const_data_ptr()), (uint32_t)t->size(0), (uint32_t)(2 * t->size(1)), (int)layout};
    return true;
}

PyObject* g_cache[4];  // "k_codes", "k_scales", "v_codes", "v_scales"
bool cache_of(PyObject* o, dmx_kv_cache& c, int64_t& index) {
    if (!PyDict_Check(o)) return false;
    const at::Tensor* t[4];
    for (int n = 0; n < 4; ++n) {
        PyObject* v = PyDict_GetItem(o, g_cache[n]);  // borrowed
        t[n] = v ? exact(v) : nullptr;
        if (!t[n] || !plain(*t[n]) || t[n]->scalar_type() != (n % 2 ? at::kByte : at::kInt) || t[n]->dim() != (n < 2 ? 4 : 5) ||
            t[n]->get_device() != t[0]->get_device())
            return false;
    }
    const int64_t pages = t[0]->size(0), heads = t[0]->size(1), page = t[0]->size(2), words = t[0]->size(3);
    if (pages >= kMost || heads >= kMost || page >= kMost || words >= kMost ||
        t[1]->sizes() != at::IntArrayRef({pages, heads, page, words / 4}) ||
        t[2]->sizes() != at::IntArrayRef({pages, heads, page / 8, words, 8}) ||
        t[3]->sizes() != at::IntArrayRef({pages, heads, page / 8, words / 4, 8}))
        return false;
    index = t[0]->get_device();
    c.k_codes = static_cast<uint32_t*>(t[0]->mutable_data_ptr());
    c.k_scales = static_cast<uint8_t*>(t[1]->mutable_data_ptr());
    c.v_codes = static_cast<uint32_t*>(t[2]->mutable_data_ptr());
    c.v_scales = static_cast<uint8_t*>(t[3]->mutable_data_ptr());
    c.pages = (uint32_t)pages, c.heads = (uint32_t)heads, c.page = (uint32_t)page, c.dim = (uint32_t)(8 * words);
    return true;
}

bool seqs_of(PyObject* table, PyObject* lengths, PyObject* cu, int64_t total, int64_t max_tokens, int64_t index,
             dmx_kv_seqs& s) {
    const at::Tensor *t = dense(table, at::kInt, 2, index), *l = dense(lengths, at::kInt, 1, index);
    const at::Tensor* c = cu == Py_None ? nullptr : dense(cu, at::kInt, 1, index);
    if (!t || !l || (cu != Py_None && !c) || total < 0 || total >= kMost) return false;
    const int64_t batch = l->size(0), cols = t->size(1);
    if (batch < 1 || batch >= kMost || cols < 1 || cols >= kMost || t->size(0) != batch || (c && c->size(0) != batch + 1) ||
        (!c && total % batch))
        return false;
    s.table = static_cast<const int32_t*>(t->const_data_ptr());
    s.lengths = static_cast<const int32_t*>(l->const_data_ptr());
    s.cu = c ? static_cast<const int32_t*>(c->const_data_ptr()) : nullptr;
    s.batch = (uint32_t)batch, s.table_cols = (uint32_t)cols, s.total = (uint32_t)total;
    s.max_tokens = (uint32_t)(c ? max_tokens : total / batch);
    return true;
}

at::Tensor dense_like(const at::Tensor& x) {
    return at::empty({x.size(0), x.size(1), x.size(2)}, at::TensorOptions().device(x.device()).dtype(x.scalar_type()));
}

PyObject* pair_of(at::Tensor&& a, at::Tensor&& b) {  // (b undefined: None)
    PyObject* p = PyTuple_New(2);
    if (!p) return nullptr;
    PyObject* x = THPVariable_Wrap(std::move(a));
    if (x) PyTuple_SET_ITEM(p, 0, x);
    PyObject* y = !x ? nullptr : b.defined() ? THPVariable_Wrap(std::move(b)) : (Py_INCREF(Py_None), Py_None);
    if (y) PyTuple_SET_ITEM(p, 1, y);
    if (!x || !y) {
        Py_DECREF(p);
        return nullptr;
    }
    return p;
}

// rotary(q, k or None, positions, table, layout code, stream) -> (q', k')
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) return launch_failed("rotary", "six arguments");
    const long layout = PyLong_AsLong(a[4]);
    void* stream = PyLong_AsVoidPtr(a[5]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *q, *k = nullptr, *p = exact(a[2]);
    dmx_rows in[2], out[2];
    dmx_rotary_table t;
    if (layout < 0 || !modes_off() || !rows_at(a[0], q, in[0])) Py_RETURN_NONE;
    const int count = a[1] == Py_None ? 1 : 2;
    if (count == 2 && (!rows_at(a[1], k, in[1]) || !like(*q, *k))) Py_RETURN_NONE;
    if (!p || !plain(*p) || p->dim() != 1 || p->size(0) != q->size(0) || p->get_device() != q->get_device() ||
        (p->scalar_type() != at::kInt && p->scalar_type() != at::kLong) || q->size(2) >= kMost ||
        !table_of(a[3], layout, q->size(2), q->get_device(), t))
        Py_RETURN_NONE;
    at::Tensor y, z;
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard on(q->device());
        y = dense_like(*q);
        out[0] = dense_rows(y);
        if (k) {
            z = dense_like(*k);
            out[1] = dense_rows(z);
        }
        st = dmx_rotary(in, out, count, (uint32_t)q->size(0), (uint32_t)q->size(2), code(q->scalar_type()), p->const_data_ptr(),
                        p->scalar_type() == at::kLong, &t, stream, err, sizeof err);
    }
    return st ? launch_failed("dmx_rotary", err) : pair_of(std::move(y), std::move(z));
    END_HANDLE_TH_ERRORS
}

// append(cache, k, v, block_table, lengths, cu, table or None, layout code, q
// or None, stream) -> True, or q'
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) return launch_failed("append", "ten arguments");
    const long layout = PyLong_AsLong(a[7]);
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    dmx_kv_cache c;
    dmx_kv_seqs s;
    dmx_rotary_table t;
    dmx_rows rk, rv, rq, out;
    const at::Tensor *k, *v, *q = nullptr;
    int64_t index;
    const bool turn = a[6] != Py_None, queries = a[8] != Py_None;
    if (layout < 0 || !modes_off() || !cache_of(a[0], c, index) || !rows_at(a[1], k, rk) || !rows_at(a[2], v, rv) ||
        !like(*k, *v) || k->get_device() != index || rk.heads != c.heads || rv.heads != c.heads || k->size(2) != c.dim ||
        !seqs_of(a[3], a[4], a[5], k->size(0), 0, index, s) || (turn && !table_of(a[6], layout, c.dim, index, t)) ||
        (queries && (!turn || !rows_at(a[8], q, rq) || !like(*q, *k))))
        Py_RETURN_NONE;
    at::Tensor y;
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard on(k->device());
        if (q) {
            y = dense_like(*q);
            out = dense_rows(y);
        }
        st = dmx_kv_append(&c, &s, &rk, &rv, q ? &rq : nullptr, q ? &out : nullptr, code(k->scalar_type()), turn ? &t : nullptr,
                           stream, err, sizeof err);
    }
    if (st) return launch_failed("dmx_kv_append", err);
    if (!q) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// read(cache, block_table, lengths, total, cu, stream) -> (k, v)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) return launch_failed("read", "six arguments");
    const int64_t total = whole(a[3]);
    void* stream = PyLong_AsVoidPtr(a[5]);
    if (PyErr_Occurred()) return nullptr;
    dmx_kv_cache c;
    dmx_kv_seqs s;
    int64_t index;
    if (!modes_off() || !cache_of(a[0], c, index) || !seqs_of(a[1], a[2], a[4], total, 0, index, s)) Py_RETURN_NONE;
    at::Tensor k, v;
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        const at::Device device(at::kCUDA, (c10::DeviceIndex)index);
        const c10::DeviceGuard on(device);
        const auto options = at::TensorOptions().device(device).dtype(at::kBFloat16);
        k = at::empty({total, (int64_t)c.heads, (int64_t)c.dim}, options);
        v = at::empty({total, (int64_t)c.heads, (int64_t)c.dim}, options);
        st = dmx_kv_read(&c, &s, static_cast<uint16_t*>(k.mutable_data_ptr()), static_cast<uint16_t*>(v.mutable_data_ptr()),
                         stream, err, sizeof err);
    }
    return st ? launch_failed("dmx_kv_read", err) : pair_of(std::move(k), std::move(v));
    END_HANDLE_TH_ERRORS
}

// One of at least 1, or 0 for None; -1 for anything less.
int64_t count_of(PyObject* o) {
    if (o == Py_None) return 0;
    const int64_t n = whole(o);
    return n < 1 ? -1 : n;
}

// attention(q, cache, block_table, lengths, cu, max_tokens or None, max_length
// or 0, scale or None, causal, window or None, lse, stream) -> out, or (out, lse)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12) return launch_failed("attention", "twelve arguments");
    const int64_t max_tokens = count_of(a[5]), max_length = whole(a[6]), window = count_of(a[9]);
    const double given = a[7] == Py_None ? 0 : PyFloat_AsDouble(a[7]);
    const int causal = PyObject_IsTrue(a[8]), want = PyObject_IsTrue(a[10]);
    void* stream = PyLong_AsVoidPtr(a[11]);
    if (PyErr_Occurred()) return nullptr;
    dmx_kv_cache c;
    dmx_kv_seqs s;
    dmx_rows r;
    const at::Tensor* q;
    int64_t index;
    if (!modes_off() || !cache_of(a[1], c, index) || !rows_at(a[0], q, r) || q->get_device() != index || q->size(2) != c.dim ||
        r.heads == 0 || c.heads == 0 || r.heads % c.heads || window < 0 || window >= kMost || max_length < 0 ||
        max_length >= (1ll << 32) || max_tokens < 0 || max_tokens >= kMost || (max_tokens && a[4] == Py_None) ||
        !seqs_of(a[2], a[3], a[4], q->size(0), max_tokens ? max_tokens : q->size(0), index, s))
        Py_RETURN_NONE;
    const double scale = a[7] == Py_None ? 1 / std::sqrt((double)c.dim) : given;
    at::Tensor out, lse, ws;
    char err[512];
    int st;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard on(q->device());
        const int dt = code(q->scalar_type());
        out = dense_like(*q);
        if (want) lse = at::empty({q->size(0), q->size(1)}, at::TensorOptions().device(q->device()).dtype(at::kFloat));
        const uint64_t bytes = s.total ? dmx_kv_attention_workspace(&c, &s, r.heads, dt, (uint32_t)max_length, (uint32_t)window) : 0;
        if (bytes) ws = at::empty({(int64_t)bytes}, at::TensorOptions().device(q->device()).dtype(at::kByte));
        st = dmx_kv_attention(&c, &s, &r, dt, (float)scale, causal, (uint32_t)window, (uint32_t)max_length,
                              out.mutable_data_ptr(), want ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr,
                              bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream, err, sizeof err);
    }
    if (st) return launch_failed("dmx_kv_attention", err);
    return want ? pair_of(std::move(out), std::move(lse)) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}
PyMethodDef g_methods[] = {{"rows", fast<rows>(), METH_FASTCALL, nullptr},
                           {"group", fast<group>(), METH_FASTCALL, nullptr},
                           {"narrow", fast<narrow>(), METH_FASTCALL, nullptr},
                           {"rotary", fast<rotary>(), METH_FASTCALL, nullptr},
                           {"append", fast<append>(), METH_FASTCALL, nullptr},
                           {"read", fast<read>(), METH_FASTCALL, nullptr},
                           {"attention", fast<attention>(), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "dmx_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dmx_calls(void) {
    const char* names[4] = {"rx_data", "rx_offsets", "rx_palette", "rx_schedule"};
    for (int i = 0; i < 4; ++i)
        if (!(g_keys[i] = PyUnicode_InternFromString(names[i]))) return nullptr;
    const char* buffers[4] = {"k_codes", "k_scales", "v_codes", "v_scales"};
    for (int i = 0; i < 4; ++i)
        if (!(g_cache[i] = PyUnicode_InternFromString(buffers[i]))) return nullptr;
    PyObject* m = PyModule_Create(&g_module);
    // (the torch whose headers this was compiled with: the loader compares)
    if (m && PyModule_AddStringConstant(m, "torch_version", DMX_TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
