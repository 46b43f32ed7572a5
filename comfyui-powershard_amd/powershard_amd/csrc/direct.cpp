// direct.cpp -- the decoder operators' calls that have nothing to convert, copy or report, as a CPython module.
//
// At one token the host's part of a call is longer than its kernel, and in Python most of it is the checks
// of up to eight tensors, the allocations and the foreign call's 16 to 27 arguments.  Host time of a call of ops.py,
// its general path and through here: add_rms_norm (x + residual, int8) 11.0 and 6.0 us, kv_write 7.6 and 3.5,
// kv_read 9.7 and 5.5, paged_attention 10.4 and 5.0 (with a second launch for the join, and memory for its parts, 15.0 and 8.1).
//
// The functions take what ops.py was called with and the current stream, and return None whenever the
// arguments are not plainly what the library takes (another type or layout, a copy to make, something to
// refuse, a tensor subclass, memory that ran out): ops.py's general path then does the work or says what is
// wrong.  They hold no rule that is not also there, and no arithmetic.
//
// bind({name: address}): the library's entry points, from the handle that the package has loaded.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>
#include <ATen/ATen.h>

#include "psquant.h"

#include <cmath>

namespace {

decltype(&psq_add_rms_norm) f_norm;
decltype(&psq_kv_write) f_write;
decltype(&psq_kv_read) f_read;
decltype(&psq_paged_attention_workspace_bytes) f_attend_bytes;
decltype(&psq_paged_attention_own_workspace) f_attend_own;
decltype(&psq_paged_attention) f_attend;

// Other threads run while memory is allocated and the kernel is launched (a full queue makes the launch wait).
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// A strided tensor on GPU `index` (-1: any), or None.
struct Arg {
    const at::Tensor *t = nullptr;
    bool none = false;
};

bool take(PyObject *o, int64_t index, Arg &a)
{
    if (o == Py_None) {
        a.none = true;
        return true;
    }
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || !t.has_storage() || t.layout() != at::kStrided || (index >= 0 && t.get_device() != index)) return false;
    a.t = &t;
    return true;
}

int half_type(at::ScalarType s) { return s == at::kBFloat16 ? PSQ_BF16 : s == at::kHalf ? PSQ_F16 : -1; }
int float_type(at::ScalarType s) { return s == at::kFloat ? PSQ_F32 : half_type(s); }
int code_type(at::ScalarType s)
{
    return s == at::kChar ? PSQ_CODES_I8 : s == at::kFloat8_e4m3fn ? PSQ_CODES_E4M3 : half_type(s) >= 0 ? PSQ_CODES_NONE : -1;
}

bool aligned(const at::Tensor &t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
bool dense(const at::Tensor &t) { return t.is_contiguous() && aligned(t); }

PyObject *none() { Py_RETURN_NONE; }

// A tuple of the tensors, None for those that are not defined.
template <class... T>
PyObject *tuple(const T &...tensors)
{
    PyObject *t = PyTuple_New(sizeof...(tensors));
    Py_ssize_t i = 0;
    bool whole = t != nullptr;
    for (const at::Tensor *each : {&tensors...}) {
        if (!whole) break;
        PyObject *o = each->defined() ? THPVariable_Wrap(*each) : none();
        whole = o != nullptr;
        PyTuple_SET_ITEM(t, i++, o);
    }
    if (!whole) Py_CLEAR(t);
    return t;
}

struct Pools {
    Arg k, v, ks, vs;
    int codes = 0;
    int64_t pages = 0, page = 0;
    int heads = 0, dim = 0;

    bool take_from(PyObject *const *o, int64_t index)
    {
        if (!take(o[0], index, k) || !take(o[1], index, v) || !take(o[2], index, ks) || !take(o[3], index, vs) || !k.t || !v.t) return false;
        codes = code_type(k.t->scalar_type());
        if (codes < 0 || v.t->scalar_type() != k.t->scalar_type() || k.t->dim() != 4 || v.t->sizes() != k.t->sizes() || !dense(*k.t) || !dense(*v.t))
            return false;
        const auto s = k.t->sizes();
        pages = s[0], heads = (int)s[1], page = s[2], dim = (int)s[3];
        if (s[1] > 0x7fffffff || s[2] > 0x7fffffff || s[3] > 0x7fffffff) return false;
        if (!codes) return ks.none && vs.none;
        if (!ks.t || !vs.t) return false;
        for (const at::Tensor *t : {ks.t, vs.t})
            if (t->scalar_type() != at::kFloat || t->dim() != 3 || t->size(0) != s[0] || t->size(1) != s[1] || t->size(2) != s[2] || !dense(*t))
                return false;
        return true;
    }
    float *scale(const Arg &a) const { return a.t ? (float *)a.t->data_ptr() : nullptr; }
};

// [tokens, heads, dim] rows that the library takes as they are
bool rows_of_heads(const at::Tensor &t)
{
    return t.dim() == 3 && t.stride(2) == 1 && ((t.stride(0) | t.stride(1)) & 7) == 0 && aligned(t);
}

bool slots_of(const Arg &a) { return a.t && a.t->scalar_type() == at::kLong && a.t->dim() == 1 && a.t->is_contiguous(); }

template <class F>
PyObject *guarded(F &&f)
{
    try {
        return f();
    } catch (const std::exception &) {   // (out of memory, say): the general path meets it and reports it
        return none();
    }
}

// add_rms_norm(x, weight, eps, residual, codes, rot_group, stream) -> (rows, scale, h)
PyObject *norm(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        Arg x, w, r;
        if (n != 7 || !f_norm || !take(o[0], -1, x) || !x.t) return none();
        const int64_t index = x.t->get_device();
        if (!take(o[1], index, w) || !w.t || !take(o[3], index, r)) return none();
        const double eps = PyFloat_AsDouble(o[2]);
        const long codes = PyLong_AsLong(o[4]), rot = PyLong_AsLong(o[5]);
        void *stream = PyLong_AsVoidPtr(o[6]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return none();
        }
        const int dt = half_type(x.t->scalar_type()), wdt = float_type(w.t->scalar_type());
        if (codes < PSQ_CODES_NONE || codes > PSQ_CODES_E4M3 || rot != (int)rot || dt < 0 || wdt < 0 || x.t->dim() != 2 || !dense(*x.t) ||
            !dense(*w.t) || w.t->numel() != x.t->size(1))
            return none();
        if (r.t && (r.t->scalar_type() != x.t->scalar_type() || r.t->sizes() != x.t->sizes() || !dense(*r.t))) return none();
        const int64_t M = x.t->size(0), K = x.t->size(1);
        const auto opt = at::TensorOptions().device(x.t->device());
        const at::ScalarType kind = codes == PSQ_CODES_I8 ? at::kChar : codes == PSQ_CODES_E4M3 ? at::kFloat8_e4m3fn : x.t->scalar_type();
        at::Tensor out, scale, h;
        int status;
        {
            Unlocked unlocked;
            out = at::empty({M, K}, opt.dtype(kind));
            if (codes) scale = at::empty({M}, opt.dtype(at::kFloat));
            if (r.t) h = at::empty({M, K}, opt.dtype(x.t->scalar_type()));
            status = f_norm((int)codes, x.t->data_ptr(), dt, K, r.t ? r.t->data_ptr() : nullptr, K, w.t->data_ptr(), wdt, (float)eps,
                            r.t ? h.data_ptr() : nullptr, K, (int)rot, nullptr, out.data_ptr(), K, codes ? (float *)scale.data_ptr() : nullptr,
                            M, K, stream);
        }
        return status ? none() : tuple(out, scale, h);
    });
}

// kv_write(k, v, slots, k_cache, v_cache, k_scale, v_scale, stream) -> True
PyObject *kv_write(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        Arg k, v, slots;
        Pools p;
        if (n != 8 || !f_write || !take(o[0], -1, k) || !k.t) return none();
        const int64_t index = k.t->get_device();
        if (!take(o[1], index, v) || !v.t || !take(o[2], index, slots) || !slots_of(slots) || !p.take_from(o + 3, index)) return none();
        void *stream = PyLong_AsVoidPtr(o[7]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return none();
        }
        const int dt = half_type(k.t->scalar_type());
        if (dt < 0 || v.t->scalar_type() != k.t->scalar_type() || (!p.codes && p.k.t->scalar_type() != k.t->scalar_type()) || !rows_of_heads(*k.t) ||
            !rows_of_heads(*v.t) || v.t->sizes() != k.t->sizes() || k.t->size(1) != p.heads || k.t->size(2) != p.dim || slots.t->size(0) != k.t->size(0))
            return none();
        int status;
        {
            Unlocked unlocked;
            status = f_write(p.codes, k.t->data_ptr(), v.t->data_ptr(), dt, k.t->stride(0), k.t->stride(1), v.t->stride(0), v.t->stride(1),
                             (const int64_t *)slots.t->data_ptr(), k.t->size(0), p.heads, p.dim, p.k.t->data_ptr(), p.v.t->data_ptr(),
                             p.scale(p.ks), p.scale(p.vs), p.pages, (int)p.page, stream);
        }
        if (status) return none();
        Py_RETURN_TRUE;
    });
}

// kv_read(slots, k_cache, v_cache, k_scale, v_scale, out_type, stream) -> (k, v)
PyObject *kv_read(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        Arg slots;
        Pools p;
        if (n != 7 || !f_read || !take(o[0], -1, slots) || !slots_of(slots) || !p.take_from(o + 1, slots.t->get_device())) return none();
        const long dt = PyLong_AsLong(o[5]);
        void *stream = PyLong_AsVoidPtr(o[6]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return none();
        }
        if (dt != PSQ_BF16 && dt != PSQ_F16 && dt != PSQ_F32) return none();
        const int64_t T = slots.t->size(0);
        const auto opt = at::TensorOptions().device(slots.t->device()).dtype(dt == PSQ_BF16 ? at::kBFloat16 : dt == PSQ_F16 ? at::kHalf : at::kFloat);
        at::Tensor k, v;
        int status;
        {
            Unlocked unlocked;
            k = at::empty({T, p.heads, p.dim}, opt);
            v = at::empty({T, p.heads, p.dim}, opt);
            status = f_read(p.codes, (const int64_t *)slots.t->data_ptr(), T, p.k.t->data_ptr(), p.v.t->data_ptr(),
                            p.codes ? 0 : half_type(p.k.t->scalar_type()), p.scale(p.ks), p.scale(p.vs), p.pages, (int)p.page, p.heads, p.dim,
                            k.data_ptr(), v.data_ptr(), (int)dt, stream);
        }
        return status ? none() : tuple(k, v);
    });
}

// paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scale (None: dim ** -0.5), window,
//                 max_len (None: the table's), return_lse, the stream's workspace, stream) -> out or (out, lse)
// Parts that a second launch joins are in memory of the call's own.
PyObject *attend(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        Arg q, table, lengths, ws;
        Pools p;
        if (n != 13 || !f_attend || !f_attend_bytes || !f_attend_own || !take(o[0], -1, q) || !q.t) return none();
        const int64_t index = q.t->get_device();
        if (!p.take_from(o + 1, index) || !take(o[5], index, table) || !table.t || !take(o[6], index, lengths) || !lengths.t || !take(o[11], index, ws))
            return none();
        const double scale = o[7] == Py_None ? 1 / std::sqrt((double)p.dim) : PyFloat_AsDouble(o[7]);
        const long long window = PyLong_AsLongLong(o[8]);
        long long max_len = o[9] == Py_None ? -1 : PyLong_AsLongLong(o[9]);
        const int want = PyObject_IsTrue(o[10]);
        void *stream = PyLong_AsVoidPtr(o[12]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return none();
        }
        const int dt = half_type(q.t->scalar_type());
        if (dt < 0 || (!p.codes && p.k.t->scalar_type() != q.t->scalar_type()) || !rows_of_heads(*q.t) || q.t->size(2) != p.dim || p.heads <= 0 ||
            q.t->size(1) % p.heads || q.t->size(1) > 0x7fffffff || table.t->scalar_type() != at::kInt || table.t->dim() != 2 ||
            table.t->size(0) != q.t->size(0) || (table.t->size(1) > 1 && table.t->stride(1) != 1) || lengths.t->scalar_type() != at::kInt ||
            lengths.t->dim() != 1 || lengths.t->size(0) != q.t->size(0) || !lengths.t->is_contiguous() || window < 0)
            return none();
        const int64_t B = q.t->size(0), H = q.t->size(1), cols = table.t->size(1);
        if (max_len < 0 || max_len > cols * p.page) max_len = cols * p.page;
        if (window && window < max_len) max_len = window;
        const int64_t need = f_attend_bytes(p.codes, B, (int)H, p.heads, p.dim, max_len);
        const bool own = need > 0 && f_attend_own(p.codes, B, (int)H, p.heads, p.dim, max_len);
        if (need > 0 && !own && (!ws.t || ws.t->numel() < need)) return none();
        const auto opt = at::TensorOptions().device(q.t->device());
        at::Tensor out, lse, parts;
        int status;
        {
            Unlocked unlocked;
            if (own) parts = at::empty({need}, opt.dtype(at::kByte));
            const at::Tensor *work = own ? &parts : ws.t;
            out = at::empty({B, H, p.dim}, opt.dtype(q.t->scalar_type()));
            if (want) lse = at::empty({B, H}, opt.dtype(at::kFloat));
            status = f_attend(p.codes, q.t->data_ptr(), dt, q.t->stride(0), q.t->stride(1), p.k.t->data_ptr(), p.v.t->data_ptr(), p.scale(p.ks),
                              p.scale(p.vs), p.pages, (int)p.page, (const int32_t *)table.t->data_ptr(), table.t->stride(0), cols,
                              (const int32_t *)lengths.t->data_ptr(), B, (int)H, p.heads, p.dim, (float)scale, window, max_len, out.data_ptr(),
                              want ? (float *)lse.data_ptr() : nullptr, need > 0 ? work->data_ptr() : nullptr, need > 0 ? work->numel() : 0,
                              stream);
        }
        return status ? none() : want ? tuple(out, lse) : THPVariable_Wrap(out);
    });
}

// bind({name: address})
PyObject *bind(PyObject *, PyObject *d)
{
    auto at = [&](const char *name) -> void * {
        PyObject *v = PyDict_Check(d) ? PyDict_GetItemString(d, name) : nullptr;
        return v ? PyLong_AsVoidPtr(v) : nullptr;
    };
    f_norm = (decltype(f_norm))at("psq_add_rms_norm");
    f_write = (decltype(f_write))at("psq_kv_write");
    f_read = (decltype(f_read))at("psq_kv_read");
    f_attend_bytes = (decltype(f_attend_bytes))at("psq_paged_attention_workspace_bytes");
    f_attend_own = (decltype(f_attend_own))at("psq_paged_attention_own_workspace");
    f_attend = (decltype(f_attend))at("psq_paged_attention");
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)bind, METH_O, nullptr},
    {"add_rms_norm", (PyCFunction)(void (*)(void))norm, METH_FASTCALL, nullptr},
    {"kv_write", (PyCFunction)(void (*)(void))kv_write, METH_FASTCALL, nullptr},
    {"kv_read", (PyCFunction)(void (*)(void))kv_read, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "psq_direct", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_psq_direct(void)
{
    PyObject *m = PyModule_Create(&module);
    if (m && (PyModule_AddStringConstant(m, "TORCH_VERSION", TORCH_VERSION) < 0 || PyModule_AddIntConstant(m, "PYTHON_VERSION", PY_VERSION_HEX >> 16) < 0))
        Py_CLEAR(m);
    return m;
}
