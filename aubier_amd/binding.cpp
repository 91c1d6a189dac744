// binding.cpp -- the calls of a paged batch's operators from Python, compiled (aubier_amd/_binding.so).
//
// A paged batch's calls run once per step or layer on a handful of small tensors, and the device's time is 3 to 12 us
// each, so what the host adds counts: descriptors straight from the tensors instead of by Python and ctypes, and outputs
// without a trip through Python's argument parser.  The entry points of the kernel library come in as addresses (bind),
// so this module links against none of its copies.  Everything that can be wrong with a call is checked where it
// always is, by the library; a negative status comes back as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mla_m4.h"

namespace {

struct {
    decltype(&mla_m4_pages) pages;
    decltype(&mla_m4_kvrows) kvrows;
    decltype(&mla_m4_kqkv_paged) kqkv_paged;
    decltype(&mla_m4_kqkv_paged_workspace_bytes) workspace_bytes;
    decltype(&mla_m4_norm) norm;
    decltype(&mla_m4_rows_i8) rows_i8;
    decltype(&mla_m4_mul_i8) mul_i8;
    decltype(&mla_m4_qrope) qrope;
    decltype(&mla_m4_mul_i8_workspace_bytes) mul_workspace_bytes;
} lib;

// The descriptors of a call's tensors, all on one GPU
struct Call {
    mla_m4_tensor d[8];
    int n = 0, device = -1, status = 0;

    // the descriptor of a tensor, null for None; where it has none, status says so
    const mla_m4_tensor * add(PyObject * o) { return o == Py_None ? nullptr : add(THPVariable_Unpack(o)); }
    const mla_m4_tensor * add(const at::Tensor & t) {
        int type = 0;
        switch (t.scalar_type()) {
            case at::kFloat: type = MLA_M4_TYPE_F32; break;
            case at::kHalf: type = MLA_M4_TYPE_F16; break;
            case at::kChar: type = MLA_M4_TYPE_I8; break;
            case at::kInt: type = MLA_M4_TYPE_I32; break;
            case at::kLong: type = MLA_M4_TYPE_I64; break;
            default: status = MLA_M4_ERR_TYPE; return nullptr;
        }
        const int64_t dims = t.dim(), es = (int64_t)t.element_size();
        if (dims < 1 || dims > 3) {
            status = MLA_M4_ERR_SHAPE;
            return nullptr;
        }
        mla_m4_tensor & v = next(t, type);
        for (int i = 0; i < 4; ++i) {
            v.ne[i] = i < dims ? t.size(dims - 1 - i) : 1;
            v.nb[i] = i < dims ? (size_t)(t.stride(dims - 1 - i) * es) : v.nb[i - 1] * (size_t)v.ne[i - 1];
        }
        return &v;
    }
    // a cache: block_q8_0 rows of ne0 values, or (ne0 = 0) a tensor
    const mla_m4_tensor * cache(PyObject * o, long ne0) {
        if (ne0 == 0) return add(o);
        const at::Tensor & t = THPVariable_Unpack(o);
        if (t.dim() != 2) {
            status = MLA_M4_ERR_SHAPE;
            return nullptr;
        }
        mla_m4_tensor & v = next(t, MLA_M4_TYPE_Q8_0);
        const int64_t rows = t.size(0), bytes = t.size(1);
        const int64_t ne[4] = {ne0, rows, 1, 1}, nb[4] = {34, bytes, bytes * rows, bytes * rows};
        for (int i = 0; i < 4; ++i) {
            v.ne[i] = ne[i];
            v.nb[i] = (size_t)nb[i];
        }
        return &v;
    }

  private:
    mla_m4_tensor & next(const at::Tensor & t, int type) {
        const int at = t.is_cuda() ? (int)t.get_device() : -1;
        if (at < 0 || (device >= 0 && at != device)) status = MLA_M4_ERR_NULL;
        device = at;
        mla_m4_tensor & v = d[n++];
        v = mla_m4_tensor{};
        v.data = t.data_ptr();
        v.type = type;
        return v;
    }
};

// whether all of n arguments are tensors (or None); else a TypeError is set
bool tensors(PyObject * const * args, int n, bool or_none = false) {
    for (int i = 0; i < n; ++i)
        if (!THPVariable_Check(args[i]) && !(or_none && args[i] == Py_None)) {
            PyErr_SetString(PyExc_TypeError, "a tensor is expected");
            return false;
        }
    return true;
}

// A new tensor where `like` is, as at::empty's: the first by it, the rest straight from the allocator that it took (0.3 us less each,
// without the fill of new memory that torch's deterministic mode may ask for; every call writes all of its results).  Under a dispatch
// mode all come by at::empty: a mode sees them, and what it makes of one (a fake tensor's allocator gives no memory) is not kept.
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Tensor & like) {
    static c10::Allocator * from = nullptr;             // (behind Python's lock)
    const bool modes = c10::impl::TorchDispatchModeTLS::any_modes_set();
    if (from == nullptr || !like.is_cuda() || modes) {
        const at::Tensor t = at::empty(size, at::TensorOptions().dtype(type).device(like.device()));
        if (!modes && t.storage().device().is_cuda()) from = t.storage().allocator();
        return t;
    }
    const c10::DeviceGuard guard(like.device());
    return at::detail::empty_generic(size, from, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, c10::nullopt);
}

at::Tensor given_or_new(PyObject * o, at::IntArrayRef size, at::ScalarType type, const at::Tensor & like) {
    if (o != Py_None) return THPVariable_Unpack(o);
    return fresh(size, type, like);
}

c10::Device gpu(int i) { return c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)i); }

// bind(pages, kvrows, kqkv_paged, workspace_bytes, norm, rows_i8, mul_i8, qrope, mul_workspace_bytes): addresses
PyObject * bind(PyObject *, PyObject * const * args, Py_ssize_t n) {
    if (n != 9) return PyErr_Format(PyExc_TypeError, "nine addresses");
    void * p[9];
    for (int i = 0; i < 9; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
    lib = {(decltype(lib.pages))p[0], (decltype(lib.kvrows))p[1], (decltype(lib.kqkv_paged))p[2], (decltype(lib.workspace_bytes))p[3],
           (decltype(lib.norm))p[4], (decltype(lib.rows_i8))p[5], (decltype(lib.mul_i8))p[6], (decltype(lib.qrope))p[7],
           (decltype(lib.mul_workspace_bytes))p[8]};
    Py_RETURN_NONE;
}

// pages(past, n_new, free, table, page_size, n_rows, slot, pos, used, stream) -> (slot, pos, used)
PyObject * pages(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) return PyErr_Format(PyExc_TypeError, "ten arguments");
    if (!tensors(a, 4) || !tensors(a + 6, 3, true)) return nullptr;
    const long page_size = PyLong_AsLong(a[4]), n_rows = PyLong_AsLong(a[5]);
    void * stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & table = THPVariable_Unpack(a[3]);
    const at::Tensor slot = given_or_new(a[6], {n_rows}, at::kLong, table);
    const at::Tensor pos = given_or_new(a[7], {n_rows}, at::kInt, table);
    const at::Tensor used = given_or_new(a[8], {2}, at::kInt, table);
    Call c;
    const mla_m4_tensor *vp = c.add(a[0]), *vn = c.add(a[1]), *vf = c.add(a[2]), *vt = c.add(table), *vs = c.add(slot), *vo = c.add(pos), *vu = c.add(used);
    if (c.status == 0) {
        const c10::DeviceGuard guard(gpu(c.device));
        c.status = page_size != (int32_t)page_size ? MLA_M4_ERR_ARG : lib.pages(vp, vn, vf, vt, (int32_t)page_size, vs, vo, vu, stream);
    }
    if (c.status != 0) return PyLong_FromLong(c.status);
    PyObject * r = PyTuple_New(3);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(slot));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(pos));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(used));
    return r;
    END_HANDLE_TH_ERRORS
}

// kvrows(x, kv_norm, kcache, ne0, slot, pos, rope, out, stream) -> out; rope: the address of the parameters
PyObject * kvrows(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) return PyErr_Format(PyExc_TypeError, "nine arguments");
    if (!tensors(a, 3) || !tensors(a + 4, 2) || !tensors(a + 7, 1, true)) return nullptr;
    const long ne0 = PyLong_AsLong(a[3]);
    const auto * rope = static_cast<const mla_m4_rope_params *>(PyLong_AsVoidPtr(a[6]));
    void * stream = PyLong_AsVoidPtr(a[8]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & x = THPVariable_Unpack(a[0]);
    const at::Tensor out = given_or_new(a[7], x.sizes(), at::kFloat, x);
    Call c;
    const mla_m4_tensor *vx = c.add(x), *vw = c.add(a[1]), *vk = c.cache(a[2], ne0), *vs = c.add(a[4]), *vo = c.add(a[5]), *vd = c.add(out);
    if (c.status == 0) {
        const c10::DeviceGuard guard(gpu(c.device));
        c.status = lib.kvrows(vx, vw, vk, vs, vo, rope, vd, stream);
    }
    return c.status != 0 ? PyLong_FromLong(c.status) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// kqkv_paged(kcache, ne0, q, past, n_new, table, page_size, kq_scale, prefix, out, d_v, workspace, stream) -> out
PyObject * kqkv_paged(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13) return PyErr_Format(PyExc_TypeError, "thirteen arguments");
    if (!tensors(a, 1) || !tensors(a + 2, 4) || !tensors(a + 8, 2, true) || !tensors(a + 11, 1, true)) return nullptr;
    const long ne0 = PyLong_AsLong(a[1]), page_size = PyLong_AsLong(a[6]), d_v = PyLong_AsLong(a[10]);
    const double scale = PyFloat_AsDouble(a[7]);
    void * stream = PyLong_AsVoidPtr(a[12]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & q = THPVariable_Unpack(a[2]);
    if (q.dim() != 3) return PyLong_FromLong(MLA_M4_ERR_SHAPE);
    const at::Tensor out = given_or_new(a[9], {q.size(1), q.size(0), d_v}, q.scalar_type(), q);
    Call c;
    const mla_m4_tensor *vk = c.cache(a[0], ne0), *vq = c.add(q), *vp = c.add(a[3]), *vn = c.add(a[4]), *vt = c.add(a[5]), *vf = c.add(a[8]), *vo = c.add(out);
    if (c.status != 0) return PyLong_FromLong(c.status);
    const c10::DeviceGuard guard(gpu(c.device));
    at::Tensor work;
    if (a[11] != Py_None) {
        work = THPVariable_Unpack(a[11]);
        if (!work.is_cuda() || (int)work.get_device() != c.device || !work.is_contiguous()) return PyLong_FromLong(MLA_M4_ERR_WORKSPACE);
    } else {
        const size_t need = lib.workspace_bytes(vk, vq, vp, vf, vo);
        if (need > 0) work = fresh({(int64_t)need}, at::kByte, q);
    }
    c.status = page_size != (int32_t)page_size ? MLA_M4_ERR_ARG
        : lib.kqkv_paged(vk, vq, vp, vn, vt, (int32_t)page_size, vf, (float)scale, vo, work.defined() ? work.data_ptr() : nullptr,
                         work.defined() ? (size_t)work.nbytes() : 0, stream);
    return c.status != 0 ? PyLong_FromLong(c.status) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// the type of a float or int8 result by its number, MLA_M4_TYPE_*
at::ScalarType float_or_i8(long type) { return type == MLA_M4_TYPE_F16 ? at::kHalf : type == MLA_M4_TYPE_I8 ? at::kChar : at::kFloat; }

// the results of a call, None for a tensor that is not there
PyObject * results(std::initializer_list<at::Tensor> ts) {
    PyObject * r = PyTuple_New((Py_ssize_t)ts.size());
    if (r == nullptr) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor & t : ts) {
        PyObject * o = Py_None;
        if (t.defined()) o = THPVariable_Wrap(t);
        else Py_INCREF(o);
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

// norm(x, post, gate, res, scale, pre, eps, res_out, out, out_scale, type, stream) -> (res_out, out, out_scale)
PyObject * norm(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12) return PyErr_Format(PyExc_TypeError, "twelve arguments");
    if (!tensors(a, 1) || !tensors(a + 1, 3, true) || !tensors(a + 5, 1, true) || !tensors(a + 7, 3, true)) return nullptr;
    const double scale = PyFloat_AsDouble(a[4]), eps = PyFloat_AsDouble(a[6]);
    const long type = PyLong_AsLong(a[10]);
    void * stream = PyLong_AsVoidPtr(a[11]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & x = THPVariable_Unpack(a[0]);
    if (x.dim() != 2) return PyLong_FromLong(MLA_M4_ERR_SHAPE);
    at::Tensor res_out, out, out_scale;
    if (a[7] != Py_None) res_out = THPVariable_Unpack(a[7]);
    else if (a[3] != Py_None) res_out = fresh(x.sizes(), THPVariable_Unpack(a[3]).scalar_type(), x);
    if (type >= 0 || a[8] != Py_None) out = given_or_new(a[8], x.sizes(), float_or_i8(type), x);
    if (a[9] != Py_None) out_scale = THPVariable_Unpack(a[9]);
    else if (out.defined() && out.scalar_type() == at::kChar) out_scale = fresh({x.size(0)}, at::kFloat, x);
    Call c;
    const mla_m4_tensor *vx = c.add(x), *vp = c.add(a[1]), *vg = c.add(a[2]), *vr = c.add(a[3]), *vw = c.add(a[5]);
    const mla_m4_tensor *vo = res_out.defined() ? c.add(res_out) : nullptr, *vd = out.defined() ? c.add(out) : nullptr;
    const mla_m4_tensor * vs = out_scale.defined() ? c.add(out_scale) : nullptr;
    if (c.status == 0) {
        const c10::DeviceGuard guard(gpu(c.device));
        c.status = lib.norm(vx, vp, vg, vr, (float)scale, vw, (float)eps, vo, vd, vs, stream);
    }
    return c.status != 0 ? PyLong_FromLong(c.status) : results({res_out, out, out_scale});
    END_HANDLE_TH_ERRORS
}

// rows_i8(x, out, scale, stream) -> (out, scale)
PyObject * rows_i8(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) return PyErr_Format(PyExc_TypeError, "four arguments");
    if (!tensors(a, 1) || !tensors(a + 1, 2, true)) return nullptr;
    void * stream = PyLong_AsVoidPtr(a[3]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & x = THPVariable_Unpack(a[0]);
    if (x.dim() != 2 && x.dim() != 3) return PyLong_FromLong(MLA_M4_ERR_SHAPE);
    const at::Tensor out = given_or_new(a[1], {x.size(0), x.dim() == 3 ? x.size(1) * x.size(2) : x.size(1)}, at::kChar, x);
    const at::Tensor scale = given_or_new(a[2], {x.size(0)}, at::kFloat, x);
    Call c;
    const mla_m4_tensor *vx = c.add(x), *vd = c.add(out), *vs = c.add(scale);
    if (c.status == 0) {
        const c10::DeviceGuard guard(gpu(c.device));
        c.status = lib.rows_i8(vx, vd, vs, stream);
    }
    return c.status != 0 ? PyLong_FromLong(c.status) : results({out, scale});
    END_HANDLE_TH_ERRORS
}

// mul_i8(w, w_scale, x, x_scale, out, type, workspace, stream) -> out
PyObject * mul_i8(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) return PyErr_Format(PyExc_TypeError, "eight arguments");
    if (!tensors(a, 4) || !tensors(a + 4, 1, true) || !tensors(a + 6, 1, true)) return nullptr;
    const long type = PyLong_AsLong(a[5]);
    void * stream = PyLong_AsVoidPtr(a[7]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & w = THPVariable_Unpack(a[0]);
    const at::Tensor & x = THPVariable_Unpack(a[2]);
    if (w.dim() != 2 || x.dim() != 2) return PyLong_FromLong(MLA_M4_ERR_SHAPE);
    const at::Tensor out = given_or_new(a[4], {x.size(0), w.size(0)}, float_or_i8(type), x);
    Call c;
    const mla_m4_tensor *vw = c.add(w), *vs = c.add(a[1]), *vx = c.add(x), *vt = c.add(a[3]), *vd = c.add(out);
    if (c.status != 0) return PyLong_FromLong(c.status);
    const c10::DeviceGuard guard(gpu(c.device));
    at::Tensor work;
    if (a[6] != Py_None) {
        work = THPVariable_Unpack(a[6]);
        if (!work.is_cuda() || (int)work.get_device() != c.device || !work.is_contiguous()) return PyLong_FromLong(MLA_M4_ERR_WORKSPACE);
    } else {
        const size_t need = lib.mul_workspace_bytes(vw, vx);
        if (need > 0) work = fresh({(int64_t)need}, at::kByte, x);
    }
    c.status = lib.mul_i8(vw, vs, vx, vt, vd, work.defined() ? work.data_ptr() : nullptr, work.defined() ? (size_t)work.nbytes() : 0, stream);
    return c.status != 0 ? PyLong_FromLong(c.status) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// qrope(q, pos, rope, out, stream) -> out; rope: the address of the parameters
PyObject * qrope(PyObject *, PyObject * const * a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) return PyErr_Format(PyExc_TypeError, "five arguments");
    if (!tensors(a, 2) || !tensors(a + 3, 1, true)) return nullptr;
    const auto * rope = static_cast<const mla_m4_rope_params *>(PyLong_AsVoidPtr(a[2]));
    void * stream = PyLong_AsVoidPtr(a[4]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor & q = THPVariable_Unpack(a[0]);
    const at::Tensor out = given_or_new(a[3], q.sizes(), at::kFloat, q);
    Call c;
    const mla_m4_tensor *vq = c.add(q), *vp = c.add(a[1]), *vd = c.add(out);
    if (c.status == 0) {
        const c10::DeviceGuard guard(gpu(c.device));
        c.status = lib.qrope(vq, vp, rope, vd, stream);
    }
    return c.status != 0 ? PyLong_FromLong(c.status) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void *)bind, METH_FASTCALL, nullptr},
    {"pages", (PyCFunction)(void *)pages, METH_FASTCALL, nullptr},
    {"kvrows", (PyCFunction)(void *)kvrows, METH_FASTCALL, nullptr},
    {"kqkv_paged", (PyCFunction)(void *)kqkv_paged, METH_FASTCALL, nullptr},
    {"norm", (PyCFunction)(void *)norm, METH_FASTCALL, nullptr},
    {"rows_i8", (PyCFunction)(void *)rows_i8, METH_FASTCALL, nullptr},
    {"mul_i8", (PyCFunction)(void *)mul_i8, METH_FASTCALL, nullptr},
    {"qrope", (PyCFunction)(void *)qrope, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
