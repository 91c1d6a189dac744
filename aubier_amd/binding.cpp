// binding.cpp -- the paged operators' calls from Python, compiled (aubier_amd/_binding.so).
//
// A paged batch's calls run once per step or layer on a handful of small tensors, and the device's time is 3 to 12 us
// each, so what the host adds counts: descriptors straight from the tensors instead of by Python and ctypes, and outputs
// without a trip through Python's argument parser.  The entry points of the kernel library come in as addresses (bind),
// so this module links against none of its copies.  Everything that can be wrong with a call is checked where it
// always is, by the library; a negative status comes back as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mla_m4.h"

namespace {

struct {
    decltype(&mla_m4_pages) pages;
    decltype(&mla_m4_kvrows) kvrows;
    decltype(&mla_m4_kqkv_paged) kqkv_paged;
    decltype(&mla_m4_kqkv_paged_workspace_bytes) workspace_bytes;
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

at::Tensor given_or_new(PyObject * o, at::IntArrayRef size, at::ScalarType type, const at::Tensor & like) {
    if (o != Py_None) return THPVariable_Unpack(o);
    return at::empty(size, at::TensorOptions().dtype(type).device(like.device()));
}

c10::Device gpu(int i) { return c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)i); }

// bind(pages, kvrows, kqkv_paged, workspace_bytes): addresses
PyObject * bind(PyObject *, PyObject * const * args, Py_ssize_t n) {
    if (n != 4) return PyErr_Format(PyExc_TypeError, "four addresses");
    void * p[4];
    for (int i = 0; i < 4; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
    lib = {(decltype(lib.pages))p[0], (decltype(lib.kvrows))p[1], (decltype(lib.kqkv_paged))p[2], (decltype(lib.workspace_bytes))p[3]};
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
        if (need > 0) work = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(q.device()));
    }
    c.status = page_size != (int32_t)page_size ? MLA_M4_ERR_ARG
        : lib.kqkv_paged(vk, vq, vp, vn, vt, (int32_t)page_size, vf, (float)scale, vo, work.defined() ? work.data_ptr() : nullptr,
                         work.defined() ? (size_t)work.nbytes() : 0, stream);
    return c.status != 0 ? PyLong_FromLong(c.status) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void *)bind, METH_FASTCALL, nullptr},
    {"pages", (PyCFunction)(void *)pages, METH_FASTCALL, nullptr},
    {"kvrows", (PyCFunction)(void *)kvrows, METH_FASTCALL, nullptr},
    {"kqkv_paged", (PyCFunction)(void *)kqkv_paged, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
