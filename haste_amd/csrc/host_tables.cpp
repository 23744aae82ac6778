// haste_amd._host, the Python module.  Here: tables of many tensors for the C ABI, made without a
// Python call for each attribute of each tensor.  An AdamW step of 195 tensors with 8-bit states reads some 40
// attributes of each: 0.9 ms in Python, more than its kernels take.
//
// grad_rows and adamw_rows return None where a tensor is not plain (dense, contiguous, not negated, no
// subclass with a dispatch of its own, on the first one's HIP device) or its state does not
// fit: the callers' Python paths then copy, create or refuse.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <vector>

#include "../../include/haste_ffi.h"
#include "host_tables.hpp"

namespace {

constexpr int64_t kStateBlock = 128;  // elements of an 8-bit state that share a scale

using haste_host::dtype_code;

bool plain(const at::Tensor& t, int64_t* device) {
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() ||
        t.key_set().has(c10::DispatchKey::Python) || !t.is_contiguous())
        return false;
    if (*device < 0) *device = t.get_device();
    return t.get_device() == *device;
}

// An entry of a state, with `n` elements of `type`; nullptr where it is anything else.
void* state_tensor(PyObject* state, PyObject* key, at::ScalarType type, int64_t n,
                   int64_t* device) {
    PyObject* o = PyDict_GetItemWithError(state, key);
    if (!o || !THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!plain(t, device) || t.scalar_type() != type || t.numel() != n) return nullptr;
    return t.data_ptr();
}

struct Keys {
    PyObject *step = PyUnicode_InternFromString("step"),
             *m = PyUnicode_InternFromString("exp_avg"),
             *v = PyUnicode_InternFromString("exp_avg_sq"),
             *u = PyUnicode_InternFromString("rms"),
             *ms = PyUnicode_InternFromString("exp_avg_scale"),
             *us = PyUnicode_InternFromString("rms_scale");
};
Keys* keys = nullptr;

PyObject* none_or_error() {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// grad_rows(tensors) -> (haste_grad_tensor[] as bytes, device)
PyObject* grad_rows(PyObject*, PyObject* list) {
    if (!PyList_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "grad_rows: a list is expected");
        return nullptr;
    }
    try {
        const Py_ssize_t n = PyList_GET_SIZE(list);
        std::vector<haste_grad_tensor> rows;
        rows.reserve((size_t)n);
        int64_t device = -1;
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o)) Py_RETURN_NONE;
            const at::Tensor& t = THPVariable_Unpack(o);
            if (!plain(t, &device)) Py_RETURN_NONE;
            const int code = dtype_code(t.scalar_type());
            if (code < 0) Py_RETURN_NONE;
            haste_grad_tensor row{};
            row.g = t.const_data_ptr();
            row.n = t.numel();
            row.dtype = code;
            rows.push_back(row);
        }
        return Py_BuildValue("(y#L)", reinterpret_cast<const char*>(rows.data()),
                             (Py_ssize_t)(rows.size() * sizeof(rows[0])), (long long)device);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

struct Stepped {
    haste_adamw_tensor row;
    int w, g;
    long long step;
    PyObject* state;
    at::Tensor param;
};

// adamw_rows(params, state, bits) -> ([(w dtype, g dtype, step, tensors, haste_adamw_tensor[] as
// bytes)], device) for the params that have a gradient, whose counts of steps and versions it
// moves.
PyObject* adamw_rows(PyObject*, PyObject* args) {
    PyObject *list, *states;
    int bits;
    if (!PyArg_ParseTuple(args, "O!O!i", &PyList_Type, &list, &PyDict_Type, &states, &bits))
        return nullptr;
    try {
        std::vector<Stepped> all;
        const Py_ssize_t count = PyList_GET_SIZE(list);
        all.reserve((size_t)count);
        int64_t device = -1;
        for (Py_ssize_t i = 0; i < count; ++i) {
            PyObject* o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o)) Py_RETURN_NONE;
            const at::Tensor& p = THPVariable_Unpack(o);
            const at::Tensor& grad = p.grad();
            if (!grad.defined()) continue;
            const int64_t n = p.numel(), blocks = (n + kStateBlock - 1) / kStateBlock;
            if (!plain(p, &device) || !plain(grad, &device) || grad.numel() != n) Py_RETURN_NONE;
            Stepped s{};
            s.w = dtype_code(p.scalar_type());
            s.g = dtype_code(grad.scalar_type());
            s.state = PyDict_GetItemWithError(states, o);
            if (s.w < 0 || s.g < 0 || !s.state || !PyDict_Check(s.state)) return none_or_error();
            PyObject* step = PyDict_GetItemWithError(s.state, keys->step);
            if (!step || !PyLong_Check(step)) return none_or_error();
            s.step = PyLong_AsLongLong(step) + 1;
            s.row.w = p.data_ptr();
            s.row.g = grad.const_data_ptr();
            s.row.n = n;
            s.row.stream = (uint32_t)i;
            const bool q8 = bits == 8;
            s.row.m = state_tensor(s.state, keys->m, q8 ? at::kFloat8_e4m3fn : at::kFloat,
                                   q8 ? blocks * kStateBlock : n, &device);
            s.row.v = state_tensor(s.state, q8 ? keys->u : keys->v,
                                   q8 ? at::kFloat8_e4m3fn : at::kFloat,
                                   q8 ? blocks * kStateBlock : n, &device);
            if (q8) {
                s.row.m_scale = static_cast<uint8_t*>(
                    state_tensor(s.state, keys->ms, at::kFloat8_e8m0fnu, blocks, &device));
                s.row.v_scale = static_cast<uint8_t*>(
                    state_tensor(s.state, keys->us, at::kFloat8_e8m0fnu, blocks, &device));
            }
            if (PyErr_Occurred()) return nullptr;
            if (n > 0 && (!s.row.m || !s.row.v || (q8 && (!s.row.m_scale || !s.row.v_scale))))
                Py_RETURN_NONE;
            s.param = p;
            all.push_back(std::move(s));
        }
        struct Group {
            int w, g;
            long long step;
            std::vector<haste_adamw_tensor> rows;
        };
        std::vector<Group> groups;
        for (Stepped& s : all) {
            PyObject* step = PyLong_FromLongLong(s.step);
            if (!step || PyDict_SetItem(s.state, keys->step, step) != 0) {
                Py_XDECREF(step);
                return nullptr;
            }
            Py_DECREF(step);
            s.param.unsafeGetTensorImpl()->bump_version();
            Group* at = nullptr;
            for (Group& g : groups)
                if (g.w == s.w && g.g == s.g && g.step == s.step) at = &g;
            if (!at) {
                groups.push_back(Group{s.w, s.g, s.step, {}});
                at = &groups.back();
                at->rows.reserve(all.size());
            }
            at->rows.push_back(s.row);
        }
        PyObject* out = PyList_New((Py_ssize_t)groups.size());
        for (size_t k = 0; out && k < groups.size(); ++k) {
            const Group& g = groups[k];
            PyObject* item =
                Py_BuildValue("(iiLny#)", g.w, g.g, g.step, (Py_ssize_t)g.rows.size(),
                              reinterpret_cast<const char*>(g.rows.data()),
                              (Py_ssize_t)(g.rows.size() * sizeof(g.rows[0])));
            if (!item) {
                Py_DECREF(out);
                return nullptr;
            }
            PyList_SET_ITEM(out, (Py_ssize_t)k, item);
        }
        return out ? Py_BuildValue("(NL)", out, (long long)device) : nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"grad_rows", grad_rows, METH_O, "grad_rows(tensors) -> (rows, device) or None"},
    {"adamw_rows", adamw_rows, METH_VARARGS,
     "adamw_rows(params, state, bits) -> ([(w, g, step, count, rows)], device) or None"},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(haste_host::layer_norm)),
     METH_FASTCALL, "layer_norm(x, weight, bias, eps, residual) -> y, or (y, h) with a residual"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host side of libhaste_ffi.so's entry points that take torch tensors.", -1,
                      methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    static Keys k;
    keys = &k;
    return PyModule_Create(&module);
}
