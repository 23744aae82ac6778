// haste_amd._host, the Python module.  Here: the calls over many tensors, whose tables are made
// without a Python call for each attribute of each tensor.  An AdamW step of 195 tensors with
// 8-bit states reads some 40 attributes of each: 0.9 ms in Python, more than its kernels take.
//
// grad_norm and adamw_step return None where a tensor is not plain (dense, contiguous, not negated,
// no subclass with a dispatch of its own, on the first one's HIP device) or its state does not
// fit: the callers' Python paths then copy, create or refuse.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/haste_ffi.h"
#include "host_tables.hpp"

namespace {

constexpr int64_t kStateBlock = 128;  // elements of an 8-bit state that share a scale

using haste_host::call;
using haste_host::dtype_code;
using haste_host::pair_of;
using haste_host::stream_of;

bool plain(const at::Tensor& t, int64_t* device) {
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() ||
        t.key_set().has(c10::DispatchKey::Python) || !t.is_contiguous())
        return false;
    if (*device < 0) *device = t.get_device();
    return t.get_device() == *device;
}

// An entry of a state, with `n` elements of `type` from a multiple of `align` bytes; nullptr where
// it is anything else.
void* state_tensor(PyObject* state, PyObject* key, at::ScalarType type, int64_t n, unsigned align,
                   int64_t* device) {
    PyObject* o = PyDict_GetItemWithError(state, key);
    if (!o || !THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!plain(t, device) || t.scalar_type() != type || t.numel() != n) return nullptr;
    void* p = t.mutable_data_ptr();
    return reinterpret_cast<uintptr_t>(p) % align ? nullptr : p;
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

// grad_norm(tensors, max_norm) -> (norm, coef)
PyObject* grad_norm(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject* list;
    double max_norm;
    if (!PyArg_ParseTuple(args, "O!d", &PyList_Type, &list, &max_norm)) return nullptr;
    haste_host::check_not_traced("grad_norm");
    const Py_ssize_t n = PyList_GET_SIZE(list);
    std::vector<haste_grad_tensor> rows;
    rows.reserve((size_t)n);
    int64_t device = -1;
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* o = PyList_GET_ITEM(list, i);
        if (!THPVariable_Check(o)) Py_RETURN_NONE;
        const at::Tensor& t = THPVariable_Unpack(o);
        haste_grad_tensor row{};
        row.dtype = dtype_code(t.scalar_type());
        if (!plain(t, &device) || row.dtype < 0) Py_RETURN_NONE;
        row.g = t.const_data_ptr();
        row.n = t.numel();
        rows.push_back(row);
    }
    if (rows.empty()) Py_RETURN_NONE;
    const auto options = at::TensorOptions().device(c10::kCUDA, (c10::DeviceIndex)device);
    const int64_t size = haste_grad_norm_workspace_size((int32_t)n);
    const c10::DeviceGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
    const at::Tensor out = at::empty({2}, options.dtype(at::kFloat));
    const at::Tensor ws = at::empty({size}, options.dtype(at::kByte));
    call(haste_grad_norm(rows.data(), (int32_t)n, max_norm, out.mutable_data_ptr<float>(),
                         ws.mutable_data_ptr(), size, stream_of(out)));
    return pair_of(out.select(0, 0), out.select(0, 1));
    END_HANDLE_TH_ERRORS
}

struct Stepped {
    haste_adamw_tensor row;
    int w, g;
    long long step;
    PyObject* state;
    at::Tensor param;
};

// adamw_step(params, state, bits, lr, beta1, beta2, eps, weight decay, stochastic rounding, seed,
// stream, grad_scale) -> True: steps the params that have a gradient, the first of them with
// random stream `stream`, and moves their counts of steps and versions.
PyObject* adamw_step(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *list, *states, *scale;
    int bits, sr;
    unsigned stream;
    double lr, beta1, beta2, eps, wd;
    unsigned long long seed;
    if (!PyArg_ParseTuple(args, "O!O!idddddpKIO", &PyList_Type, &list, &PyDict_Type, &states, &bits,
                          &lr, &beta1, &beta2, &eps, &wd, &sr, &seed, &stream, &scale))
        return nullptr;
    haste_host::check_not_traced("AdamW.step");
    std::vector<Stepped> all;
    const Py_ssize_t count = PyList_GET_SIZE(list);
    all.reserve((size_t)count);
    int64_t device = -1;
    const bool q8 = bits == 8;
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
        s.row.w = p.mutable_data_ptr();
        s.row.g = grad.const_data_ptr();
        s.row.n = n;
        s.row.stream = stream + (uint32_t)i;
        const at::ScalarType type = q8 ? at::kFloat8_e4m3fn : at::kFloat;
        const int64_t size = q8 ? blocks * kStateBlock : n;
        const unsigned align = q8 ? 8 : 16;
        s.row.m = state_tensor(s.state, keys->m, type, size, align, &device);
        s.row.v = state_tensor(s.state, q8 ? keys->u : keys->v, type, size, align, &device);
        if (q8) {
            s.row.m_scale = static_cast<uint8_t*>(
                state_tensor(s.state, keys->ms, at::kFloat8_e8m0fnu, blocks, 1, &device));
            s.row.v_scale = static_cast<uint8_t*>(
                state_tensor(s.state, keys->us, at::kFloat8_e8m0fnu, blocks, 1, &device));
        }
        if (PyErr_Occurred()) return nullptr;
        if (n > 0 && (!s.row.m || !s.row.v || (q8 && (!s.row.m_scale || !s.row.v_scale))))
            Py_RETURN_NONE;
        s.param = p;
        all.push_back(std::move(s));
    }
    const float* factor = nullptr;
    if (scale != Py_None && !all.empty()) {
        if (!THPVariable_Check(scale)) Py_RETURN_NONE;
        const at::Tensor& t = THPVariable_Unpack(scale);
        if (!plain(t, &device) || t.scalar_type() != at::kFloat || t.numel() != 1) Py_RETURN_NONE;
        factor = t.const_data_ptr<float>();
    }
    if (all.empty()) Py_RETURN_TRUE;
    const c10::DeviceGuard guard(all[0].param.device());
    struct Group {
        int w, g;
        long long step;
        std::vector<haste_adamw_tensor> rows;
        std::vector<const Stepped*> stepped;
    };
    std::vector<Group> groups;
    for (const Stepped& s : all) {
        Group* at = nullptr;
        for (Group& g : groups)
            if (g.w == s.w && g.g == s.g && g.step == s.step) at = &g;
        if (!at) {
            groups.push_back(Group{s.w, s.g, s.step, {}, {}});
            at = &groups.back();
            at->rows.reserve(all.size());
            at->stepped.reserve(all.size());
        }
        at->rows.push_back(s.row);
        at->stepped.push_back(&s);
    }
    for (const Group& g : groups) {
        call(haste_adamw_step(g.rows.data(), (int32_t)g.rows.size(), g.w, g.g, bits, lr, beta1, beta2,
                              eps, wd, g.step, sr, seed, factor, stream_of(all[0].param)));
        // (only now: a refused step leaves the counts as they were)
        PyObject* step = PyLong_FromLongLong(g.step);
        if (!step) return nullptr;
        for (const Stepped* s : g.stepped) {
            s->param.unsafeGetTensorImpl()->bump_version();
            if (PyDict_SetItem(s->state, keys->step, step) != 0) {
                Py_DECREF(step);
                return nullptr;
            }
        }
        Py_DECREF(step);
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"grad_norm", grad_norm, METH_VARARGS, "grad_norm(tensors, max_norm) -> (norm, coef) or None"},
    {"adamw_step", adamw_step, METH_VARARGS,
     "adamw_step(params, state, bits, lr, beta1, beta2, eps, weight_decay, stochastic_rounding, "
     "seed, stream, grad_scale) -> True or None"},
    {"layer_norm", fast(haste_host::layer_norm), METH_FASTCALL,
     "layer_norm(x, weight, bias, eps, residual) -> y, or (y, h) with a residual"},
    {"embedding", fast(haste_host::embedding), METH_FASTCALL,
     "embedding(tokens, weight, scale, padding_idx) -> y"},
    {"gated_mlp", fast(haste_host::gated_mlp), METH_FASTCALL,
     "gated_mlp(x, w_gate, w_up, w_down, activation) -> y"},
    {"label_log_probs", fast(haste_host::label_log_probs), METH_FASTCALL,
     "label_log_probs(logits, labels, top) -> (log_probs, entropy, top_log_probs, top_labels)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT,
                      "_host",
                      "Entry points of libhaste_ffi.so that take torch tensors.",
                      -1,
                      methods,
                      nullptr,
                      nullptr,
                      nullptr,
                      nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    static Keys k;
    keys = &k;
    return PyModule_Create(&module);
}
