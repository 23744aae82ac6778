// What the operators with an autograd node share.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "host_tables.hpp"

namespace haste_host {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// t as rows [N, D] with contiguous columns, `ld` elements apart (0: one row for all), copied only
// where it has no such view.
struct Rows {
    at::Tensor t;
    int64_t ld = 0;
};
inline Rows rows_of(const at::Tensor& x, int64_t D) {
    at::Tensor t = x.is_neg() ? x.resolve_neg() : x;
    if (t.dim() != 2) t = t.reshape({-1, D});
    int64_t ld = t.size(0) > 1 ? t.stride(0) : D;
    if ((t.stride(1) != 1 && D > 1) || (ld < D && ld != 0)) {
        t = t.contiguous();
        ld = D;
    }
    return Rows{t, ld};
}

// t contiguous and with its sign applied, or undefined.
inline at::Tensor dense(const at::Tensor& t) {
    return t.defined() ? (t.is_neg() ? t.resolve_neg() : t).contiguous() : t;
}

inline const void* ptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* out_ptr(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

inline void check_device(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a tensor on a HIP device (MI355X); got a ", t.device(),
                " tensor");
}

// A tensor, or an undefined one for None.
inline at::Tensor tensor_arg(PyObject* o, const char* name, bool optional) {
    if (optional && o == Py_None) return at::Tensor();
    TORCH_CHECK(THPVariable_Check(o), name, " must be a tensor on a HIP device (MI355X); got ",
                Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

// Refuses tangents, also where no gradient is recorded: the kernels are handed addresses, without them.
inline void check_no_tangent(const char* what, std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what,
                                    ": forward-mode derivatives are not supported");
}

// A backward's own checks: a tangent may come with its gradients alone, and a tracer run over it alone.
inline void check_gradients(const char* what, const variable_list& grads) {
    check_not_traced(what);
    for (const at::Tensor& g : grads) check_no_tangent(what, {&g});
}

// A backward's results under create_graph: what is differentiated again says so, and is not taken for a
// constant.
inline void once_differentiable(const char* what, variable_list& out) {
    if (!at::GradMode::is_enabled()) return;
    variable_list marked;
    for (const at::Tensor& t : out)
        if (t.defined()) marked.push_back(t.detach().set_requires_grad(true));
    if (marked.empty()) return;
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + ": its backward cannot be differentiated", (int64_t)marked.size());
    marked = (*error)(std::move(marked));
    size_t k = 0;
    for (at::Tensor& t : out)
        if (t.defined()) t = marked[k++];
}

}  // namespace haste_host
