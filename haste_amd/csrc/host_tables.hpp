// What the parts of haste_amd._host share.
#pragma once

#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/haste_ffi.h"

namespace haste_host {

// HASTE_DTYPE_* of a dtype that the kernels take for rows, weights and gradients, or -1.
inline int dtype_code(c10::ScalarType t) {
    return t == c10::kBFloat16 ? HASTE_DTYPE_BF16
           : t == c10::kHalf   ? HASTE_DTYPE_F16
           : t == c10::kFloat  ? HASTE_DTYPE_F32
                               : -1;
}

inline void* stream_of(const at::Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

// Refuses under torch.jit.trace and fx's tracing, whose graph would hold the empty outputs and not
// the kernels that fill them.
inline void check_not_traced(const char* what) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                what, ": cannot be traced (its kernels are called by address)");
}

inline void call(int rc) { TORCH_CHECK(rc == HASTE_OK, haste_last_error()); }

// (a, b) as Python tensors.
inline PyObject* pair_of(const at::Tensor& a, const at::Tensor& b) {
    PyObject *x = THPVariable_Wrap(a), *y = x ? THPVariable_Wrap(b) : nullptr;
    PyObject* pair = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return pair;
}

// layer_norm(x, weight, bias, eps, residual) -> y, or (y, h) with a residual
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t count);

}  // namespace haste_host
