// What the parts of haste_amd._host share.
#pragma once

#include <Python.h>

#include <c10/core/ScalarType.h>

#include "../../include/haste_ffi.h"

namespace haste_host {

// HASTE_DTYPE_* of a dtype that the kernels take for rows, weights and gradients, or -1.
inline int dtype_code(c10::ScalarType t) {
    return t == c10::kBFloat16 ? HASTE_DTYPE_BF16
           : t == c10::kHalf   ? HASTE_DTYPE_F16
           : t == c10::kFloat  ? HASTE_DTYPE_F32
                               : -1;
}

// layer_norm(x, weight, bias, eps, residual) -> y, or (y, h) with a residual
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t count);

}  // namespace haste_host
