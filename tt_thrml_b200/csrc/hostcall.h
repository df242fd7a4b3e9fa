// What the parts of the host module share.
#pragma once

#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/tthrml.h"

namespace hostcall {

inline int32_t dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TTHRML_DT_F32;
    case at::kBFloat16: return TTHRML_DT_BF16;
    case at::kHalf: return TTHRML_DT_F16;
    default: return -1;
  }
}
inline bool plain_cuda(const at::Tensor& t, long device) {
  return t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && !t.is_neg() && !t.is_conj();
}
// Whether a derivative is asked of t: a gradient, or the tangent of a forward-mode dual tensor.
inline bool wants_grad(const at::Tensor& t) {
  return (c10::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(/*level=*/0).defined();
}

// Entry points of libtthrml_b200.so, in the order of bind_library's arguments (_native.py).
struct Library {
  decltype(&tthrml_set_device) set_device;
  decltype(&tthrml_last_error) last_error;
  decltype(&tthrml_pack_rows) pack_rows;
  decltype(&tthrml_xent_forward) xent_forward;
  decltype(&tthrml_xent_forward_workspace) xent_forward_workspace;
  decltype(&tthrml_xent_backward) xent_backward;
  decltype(&tthrml_xent_backward_workspace) xent_backward_workspace;
  decltype(&tthrml_dropout) dropout;
  decltype(&tthrml_fp4_quantize) fp4_quantize;
  decltype(&tthrml_fp4_scale_bytes) fp4_scale_bytes;
  decltype(&tthrml_fp4_values) fp4_values;
  decltype(&tthrml_fp4_linear) fp4_linear;
  decltype(&tthrml_fp4_linear_workspace) fp4_linear_workspace;
};
extern Library library;

PyObject* bind_library(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* softmax_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* softmax_cross_entropy_gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* dropout(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* quantize_fp4(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* fp4_values(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* fp4_product(PyObject*, PyObject* const* args, Py_ssize_t nargs);

}  // namespace hostcall
