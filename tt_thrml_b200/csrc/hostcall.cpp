// Host side of calls that take many tensors: reads the tensors' addresses and layouts in one pass (Python needs about
// 0.4 us per tensor and attribute).  A CPython module; the kernels stay behind the C ABI of libtthrml_b200.so.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/tthrml.h"

namespace {

int32_t dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TTHRML_DT_F32;
    case at::kBFloat16: return TTHRML_DT_BF16;
    case at::kHalf: return TTHRML_DT_F16;
    default: return -1;
  }
}

bool plain_cuda(const at::Tensor& t, long device) {
  return t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && !t.is_neg() && !t.is_conj();
}

// adamw_rows(params, grads, rows address, number of rows, device) -> -1, or the place of the first pair that is not the
// plain case (the parameter as the row has it, a gradient of its sizes and strides and of its type or float32).  Fills the
// gradients' addresses and types into the rows (tthrml_adamw_tensor), which stand for the parameters with elements.
PyObject* adamw_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 5 || !PyList_Check(args[0]) || !PyList_Check(args[1]) ||
      PyList_GET_SIZE(args[0]) != PyList_GET_SIZE(args[1])) {
    PyErr_SetString(PyExc_TypeError, "adamw_rows(params, grads, rows, n_rows, device): two lists of one length");
    return nullptr;
  }
  auto* rows = reinterpret_cast<tthrml_adamw_tensor*>(PyLong_AsVoidPtr(args[2]));
  const Py_ssize_t n_rows = PyLong_AsSsize_t(args[3]);
  const long device = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  Py_ssize_t row = 0;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *po = PyList_GET_ITEM(args[0], i), *go = PyList_GET_ITEM(args[1], i);
    if (!THPVariable_Check(po) || !THPVariable_Check(go)) return PyLong_FromSsize_t(i);
    const at::Tensor &p = THPVariable_Unpack(po), &g = THPVariable_Unpack(go);
    if (!plain_cuda(p, device) || !plain_cuda(g, device)) return PyLong_FromSsize_t(i);
    const int32_t gd = dtype_code(g);
    if (p.sizes() != g.sizes() || p.strides() != g.strides() || !p.is_non_overlapping_and_dense() ||
        (gd != TTHRML_DT_F32 && gd != dtype_code(p)))
      return PyLong_FromSsize_t(i);
    if (p.numel() == 0) continue;
    if (row >= n_rows) return PyLong_FromSsize_t(i);
    tthrml_adamw_tensor& r = rows[row++];
    if (r.param != p.data_ptr() || r.n != p.numel() || r.param_dtype != dtype_code(p)) return PyLong_FromSsize_t(i);
    r.grad = g.data_ptr();
    r.grad_dtype = gd;
  }
  return PyLong_FromSsize_t(row == n_rows ? -1 : n - 1);
}

// bump_versions(tensors): tells autograd that the tensors were written.
PyObject* bump_versions(PyObject*, PyObject* list) {
  if (!PyList_Check(list)) {
    PyErr_SetString(PyExc_TypeError, "bump_versions(tensors): a list");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) continue;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"adamw_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw_rows)), METH_FASTCALL,
     "Fills gradient addresses into AdamW rows; -1 or the first pair that needs a closer look."},
    {"bump_versions", bump_versions, METH_O, "Marks tensors as written for autograd."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcall", "Host side of calls with many tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hostcall() { return PyModule_Create(&module); }
