// Host side of the operators' calls: reads tensors' addresses and layouts, allocates outputs and calls the C ABI of
// libtthrml_b200.so in one pass.  Python needs about 0.4 us per tensor and attribute, 2.3 us per allocation and 2 us per
// ctypes call, which is more than the smallest kernels take.  Each function handles the plain case and returns None for
// any other, which the Python caller then checks, refuses or lays out.
#include "hostcall.h"

namespace {

using hostcall::dtype_code;
using hostcall::plain_cuda;
using hostcall::wants_grad;

// Tells autograd that the tensors of a list were written.
void bump(PyObject* list) {
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) continue;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
}
PyObject* bump_versions(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  if (!PyList_Check(list)) {
    PyErr_SetString(PyExc_TypeError, "bump_versions(tensors): a list");
    return nullptr;
  }
  bump(list);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <typename Fn>
Fn address(PyObject* o) {
  return reinterpret_cast<Fn>(PyLong_AsVoidPtr(o));
}

// What stays the same from step to step of an optimizer (AdamWCall in _native.py).
struct AdamWCall {
  tthrml_adamw_tensor* rows;  // of the parameters that have elements
  int64_t n_rows;
  int64_t state_bits;
  void *exp_avg, *exp_avg_sq;
  float *exp_avg_scale, *exp_avg_sq_scale;
  tthrml_adamw_ctl* ctl;
  double beta1, beta2, eps, weight_decay;
  uint64_t seed;
};
using AdamWFn = decltype(&tthrml_adamw_step);

// adamw_step(params, grads, call, function, stream, device) -> -1 for a step queued, the place of the first pair that is not
// the plain case (the parameter as its row has it, a gradient of its sizes and strides and of its type or float32), or an
// error code less 1000.
PyObject* adamw_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 6 || !PyList_Check(args[0]) || !PyList_Check(args[1]) ||
      PyList_GET_SIZE(args[0]) != PyList_GET_SIZE(args[1])) {
    PyErr_SetString(PyExc_TypeError, "adamw_step(params, grads, call, function, stream, device): two lists of one length");
    return nullptr;
  }
  AdamWCall* call = address<AdamWCall*>(args[2]);
  void* stream = PyLong_AsVoidPtr(args[4]);
  const long device = PyLong_AsLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  Py_ssize_t row = 0;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *po = PyList_GET_ITEM(args[0], i), *go = PyList_GET_ITEM(args[1], i);
    if (!THPVariable_Check(po) || !THPVariable_Check(go)) return PyLong_FromSsize_t(i);
    const at::Tensor &p = THPVariable_Unpack(po), &g = THPVariable_Unpack(go);
    // the same keys: what holds for the parameter's device type and layout holds for the gradient's
    const bool alike = p.key_set() == g.key_set() && p.device() == g.device();
    if (!plain_cuda(p, device) || !(alike || plain_cuda(g, device))) return PyLong_FromSsize_t(i);
    const int32_t pd = dtype_code(p), gd = p.dtype() == g.dtype() ? pd : dtype_code(g);
    if (p.sizes() != g.sizes() || p.strides() != g.strides() || !p.is_non_overlapping_and_dense() ||
        (gd != TTHRML_DT_F32 && gd != pd))
      return PyLong_FromSsize_t(i);
    const int64_t numel = p.numel();
    if (numel == 0) continue;
    if (row >= call->n_rows) return PyLong_FromSsize_t(i);
    tthrml_adamw_tensor& r = call->rows[row++];
    if (r.param != p.data_ptr() || r.n != numel || r.param_dtype != pd) return PyLong_FromSsize_t(i);
    r.grad = g.const_data_ptr();
    r.grad_dtype = gd;
  }
  if (row != call->n_rows) return PyLong_FromSsize_t(n - 1);
  const int rc = address<AdamWFn>(args[3])(call->rows, call->n_rows, (int32_t)call->state_bits, call->exp_avg,
                                           call->exp_avg_sq, call->exp_avg_scale, call->exp_avg_sq_scale, call->ctl,
                                           call->beta1, call->beta2, call->eps, call->weight_decay, call->seed, stream);
  if (rc) return PyLong_FromLong(rc - 1000);
  bump(args[0]);
  return PyLong_FromLong(-1);
  END_HANDLE_TH_ERRORS
}

using AdamWValuesFn = decltype(&tthrml_adamw_values);

// adamw_values(call, codes, elements, function, stream) -> both moments as float32 tensors of `elements` on the codes' device
// (the padded segments, at least one block), or an error code.
PyObject* adamw_values(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5 || !THPVariable_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "adamw_values(call, codes, elements, function, stream)");
    return nullptr;
  }
  const AdamWCall* call = address<const AdamWCall*>(args[0]);
  const int64_t elements = PyLong_AsLongLong(args[2]);
  void* stream = PyLong_AsVoidPtr(args[4]);
  if (PyErr_Occurred()) return nullptr;
  const auto options = THPVariable_Unpack(args[1]).options().dtype(at::kFloat);
  at::Tensor m = at::empty({elements}, options), v = at::empty({elements}, options);
  const int rc = address<AdamWValuesFn>(args[3])(static_cast<const int8_t*>(call->exp_avg),
                                                 static_cast<const uint8_t*>(call->exp_avg_sq), call->exp_avg_scale,
                                                 call->exp_avg_sq_scale, elements, m.mutable_data_ptr<float>(),
                                                 v.mutable_data_ptr<float>(), stream);
  if (rc) return PyLong_FromLong(rc);
  PyObject *a = THPVariable_Wrap(m), *b = THPVariable_Wrap(v);
  PyObject* t = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return t;
  END_HANDLE_TH_ERRORS
}

using LinearFn = decltype(&tthrml_int8_linear);
using MomentsFn = decltype(&tthrml_pair_moments);
using PackedMomentsFn = decltype(&tthrml_pair_moments_packed);

// int8_product(x, weights, weight scales, pitch, bias or None, function, error word, stream, device) -> the product in x's
// type, an error code, or None.
PyObject* int8_product(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) ||
      !(args[4] == Py_None || THPVariable_Check(args[4])))
    Py_RETURN_NONE;
  const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]), &ws = THPVariable_Unpack(args[2]);
  const long device = PyLong_AsLong(args[8]);
  const int64_t pitch = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const int32_t code = dtype_code(x);
  if (!plain_cuda(x, device) || code < 0 || x.dim() < 1 || wants_grad(x) || wants_grad(ws) || (x.dim() != 2 && !x.is_contiguous()))
    Py_RETURN_NONE;
  const int64_t K = x.size(-1), N = w.size(0);
  if (K != w.size(1) || K < 1 || N < 1 || x.numel() == 0) Py_RETURN_NONE;
  const int64_t M = x.numel() / K;
  const float* bias = nullptr;
  if (args[4] != Py_None) {
    const at::Tensor& b = THPVariable_Unpack(args[4]);
    if (!plain_cuda(b, device) || b.scalar_type() != at::kFloat || b.dim() != 1 || b.size(0) != N || !b.is_contiguous() ||
        wants_grad(b))
      Py_RETURN_NONE;
    bias = b.const_data_ptr<float>();
  }
  const int64_t rs = x.dim() == 2 ? x.stride(0) : K, cs = x.dim() == 2 && K > 1 ? x.stride(1) : 1;
  if (cs == 0 || (cs == 1 && M > 1 && rs < K)) Py_RETURN_NONE;
  at::DimVector sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = N;
  at::Tensor out = at::empty(sizes, x.options().requires_grad(false)), space;
  int64_t bytes = 0;
  const int64_t padded = (K + 15) / 16 * 16;
  if (M > 2 || M * padded > TTHRML_INT8_FEW_BYTES || cs != 1) {
    bytes = M * padded + (M * 4 + 15) / 16 * 16;
    space = at::empty({bytes}, x.options().dtype(at::kChar).requires_grad(false));
  }
  const int rc = address<LinearFn>(args[5])(
      x.const_data_ptr(), code, M, K, rs, cs, bytes ? space.mutable_data_ptr() : nullptr, bytes,
      w.const_data_ptr<int8_t>(), pitch, ws.const_data_ptr<float>(), N, bias, out.mutable_data_ptr(), code, N,
      address<int32_t*>(args[6]), PyLong_AsVoidPtr(args[7]));
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// pair_moments(xs, ys, scales, units, function, its form for packed operands, error word, stream, device) -> the moments (with `units` a
// triple), an error code, or None.
PyObject* pair_moments(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9 || !PyList_Check(args[0]) || !PyList_Check(args[1]) || !PyList_Check(args[2])) Py_RETURN_NONE;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  if (n < 1 || n > TTHRML_MAX_PHASES || PyList_GET_SIZE(args[1]) != n || PyList_GET_SIZE(args[2]) != n) Py_RETURN_NONE;
  const bool units = args[3] == Py_True;
  const long device = PyLong_AsLong(args[8]);
  if (PyErr_Occurred()) return nullptr;
  tthrml_moment_phase phases[TTHRML_MAX_PHASES] = {};
  tthrml_pack_matrix packed[TTHRML_MAX_PACKED];
  const void** packed_into[TTHRML_MAX_PACKED];
  int32_t n_packed = 0;
  int64_t M = 0, N = 0, elements = 0;
  int32_t code = -1;
  for (Py_ssize_t p = 0; p < n; ++p) {
    tthrml_moment_phase& ph = phases[p];
    for (int side = 0; side < 2; ++side) {
      PyObject* o = PyList_GET_ITEM(args[side], p);
      if (!THPVariable_Check(o)) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!plain_cuda(t, device) || t.dim() != 2 || wants_grad(t)) Py_RETURN_NONE;
      const int32_t c = dtype_code(t);
      if ((c != TTHRML_DT_BF16 && c != TTHRML_DT_F16) || (code >= 0 && c != code)) Py_RETURN_NONE;
      code = c;
      const int64_t chains = t.size(0), u = t.size(1);
      int64_t& want = side ? N : M;
      if (u < 1 || (p > 0 && u != want) || (side && chains != ph.chains)) Py_RETURN_NONE;
      want = u;
      ph.chains = chains;
      const void*& at = side ? ph.y : ph.x;
      int64_t& ld = side ? ph.y_ld : ph.x_ld;
      ld = chains > 1 ? t.stride(0) : (u + 7) / 8 * 8;
      at = t.const_data_ptr();
      if ((u == 1 || t.stride(1) == 1) && ld % 8 == 0 && ld >= u && reinterpret_cast<uintptr_t>(at) % 16 == 0) continue;
      ld = (u + 7) / 8 * 8;
      packed_into[n_packed] = &at;
      packed[n_packed++] = {at, reinterpret_cast<void*>(elements * 2), chains, u, t.stride(0), t.stride(1), ld};
      elements += chains * ld;
    }
    const double s = PyFloat_AsDouble(PyList_GET_ITEM(args[2], p));
    if (s == -1.0 && PyErr_Occurred()) return nullptr;
    ph.scale = ph.x_scale = ph.y_scale = (float)s;
  }
  void* stream = PyLong_AsVoidPtr(args[7]);
  const at::Tensor& first = THPVariable_Unpack(PyList_GET_ITEM(args[0], 0));
  const auto options = first.options().dtype(at::kFloat).requires_grad(false);
  at::Tensor out = at::empty({M, N}, options), xs, ys, space;
  if (units) {
    xs = at::empty({M}, options);
    ys = at::empty({N}, options);
  }
  int rc = 0;
  if (n_packed) {
    space = at::empty({elements > 0 ? elements : 8}, first.options().requires_grad(false));
    char* base = static_cast<char*>(space.mutable_data_ptr());
    for (int i = 0; i < n_packed; ++i) {
      packed[i].dst = base + reinterpret_cast<uintptr_t>(packed[i].dst);
      *packed_into[i] = packed[i].dst;
    }
  }
  float *o = out.mutable_data_ptr<float>(), *xo = units ? xs.mutable_data_ptr<float>() : nullptr,
        *yo = units ? ys.mutable_data_ptr<float>() : nullptr;
  int32_t* error = address<int32_t*>(args[6]);
  if (n_packed)
    rc = address<PackedMomentsFn>(args[5])(packed, n_packed, phases, (int32_t)n, code, M, N, o, N, xo, yo, 0, error, stream);
  else
    rc = address<MomentsFn>(args[4])(phases, (int32_t)n, code, M, N, o, N, xo, yo, 0, error, stream);
  if (rc) return PyLong_FromLong(rc);
  if (!units) return THPVariable_Wrap(out);
  PyObject *a = THPVariable_Wrap(out), *b = THPVariable_Wrap(xs), *c = THPVariable_Wrap(ys);
  PyObject* t = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  Py_XDECREF(c);
  return t;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"int8_product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(int8_product)), METH_FASTCALL,
     "Product of float rows and 8-bit weights: the plain case, or None."},
    {"pair_moments", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pair_moments)), METH_FASTCALL,
     "Pair moments of lists of phases: the plain case, or None."},
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw_step)), METH_FASTCALL,
     "A step of all parameters: the plain case, or where it is not."},
    {"adamw_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw_values)), METH_FASTCALL,
     "The 8-bit moments as float32."},
    {"bind_library", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::bind_library)), METH_FASTCALL,
     "Takes the addresses of the library's entry points."},
    {"softmax_cross_entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::softmax_cross_entropy)), METH_FASTCALL,
     "Losses of checked tensors, differentiable."},
    {"softmax_cross_entropy_gradients",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::softmax_cross_entropy_gradients)), METH_FASTCALL,
     "The mean loss of checked tensors, its gradients written."},
    {"dropout", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::dropout)), METH_FASTCALL,
     "Kept elements of a checked tensor, differentiable."},
    {"quantize_fp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::quantize_fp4)), METH_FASTCALL,
     "Rows in 4 bits: the plain case, or None."},
    {"fp4_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::fp4_values)), METH_FASTCALL,
     "The float32 values of 4-bit rows."},
    {"fp4_product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(hostcall::fp4_product)), METH_FASTCALL,
     "Product of float rows and 4-bit weights: the plain case, or None."},
    {"bump_versions", bump_versions, METH_O, "Marks tensors as written for autograd."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcall", "Host side of calls with many tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hostcall() { return PyModule_Create(&module); }
