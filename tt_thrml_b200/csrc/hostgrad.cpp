// Host side of the operators that autograd differentiates, and of the 4-bit rows: one node of the graph each, written in
// C++ (a Python one costs 30 us forward and 40 backward, more than the smallest kernels take).  Python checks the arguments
// of the differentiable operators before the call; the 4-bit calls handle the plain case and return None for any other.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>

#include "hostcall.h"

namespace hostcall {

Library library = {};

PyObject* bind_library(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  constexpr Py_ssize_t n = sizeof(Library) / sizeof(void*);
  if (nargs != n) {
    PyErr_Format(PyExc_TypeError, "bind_library: %zd addresses expected, got %zd", n, nargs);
    return nullptr;
  }
  void* at[n];
  for (Py_ssize_t i = 0; i < n; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  memcpy(&library, at, sizeof(Library));
  Py_RETURN_NONE;
}

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

void check(int rc, const char* what) { TORCH_CHECK(rc == TTHRML_OK, what, " failed (", rc, "): ", library.last_error()); }

// Makes a tensor's device current for torch and for the library on this thread (a backward pass has a thread of its own), and
// the old one again at the end.
class On {
 public:
  explicit On(const Tensor& t) : guard_(t.device()), before_(guard_.original_device().index()), now_(t.device().index()) {
    check(library.set_device(now_), "tthrml_set_device");
  }
  ~On() {
    if (before_ != now_) library.set_device(before_);
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(now_).stream(); }

 private:
  c10::cuda::CUDAGuard guard_;
  c10::DeviceIndex before_, now_;
};

Tensor floats(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kFloat).requires_grad(false)); }
Tensor bytes(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }

// The operands as the kernels read them: rows of 16-byte multiples from 16-byte boundaries, as they lie or in a copy of their own.
struct Operand {
  const void* at;
  int64_t ld;
};
bool as_it_lies(const Tensor& t, Operand& o) {
  const int64_t rows = t.size(0), cols = t.size(1);
  o.at = t.const_data_ptr();
  o.ld = rows > 1 ? t.stride(0) : (cols + 7) / 8 * 8;
  return (cols == 1 || t.stride(1) == 1) && o.ld % 8 == 0 && o.ld >= cols && reinterpret_cast<uintptr_t>(o.at) % 16 == 0;
}
// laid[i]: the copy that was made of t[i], [rows, pitch], or undefined.
void lay_out(const Tensor* const (&t)[2], Operand (&o)[2], Tensor (&laid)[2], void* stream) {
  tthrml_pack_matrix m[2];
  int n = 0;
  for (int i = 0; i < 2; ++i) {
    if (as_it_lies(*t[i], o[i])) continue;
    const int64_t rows = t[i]->size(0), cols = t[i]->size(1), ld = (cols + 7) / 8 * 8;
    laid[i] = at::empty({rows, ld}, t[i]->options().requires_grad(false));
    m[n++] = {o[i].at, laid[i].mutable_data_ptr(), rows, cols, t[i]->stride(0), t[i]->stride(1), ld};
    o[i] = {laid[i].const_data_ptr(), ld};
  }
  if (n) check(library.pack_rows(m, n, stream), "tthrml_pack_rows");
}

struct XentSaved {
  Tensor laid[2], sums, inv_count;
};

tthrml_xent problem(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& targets, int64_t ignored, const Operand (&o)[2]) {
  tthrml_xent p = {};
  p.x = o[0].at, p.x_ld = o[0].ld;
  p.w = o[1].at, p.w_ld = o[1].ld;
  p.targets = targets.const_data_ptr();
  p.bias = bias.defined() ? bias.const_data_ptr<float>() : nullptr;
  p.rows = x.size(0), p.cols = x.size(1), p.categories = w.size(0);
  p.ignored = ignored;
  p.dtype = dtype_code(x);
  p.wide_targets = targets.scalar_type() == at::kLong;
  return p;
}

constexpr const char* kRestored = "a saved tensor came back on another device, in another type or of another size";
void restored(const Tensor& t, const Tensor& x, at::ScalarType type, int64_t numel) {
  TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.device() == x.device() && t.scalar_type() == type && t.numel() == numel &&
                  !t.is_neg(),
              kRestored);
}

// bias and targets dense.
Tensor xent_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& targets, int64_t reduction, int64_t ignored,
                    int64_t error, XentSaved& saved) {
  const On on(x);
  const Tensor* const operands[2] = {&x, &w};
  Operand o[2];
  lay_out(operands, o, saved.laid, on.stream());
  const tthrml_xent p = problem(x, w, bias, targets, ignored, o);
  const int64_t size = library.xent_forward_workspace(p.rows, p.categories, p.cols);
  if (size < 0) check((int)size, "tthrml_xent_forward_workspace");
  const Tensor space = bytes(x, size);
  saved.sums = floats(x, {p.rows, 2});
  Tensor rows = floats(x, {p.rows}), total;
  if (reduction) {
    total = floats(x, {});
    saved.inv_count = floats(x, {});
  }
  check(library.xent_forward(&p, saved.sums.mutable_data_ptr<float>(), rows.mutable_data_ptr<float>(),
                             reduction ? total.mutable_data_ptr<float>() : nullptr,
                             reduction ? saved.inv_count.mutable_data_ptr<float>() : nullptr, (int32_t)reduction,
                             space.mutable_data_ptr(), size, reinterpret_cast<int32_t*>(error), on.stream()),
        "tthrml_xent_forward");
  return reduction ? total : rows;
}

// Gradients into dx and dw (one type, dense rows) and db, each may be undefined.
void xent_backward(const Tensor& x, const tthrml_xent& p, const Tensor& sums, const Tensor& grad, const Tensor& inv_count,
                   const Tensor& dx, const Tensor& dw, const Tensor& db, int64_t error, void* stream) {
  const int64_t size = library.xent_backward_workspace(p.rows, p.categories, p.cols, dx.defined(), dw.defined(), db.defined());
  if (size < 0) check((int)size, "tthrml_xent_backward_workspace");
  const Tensor space = bytes(x, size);
  check(library.xent_backward(&p, sums.const_data_ptr<float>(), grad.const_data_ptr<float>(), grad.dim() ? 1 : 0,
                              inv_count.defined() ? inv_count.const_data_ptr<float>() : nullptr,
                              dx.defined() ? dx.mutable_data_ptr() : nullptr, p.cols, dw.defined() ? dw.mutable_data_ptr() : nullptr,
                              p.cols, dx.defined() ? dtype_code(dx) : (dw.defined() ? dtype_code(dw) : p.dtype),
                              db.defined() ? db.mutable_data_ptr<float>() : nullptr, space.mutable_data_ptr(), size,
                              reinterpret_cast<int32_t*>(error), stream),
        "tthrml_xent_backward");
}

struct SoftmaxCrossEntropy : Function<SoftmaxCrossEntropy> {
  // every argument of a node is a defined tensor: without a bias the targets stand in its place
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& bias_or_targets, const Tensor& targets,
                        bool with_bias, int64_t reduction, int64_t ignored, int64_t error) {
    XentSaved s;
    const Tensor bias = with_bias ? bias_or_targets : Tensor();
    Tensor loss = xent_forward(x, w, bias, targets, reduction, ignored, error, s);
    // the tensors themselves, so that a change in place before the backward pass is noticed, beside their copies
    ctx->save_for_backward({x, w, bias, targets, s.laid[0], s.laid[1], s.sums, s.inv_count});
    ctx->saved_data["ignored"] = ignored;
    ctx->saved_data["error"] = error;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), "softmax_cross_entropy has no second derivative (create_graph=True)");
    variable_list s = ctx->get_saved_variables(), out(8);
    if (!grads[0].defined()) return out;
    // a hook on saved tensors may have given them back elsewhere and with other strides
    const Tensor &x = s[0], &w = s[1], &bias = s[2], &targets = s[3], &sums = s[6], &inv_count = s[7];
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && w.dim() == 2 && x.numel() && w.numel(), kRestored);
    const int64_t rows = x.size(0), K = x.size(1), V = w.size(0);
    const bool wide = targets.scalar_type() == at::kLong;
    restored(x, x, dtype_code(x) == TTHRML_DT_F16 ? at::kHalf : at::kBFloat16, rows * K);
    restored(w, x, x.scalar_type(), V * K);
    restored(s[3], x, wide ? at::kLong : at::kInt, rows);
    restored(s[6], x, at::kFloat, 2 * rows);
    if (bias.defined()) restored(s[2], x, at::kFloat, V);
    if (inv_count.defined()) restored(s[7], x, at::kFloat, 1);
    for (int i : {2, 3, 6, 7})
      if (s[i].defined()) s[i] = s[i].contiguous();
    const On on(x);
    Operand o[2];
    const Tensor* operands[2] = {&x, &w};
    Tensor again[2];
    for (int i = 0; i < 2; ++i) {  // the forward pass's copies where it made them; what does not lie as it has to now is copied here
      const Tensor& laid = s[4 + i];
      if (!laid.defined()) continue;
      TORCH_CHECK(laid.dim() == 2 && laid.size(0) == s[i].size(0) && laid.size(1) >= K, kRestored);
      restored(laid, x, x.scalar_type(), laid.numel());
      operands[i] = &laid;
    }
    lay_out({operands[0], operands[1]}, o, again, on.stream());
    const tthrml_xent p = problem(x, w, bias, targets, ctx->saved_data["ignored"].toInt(), o);
    const Tensor grad = grads[0].to(at::kFloat).resolve_neg().contiguous();
    TORCH_CHECK(grad.device() == x.device() && grad.dim() <= 1 && grad.numel() == (inv_count.defined() ? 1 : rows),
                "softmax_cross_entropy: the loss' gradient has another device or shape than the loss");
    if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options().requires_grad(false));
    if (ctx->needs_input_grad(1)) out[1] = at::empty(w.sizes(), w.options().requires_grad(false));
    if (bias.defined() && ctx->needs_input_grad(2)) out[2] = floats(x, bias.sizes());
    xent_backward(x, p, sums, grad, inv_count, out[0], out[1], out[2], ctx->saved_data["error"].toInt(), on.stream());
    return out;
  }
};

Tensor drop(const Tensor& x, int64_t cut, int64_t seed, int64_t step, const Tensor& step_at, const Tensor& used) {
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  if (!x.numel()) return y;
  const On on(x);
  const Tensor in = x.resolve_neg().contiguous();
  check(library.dropout(in.const_data_ptr(), dtype_code(x), in.numel(), (int32_t)cut, (uint64_t)seed, (uint32_t)step,
                        step_at.defined() ? step_at.const_data_ptr() : nullptr,
                        step_at.defined() && step_at.scalar_type() == at::kLong,
                        used.defined() ? static_cast<uint32_t*>(used.mutable_data_ptr()) : nullptr, y.mutable_data_ptr(),
                        on.stream()),
        "tthrml_dropout");
  return y;
}

struct Dropout : Function<Dropout> {
  // step_at: a pointer, so that it is no argument of the node; it may be undefined
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor* step_at, int64_t cut, int64_t seed, int64_t step) {
    // a step on the device may have moved on by the time of the backward pass: the kernel leaves what it used
    Tensor used;
    if (step_at->defined() && x.numel()) used = at::empty({1}, x.options().dtype(at::kInt).requires_grad(false));
    ctx->save_for_backward({used});
    ctx->saved_data["cut"] = cut;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["step"] = step;
    return drop(x, cut, seed, step, *step_at, used);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    if (s[0].defined()) restored(s[0], grads[0], at::kInt, 1);
    const int64_t cut = ctx->saved_data["cut"].toInt(), seed = ctx->saved_data["seed"].toInt(), step = ctx->saved_data["step"].toInt();
    // a node of its own only where this pass is differentiated in turn
    out[0] = c10::GradMode::is_enabled() ? apply(grads[0], &s[0], cut, seed, step) : drop(grads[0], cut, seed, step, s[0], Tensor());
    return out;
  }
};

// The tensor, its values in memory (not those of a negated view); undefined for None.
Tensor tensor_or_none(PyObject* o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o).resolve_neg(); }

}  // namespace

// softmax_cross_entropy(x, weights, bias or None, targets, reduction, ignored, error word) -> the loss; x, weights and targets
// as checked by the caller (two, two and one dimensions).
PyObject* softmax_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7) {
    PyErr_SetString(PyExc_TypeError, "softmax_cross_entropy(x, weights, bias, targets, reduction, ignored, error)");
    return nullptr;
  }
  const Tensor x = tensor_or_none(args[0]), w = tensor_or_none(args[1]);
  Tensor bias = tensor_or_none(args[2]);
  const int64_t reduction = PyLong_AsLongLong(args[4]), ignored = PyLong_AsLongLong(args[5]), error = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  if (bias.defined()) bias = bias.contiguous();
  const Tensor targets = tensor_or_none(args[3]).contiguous();
  if (wants_grad(x) || wants_grad(w) || (bias.defined() && wants_grad(bias)))
    return THPVariable_Wrap(SoftmaxCrossEntropy::apply(x, w, bias.defined() ? bias : targets, targets, bias.defined(), reduction,
                                                       ignored, error));
  XentSaved s;
  return THPVariable_Wrap(xent_forward(x, w, bias, targets, reduction, ignored, error, s));
  END_HANDLE_TH_ERRORS
}

// softmax_cross_entropy_gradients(x, weights, bias, targets, ignored, error word, one, dw, db) -> the mean loss, with its
// gradients in dw (float32 or the weights' type, dense) and db; no node of a graph.  one: the float32 number 1 on the device.
PyObject* softmax_cross_entropy_gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9) {
    PyErr_SetString(PyExc_TypeError, "softmax_cross_entropy_gradients(x, weights, bias, targets, ignored, error, one, dw, db)");
    return nullptr;
  }
  const Tensor x = tensor_or_none(args[0]);
  const Tensor &w = THPVariable_Unpack(args[1]), &bias = THPVariable_Unpack(args[2]);
  const Tensor targets = tensor_or_none(args[3]).contiguous();
  const int64_t ignored = PyLong_AsLongLong(args[4]), error = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor &unit = THPVariable_Unpack(args[6]), &dw = THPVariable_Unpack(args[7]), &db = THPVariable_Unpack(args[8]);
  const On on(x);
  XentSaved s;
  Tensor loss = xent_forward(x, w, bias, targets, 1, ignored, error, s);
  const Tensor* const operands[2] = {s.laid[0].defined() ? &s.laid[0] : &x, s.laid[1].defined() ? &s.laid[1] : &w};
  Operand o[2];
  for (int i = 0; i < 2; ++i) as_it_lies(*operands[i], o[i]);
  xent_backward(x, problem(x, w, bias, targets, ignored, o), s.sums, unit, s.inv_count, Tensor(), dw, db, error, on.stream());
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// dropout(x, cut, seed, step, step tensor or None) -> the kept elements, scaled.
PyObject* dropout(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "dropout(x, cut, seed, step, step_at)");
    return nullptr;
  }
  const Tensor& x = THPVariable_Unpack(args[0]);
  const int64_t cut = PyLong_AsLongLong(args[1]), seed = (int64_t)PyLong_AsUnsignedLongLongMask(args[2]),
                step = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor step_at = tensor_or_none(args[4]);
  if (wants_grad(x)) return THPVariable_Wrap(Dropout::apply(x, &step_at, cut, seed, step));
  return THPVariable_Wrap(drop(x, cut, seed, step, step_at, Tensor()));
  END_HANDLE_TH_ERRORS
}

// quantize_fp4(x, stream, device) -> (codes [rows, pitch], block scales, scales), an error code, or None.
PyObject* quantize_fp4(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 3 || !THPVariable_Check(args[0])) Py_RETURN_NONE;
  const Tensor& x = THPVariable_Unpack(args[0]);
  const long device = PyLong_AsLong(args[2]);
  void* stream = PyLong_AsVoidPtr(args[1]);
  if (PyErr_Occurred()) return nullptr;
  const int32_t code = dtype_code(x);
  if (!plain_cuda(x, device) || code < 0 || x.dim() != 2 || wants_grad(x) || x.numel() == 0 || x.size(1) > TTHRML_FP4_MAX_COLS ||
      (x.size(1) > 1 && x.stride(1) != 1))
    Py_RETURN_NONE;
  const int64_t rows = x.size(0), cols = x.size(1), pitch = (cols + 31) / 32 * 16;
  Tensor codes = at::empty({rows, pitch}, x.options().dtype(at::kByte).requires_grad(false));
  Tensor blocks = bytes(x, library.fp4_scale_bytes(rows, cols)), scale = floats(x, {rows});
  const int rc = library.fp4_quantize(x.const_data_ptr(), code, rows, cols, x.stride(0), 1, codes.mutable_data_ptr(), pitch,
                                      blocks.mutable_data_ptr(), scale.mutable_data_ptr<float>(), stream);
  if (rc) return PyLong_FromLong(rc);
  PyObject *a = THPVariable_Wrap(codes), *b = THPVariable_Wrap(blocks), *c = THPVariable_Wrap(scale);
  PyObject* t = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  Py_XDECREF(c);
  return t;
  END_HANDLE_TH_ERRORS
}

// fp4_values(codes, pitch, block scales, scales, columns, stream) -> the float32 matrix, or an error code.
PyObject* fp4_values(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 6) {
    PyErr_SetString(PyExc_TypeError, "fp4_values(codes, pitch, blocks, scale, cols, stream)");
    return nullptr;
  }
  const Tensor &codes = THPVariable_Unpack(args[0]), &blocks = THPVariable_Unpack(args[2]), &scale = THPVariable_Unpack(args[3]);
  const int64_t pitch = PyLong_AsLongLong(args[1]), cols = PyLong_AsLongLong(args[4]), rows = codes.size(0);
  void* stream = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred()) return nullptr;
  Tensor out = floats(codes, {rows, cols});
  const int rc = library.fp4_values(codes.const_data_ptr(), pitch, blocks.const_data_ptr(), scale.const_data_ptr<float>(), rows, cols,
                                    out.mutable_data_ptr<float>(), stream);
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// fp4_product(x, codes, pitch, block scales, scales, columns, bias or None, error word, stream, device) -> the product in x's
// type, an error code, or None.
PyObject* fp4_product(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10 || !THPVariable_Check(args[0]) || !(args[6] == Py_None || THPVariable_Check(args[6]))) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &codes = THPVariable_Unpack(args[1]), &blocks = THPVariable_Unpack(args[3]),
               &scale = THPVariable_Unpack(args[4]);
  const int64_t pitch = PyLong_AsLongLong(args[2]), K = PyLong_AsLongLong(args[5]), N = codes.size(0);
  const long device = PyLong_AsLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const int32_t code = dtype_code(x);
  if (!plain_cuda(x, device) || code < 0 || x.dim() < 1 || wants_grad(x) || wants_grad(scale) || (x.dim() != 2 && !x.is_contiguous()) ||
      x.size(-1) != K || N < 1 || x.numel() == 0)
    Py_RETURN_NONE;
  if (x.dim() == 2 && K > 1 && x.stride(1) != 1) Py_RETURN_NONE;
  const float* bias = nullptr;
  if (args[6] != Py_None) {
    const Tensor& b = THPVariable_Unpack(args[6]);
    if (!plain_cuda(b, device) || b.scalar_type() != at::kFloat || b.dim() != 1 || b.size(0) != N || !b.is_contiguous() || wants_grad(b))
      Py_RETURN_NONE;
    bias = b.const_data_ptr<float>();
  }
  const int64_t M = x.numel() / K;
  at::DimVector sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = N;
  Tensor out = at::empty(sizes, x.options().requires_grad(false));
  const int64_t size = library.fp4_linear_workspace(M, K, N);
  Tensor space;
  if (size) space = bytes(x, size);
  const int rc = library.fp4_linear(x.const_data_ptr(), code, M, K, x.dim() == 2 ? x.stride(0) : K, 1, size ? space.mutable_data_ptr() : nullptr, size,
                                    codes.const_data_ptr(), pitch, blocks.const_data_ptr(), scale.const_data_ptr<float>(), N, bias,
                                    out.mutable_data_ptr(), code, N, reinterpret_cast<int32_t*>(PyLong_AsVoidPtr(args[7])),
                                    PyLong_AsVoidPtr(args[8]));
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace hostcall
