// Python module `hetuctr_nn`: the dense operators of the C ABI on torch tensors, for hetuctr_amd/nn.py.  Host-only C++: argument
// checks, results from torch's allocator, one hctr_* call.  It is here because a call of few rows is the host's time: the same
// steps in Python took 5 us of a layer_norm call, of which the launch is 2.9.
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include <forward_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>

#include "hetuctr_hip.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> Maybe;

[[noreturn]] void refuse(const std::string &why) { throw std::runtime_error("hetuctr_amd.nn: " + why); }
void done(int status) {
  if (status) throw std::runtime_error(hctr_last_error());
}

// ---- arguments ------------------------------------------------------------------------------------------------------
struct Arguments {
  PyObject *const *given;
  Py_ssize_t count;
  void expect(Py_ssize_t n) const {
    if (count != n) refuse("wrong number of arguments");
  }
  mutable std::forward_list<Tensor> made; // in place of what was given, until the call is made
  const Tensor &as_read(const Tensor &t) const {
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
      refuse("there are no forward-mode derivatives, and a tensor has a tangent");
    if (!t.is_neg()) return t;
    return made.emplace_front(t.resolve_neg()); // a view of memory that holds the values with the other sign
  }
  const Tensor &tensor(int i, const char *what) const {
    if (!THPVariable_Check(given[i])) refuse(std::string(what) + " must be a tensor");
    return as_read(THPVariable_Unpack(given[i]));
  }
  Maybe maybe(int i, const char *what) const {
    if (given[i] == Py_None) return std::nullopt;
    return tensor(i, what);
  }
  bool flag(int i) const {
    const int v = PyObject_IsTrue(given[i]);
    if (v < 0) throw python_error();
    return v;
  }
  double number(int i) const {
    const double v = PyFloat_AsDouble(given[i]);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
  void *stream(int i) const {
    void *p = PyLong_AsVoidPtr(given[i]);
    if (!p && PyErr_Occurred()) throw python_error();
    return p;
  }
};

uint64_t word(PyObject *o) { // modulo 2^64
  const uint64_t v = PyLong_AsUnsignedLongLongMask(o);
  if (v == (uint64_t)-1 && PyErr_Occurred()) throw python_error();
  return v;
}

int type_of(at::ScalarType t, const char *what) {
  if (t == at::kFloat) return HCTR_F32;
  if (t == at::kBFloat16) return HCTR_BF16;
  if (t == at::kHalf) return HCTR_F16;
  refuse(std::string(what) + " must be float32, bfloat16 or float16, not " + c10::toString(t));
}

// argument i: a Drop (p, seed, step, step_tensor), or None
hctr_drop drop_of(const Arguments &a, int i, const Tensor &like) {
  PyObject *o = a.given[i];
  hctr_drop d = {0.0, 0, 0, nullptr};
  if (o == Py_None) return d;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("drop must be a Drop");
  d.p = PyFloat_AsDouble(PyTuple_GET_ITEM(o, 0));
  if (d.p == -1.0 && PyErr_Occurred()) throw python_error();
  d.seed = word(PyTuple_GET_ITEM(o, 1));
  d.step = word(PyTuple_GET_ITEM(o, 2));
  PyObject *extra = PyTuple_GET_ITEM(o, 3);
  if (extra != Py_None) {
    if (!THPVariable_Check(extra)) refuse("the step tensor must be one int64 on the device of the values");
    const Tensor &t = a.as_read(THPVariable_Unpack(extra));
    if (t.device() != like.device() || t.scalar_type() != at::kLong || t.numel() != 1)
      refuse("the step tensor must be one int64 on the device of the values");
    d.step_dev = (const uint64_t *)t.data_ptr();
    if (!d.step_dev) refuse("the step tensor has no memory");
  }
  return d;
}

// A tensor as rows of its last dimension; a copy where its memory order does not allow that, kept until the call is made.
struct Matrix {
  Tensor kept;
  size_t rows, width;
  hctr_matrix at;
};
Matrix matrix_of(const Tensor &given, const char *what) {
  if (!given.is_cuda()) refuse(std::string(what) + " must be on the GPU");
  Tensor t = given;
  if (t.dim() != 2) {
    if (t.dim() == 0) refuse(std::string(what) + " must have at least one dimension");
    const int64_t width = t.size(-1);
    t = t.reshape({width ? t.numel() / width : 0, width});
  }
  if (t.stride(1) != 1 && t.size(1) != 1) t = t.contiguous();
  const hctr_matrix at = {t.data_ptr(), t.stride(0)};
  return {t, (size_t)t.size(0), (size_t)t.size(1), at};
}

std::string text(at::IntArrayRef sizes) {
  std::string s = "(";
  for (size_t i = 0; i < sizes.size(); i++) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + ")";
}
void same(const Tensor &t, const Tensor &like, at::ScalarType dtype, const char *what) {
  if (t.sizes() != like.sizes() || t.scalar_type() != dtype || t.device() != like.device())
    refuse(std::string(what) + " must be " + c10::toString(dtype) + " of shape " + text(like.sizes()) + " on " + like.device().str());
}

// weight and bias, ready to be read
struct Affine {
  Maybe weight, bias;
  int type = HCTR_F32;
};
Affine affine_of(Maybe weight, Maybe bias, size_t width, at::ScalarType act, const Tensor &like) {
  Affine a;
  const auto check = [&](Maybe &t, const char *what) {
    if (!t) return;
    if (t->dim() != 1 || (size_t)t->size(0) != width || t->device() != like.device() || (t->scalar_type() != at::kFloat && t->scalar_type() != act))
      refuse(std::string(what) + " must hold " + std::to_string(width) + " values of Float or " + c10::toString(act) + " on " + like.device().str());
    if (!t->is_contiguous()) t = t->contiguous();
    a.type = type_of(t->scalar_type(), what);
  };
  check(weight, "weight");
  check(bias, "bias");
  if (weight && bias && weight->scalar_type() != bias->scalar_type()) refuse("weight and bias must be of one type");
  a.weight = std::move(weight);
  a.bias = std::move(bias);
  return a;
}
// null: there is no such tensor.  One whose memory is missing must not be taken for that.
void *pointer(const Maybe &t, const char *what) {
  if (!t) return nullptr;
  void *p = t->data_ptr();
  if (!p && t->numel()) refuse(std::string(what) + " has no memory");
  return p;
}

Tensor result(at::IntArrayRef sizes, const Tensor &like, at::ScalarType dtype) { return at::empty(sizes, like.options().dtype(dtype)); }
hctr_matrix whole(const Tensor &t, size_t width) { return {t.data_ptr(), (int64_t)width}; }

Tensor statistic(const Tensor &t, size_t rows, const Tensor &like, const char *what) {
  if ((size_t)t.numel() != rows || t.scalar_type() != at::kFloat || t.device() != like.device())
    refuse(std::string(what) + " must hold a float32 for each of the " + std::to_string(rows) + " rows on " + like.device().str());
  return t.is_contiguous() ? t : t.contiguous();
}

PyObject *wrap(const Maybe &t) {
  if (!t) Py_RETURN_NONE;
  return THPVariable_Wrap(*t);
}
template <typename... T> PyObject *tuple(const T &...t) {
  PyObject *items[] = {wrap(t)...}, *all = PyTuple_New(sizeof...(T));
  for (size_t i = 0; i < sizeof...(T); i++) PyTuple_SET_ITEM(all, (Py_ssize_t)i, items[i]);
  return all;
}

// ---- the operators ----------------------------------------------------------------------------------------------------
// (x, drop, stream)
PyObject *dropout(const Arguments &a) {
  a.expect(3);
  const Tensor &x = a.tensor(0, "x");
  const Matrix m = matrix_of(x, "x");
  hctr_dropout_args r = {};
  r.rows = m.rows, r.width = m.width;
  r.dtype = type_of(x.scalar_type(), "x");
  r.drop = drop_of(a, 1, x);
  const Tensor y = result(x.sizes(), x, x.scalar_type());
  r.x = m.at, r.y = whole(y, m.width);
  r.stream = a.stream(2);
  done(hctr_dropout(&r));
  return wrap(y);
}

// (x, residual or None, weight, bias, eps, drop, dtype or None, stats, stream): y, [sum,] mean or None, rstd or None
PyObject *forward(const Arguments &a) {
  a.expect(9);
  const Tensor &x = a.tensor(0, "x");
  const Maybe residual = a.maybe(1, "residual");
  const at::ScalarType act = a.given[6] == Py_None ? x.scalar_type()
                             : THPDtype_Check(a.given[6]) ? reinterpret_cast<THPDtype *>(a.given[6])->scalar_type
                                                          : (refuse("dtype must be a torch.dtype"), at::kFloat);
  const Matrix m = matrix_of(x, "x");
  hctr_norm_args r = {};
  r.rows = m.rows, r.width = m.width;
  r.x = m.at;
  Matrix other;
  Maybe sum;
  if (residual) {
    same(*residual, x, residual->scalar_type(), "residual");
    other = matrix_of(*residual, "residual");
    r.residual = other.at;
  }
  r.stream_dtype = residual ? type_of(residual->scalar_type(), "residual") : type_of(x.scalar_type(), "x");
  r.act_dtype = type_of(act, residual ? "x" : "the result");
  const Affine affine = affine_of(a.maybe(2, "weight"), a.maybe(3, "bias"), m.width, act, x);
  r.weight = pointer(affine.weight, "weight"), r.bias = pointer(affine.bias, "bias"), r.affine_dtype = affine.type;
  r.eps = (float)a.number(4);
  r.drop = drop_of(a, 5, x);
  const Tensor y = result(x.sizes(), x, act);
  r.y = whole(y, m.width);
  if (residual) {
    sum = result(x.sizes(), x, residual->scalar_type());
    r.sum = whole(*sum, m.width);
  }
  Maybe mean, rstd;
  if (a.flag(7)) {
    mean = result({(int64_t)m.rows}, x, at::kFloat);
    rstd = result({(int64_t)m.rows}, x, at::kFloat);
    r.mean = (float *)mean->data_ptr(), r.rstd = (float *)rstd->data_ptr();
  }
  r.stream = a.stream(8);
  done(residual ? hctr_dropout_add_layer_norm(&r) : hctr_layer_norm(&r));
  return residual ? tuple(Maybe(y), sum, mean, rstd) : tuple(Maybe(y), mean, rstd);
}

// (add, dy, ds or None, s, mean, rstd, weight, bias, drop, need_x, need_weight, need_bias, stream): dx, [dresidual,] dweight, dbias
PyObject *backward(const Arguments &a) {
  a.expect(13);
  const bool add = a.flag(0);
  const char *normed = add ? "s" : "x";
  const Tensor &dy = a.tensor(1, "dy"), &s = a.tensor(3, normed);
  const Maybe ds = a.maybe(2, "ds");
  same(dy, s, dy.scalar_type(), "dy");
  const Matrix m = matrix_of(s, normed), g = matrix_of(dy, "dy");
  hctr_norm_grad_args r = {};
  r.rows = m.rows, r.width = m.width;
  r.s = m.at, r.dy = g.at;
  Matrix more;
  if (ds) {
    same(*ds, s, s.scalar_type(), "ds");
    more = matrix_of(*ds, "ds");
    r.dsum = more.at;
    pointer(more.kept, "ds");
  }
  r.stream_dtype = type_of(s.scalar_type(), normed);
  r.act_dtype = type_of(dy.scalar_type(), "dy");
  const Affine affine = affine_of(a.maybe(6, "weight"), a.maybe(7, "bias"), m.width, dy.scalar_type(), s);
  r.weight = pointer(affine.weight, "weight"), r.affine_dtype = affine.type;
  const Tensor mean = statistic(a.tensor(4, "mean"), m.rows, s, "mean"), rstd = statistic(a.tensor(5, "rstd"), m.rows, s, "rstd");
  r.mean = (const float *)mean.data_ptr(), r.rstd = (const float *)rstd.data_ptr();
  r.drop = drop_of(a, 8, s);
  Maybe dx, dresidual, dweight, dbias, space;
  bool one = false; // dx and dresidual are one tensor
  if (add) {
    dresidual = result(s.sizes(), s, s.scalar_type());
    r.dresidual = whole(*dresidual, m.width);
    one = dy.scalar_type() == s.scalar_type() && r.drop.p == 0.0;
    if (a.flag(9) && !one) dx = result(s.sizes(), s, dy.scalar_type());
  } else {
    dx = result(s.sizes(), s, s.scalar_type());
  }
  if (dx) r.dx = whole(*dx, m.width);
  if (affine.weight && a.flag(10)) dweight = result(affine.weight->sizes(), s, affine.weight->scalar_type());
  if (affine.bias && a.flag(11)) dbias = result(affine.bias->sizes(), s, affine.bias->scalar_type());
  r.dweight = pointer(dweight, "dweight"), r.dbias = pointer(dbias, "dbias");
  if (dweight || dbias) {
    r.workspace_bytes = hctr_layer_norm_workspace(m.rows, m.width);
    if (r.workspace_bytes) {
      space = result({(int64_t)r.workspace_bytes}, s, at::kByte);
      r.workspace = space->data_ptr();
    }
  }
  r.stream = a.stream(12);
  done(add ? hctr_dropout_add_layer_norm_backward(&r) : hctr_layer_norm_backward(&r));
  if (add) return tuple(one && a.flag(9) ? dresidual : dx, dresidual, dweight, dbias);
  return tuple(dx, dweight, dbias);
}

// The GPU on which tensor x lies; -1: on none, or something sees, and may record or change, what goes through torch's dispatcher (a
// dispatch mode, a tracer)
PyObject *unseen_on(PyObject *, PyObject *x) {
  if (!THPVariable_Check(x)) {
    PyErr_SetString(PyExc_TypeError, "hetuctr_amd.nn: a tensor is needed");
    return nullptr;
  }
  const bool seen = c10::impl::dispatch_mode_enabled() || at::tracer::impl::is_dispatch_enabled();
  const Tensor &t = THPVariable_Unpack(x);
  return PyLong_FromLong(!seen && t.is_cuda() ? t.get_device() : -1);
}

// Whether a tracer records torch's operators
PyObject *traced(PyObject *, PyObject *) { return PyBool_FromLong(at::tracer::impl::is_dispatch_enabled()); }

// An error comes out as torch's own operators raise it: memory that runs out as torch.OutOfMemoryError, what Python has set already
// (python_error) as it is.
template <PyObject *(*F)(const Arguments &)> PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  at::NoGradGuard off;
  return F({args, count});
  END_HANDLE_TH_ERRORS
}
template <PyObject *(*F)(const Arguments &)> PyCFunction method() { return (PyCFunction)(void (*)())call<F>; }

PyMethodDef methods[] = {{"dropout", method<dropout>(), METH_FASTCALL, nullptr},
                         {"forward", method<forward>(), METH_FASTCALL, nullptr},
                         {"backward", method<backward>(), METH_FASTCALL, nullptr},
                         {"unseen_on", unseen_on, METH_O, nullptr},
                         {"traced", traced, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hetuctr_nn", "The dense operators on torch tensors; use hetuctr_amd.nn.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_hetuctr_nn() { return PyModule_Create(&module); }
