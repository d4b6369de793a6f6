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

#include <algorithm>
#include <forward_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

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
  long long whole(int i) const {
    const long long v = PyLong_AsLongLong(given[i]);
    if (v == -1 && PyErr_Occurred()) throw python_error();
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

// A result's matrix, and memory for a call's workspace
hctr_matrix matrix(const Maybe &t, size_t width) { return t ? whole(*t, width) : hctr_matrix{nullptr, 0}; }
template <typename R> Tensor with_space(R &r, size_t bytes, const Tensor &like) {
  if (bytes == (size_t)-1) done(1);
  if (!bytes) return Tensor();
  const Tensor space = result({(int64_t)bytes}, like, at::kByte);
  r.workspace = space.data_ptr(), r.workspace_bytes = bytes;
  return space;
}
// A matrix that is read, of the type and on the device of `like`
Matrix matrix_like(const Tensor &t, const Tensor &like, size_t rows, size_t width, const char *what) {
  const Matrix m = matrix_of(t, what);
  if (m.rows != rows || m.width != width || t.scalar_type() != like.scalar_type() || t.device() != like.device())
    refuse(std::string(what) + " must be " + c10::toString(like.scalar_type()) + " of " + std::to_string(rows) + " rows of " + std::to_string(width) + " on " + like.device().str());
  if (!m.at.data && rows && width) refuse(std::string(what) + " has no memory");
  return m;
}
// weights: a matrix of as many columns as x has
Matrix weights_of(const Tensor &t, const Tensor &x, size_t width, const char *what) {
  if (t.dim() != 2) refuse(std::string(what) + " must be a matrix");
  return matrix_like(t, x, (size_t)t.size(0), width, what);
}
struct Bias {
  Maybe t;
  void *at = nullptr;
};
Bias bias_of(Maybe t, size_t n, const Tensor &x, int &type, bool &any, const char *what) {
  Bias b;
  if (!t) return b;
  if (t->dim() != 1 || (size_t)t->size(0) != n || t->device() != x.device() || (t->scalar_type() != at::kFloat && t->scalar_type() != x.scalar_type()))
    refuse(std::string(what) + " must hold " + std::to_string(n) + " values of Float or " + c10::toString(x.scalar_type()) + " on " + x.device().str());
  const int own = type_of(t->scalar_type(), what);
  if (any && own != type) refuse("the biases must be of one type");
  type = own, any = true;
  b.t = t->is_contiguous() ? std::move(t) : Maybe(t->contiguous());
  b.at = pointer(b.t, what);
  return b;
}
std::vector<int64_t> rows_shape(const Tensor &x) { return {x.sizes().begin(), x.sizes().end() - 1}; }
std::vector<int64_t> rows_shape(const Tensor &x, size_t width) {
  std::vector<int64_t> s = rows_shape(x);
  s.push_back((int64_t)width);
  return s;
}
int activation_of(const Arguments &a, int i) { return (int)std::clamp(a.whole(i), -1LL, 100LL); }

// (x, gate_weight, up_weight, gate_bias, up_bias, activation, saved, stream): h, gate or None, up or None
PyObject *gated(const Arguments &a) {
  a.expect(8);
  const Tensor &x = a.tensor(0, "x");
  hctr_gated_args r = {};
  r.dtype = type_of(x.scalar_type(), "x");
  const Matrix m = matrix_of(x, "x");
  const Matrix gate_weight = weights_of(a.tensor(1, "gate_weight"), x, m.width, "gate_weight");
  const Matrix up_weight = matrix_like(a.tensor(2, "up_weight"), x, gate_weight.rows, m.width, "up_weight");
  r.rows = m.rows, r.width = m.width, r.hidden = gate_weight.rows;
  r.x = m.at, r.gate_weight = gate_weight.at, r.up_weight = up_weight.at;
  bool any = false;
  const Bias gate_bias = bias_of(a.maybe(3, "gate_bias"), r.hidden, x, r.bias_dtype, any, "gate_bias");
  const Bias up_bias = bias_of(a.maybe(4, "up_bias"), r.hidden, x, r.bias_dtype, any, "up_bias");
  r.gate_bias = gate_bias.at, r.up_bias = up_bias.at;
  r.activation = activation_of(a, 5);
  const bool saved = a.flag(6);
  const std::vector<int64_t> shape = rows_shape(x, r.hidden);
  const Tensor h = result(shape, x, x.scalar_type());
  Maybe gate, up;
  if (saved) gate = result(shape, x, x.scalar_type()), up = result(shape, x, x.scalar_type());
  r.h = whole(h, r.hidden), r.gate = matrix(gate, r.hidden), r.up = matrix(up, r.hidden);
  const Tensor space = with_space(r, hctr_gated_linear_workspace(&r), x);
  r.stream = a.stream(7);
  done(hctr_gated_linear(&r));
  return tuple(Maybe(h), gate, up);
}

// (dh, x, gate, up, gate_weight, up_weight, gate_bias, up_bias, activation, need_x, need_gate_weight, need_up_weight, need_gate_bias,
// need_up_bias, stream): dx, dgate_weight, dup_weight, dgate_bias, dup_bias
PyObject *gated_backward(const Arguments &a) {
  a.expect(15);
  const Tensor &x = a.tensor(1, "x"), &gate_weight = a.tensor(4, "gate_weight"), &up_weight = a.tensor(5, "up_weight");
  hctr_gated_grad_args r = {};
  r.dtype = type_of(x.scalar_type(), "x");
  const Matrix m = matrix_of(x, "x");
  const Matrix gw = weights_of(gate_weight, x, m.width, "gate_weight");
  const Matrix uw = matrix_like(up_weight, x, gw.rows, m.width, "up_weight");
  r.rows = m.rows, r.width = m.width, r.hidden = gw.rows;
  const Matrix dh = matrix_like(a.tensor(0, "dh"), x, r.rows, r.hidden, "dh");
  const Matrix gate = matrix_like(a.tensor(2, "gate"), x, r.rows, r.hidden, "gate"), up = matrix_like(a.tensor(3, "up"), x, r.rows, r.hidden, "up");
  r.dh = dh.at, r.x = m.at, r.gate = gate.at, r.up = up.at, r.gate_weight = gw.at, r.up_weight = uw.at;
  bool any = false;
  const Maybe gate_bias = a.maybe(6, "gate_bias"), up_bias = a.maybe(7, "up_bias"); // what they hold is not read
  for (const auto &[bias, what] : {std::pair(&gate_bias, "gate_bias"), std::pair(&up_bias, "up_bias")}) {
    if (!*bias) continue;
    if ((size_t)(*bias)->numel() != r.hidden || ((*bias)->scalar_type() != at::kFloat && (*bias)->scalar_type() != x.scalar_type()))
      refuse(std::string(what) + " must hold " + std::to_string(r.hidden) + " values of Float or " + c10::toString(x.scalar_type()));
    const int own = type_of((*bias)->scalar_type(), what);
    if (any && own != r.bias_dtype) refuse("the biases must be of one type");
    r.bias_dtype = own, any = true;
  }
  r.activation = activation_of(a, 8);
  Maybe dx, dgate_weight, dup_weight, dgate_bias, dup_bias;
  if (a.flag(9)) dx = result(x.sizes(), x, x.scalar_type());
  if (a.flag(10)) dgate_weight = result(gate_weight.sizes(), x, x.scalar_type());
  if (a.flag(11)) dup_weight = result(up_weight.sizes(), x, x.scalar_type());
  if (gate_bias && a.flag(12)) dgate_bias = result(gate_bias->sizes(), x, gate_bias->scalar_type());
  if (up_bias && a.flag(13)) dup_bias = result(up_bias->sizes(), x, up_bias->scalar_type());
  r.dx = matrix(dx, r.width), r.dgate_weight = matrix(dgate_weight, r.width), r.dup_weight = matrix(dup_weight, r.width);
  r.dgate_bias = pointer(dgate_bias, "dgate_bias"), r.dup_bias = pointer(dup_bias, "dup_bias");
  const Tensor space = with_space(r, hctr_gated_linear_backward_workspace(&r), x);
  r.stream = a.stream(14);
  done(hctr_gated_linear_backward(&r));
  return tuple(dx, dgate_weight, dup_weight, dgate_bias, dup_bias);
}

Tensor targets_of(const Tensor &t, const Tensor &x) {
  if (t.sizes() != at::IntArrayRef(rows_shape(x)) || t.scalar_type() != at::kLong || t.device() != x.device())
    refuse("target must be Long of shape " + text(rows_shape(x)) + " on " + x.device().str());
  return t.contiguous();
}
Tensor per_row(const Tensor &t, const Tensor &x, const char *what) {
  if (t.sizes() != at::IntArrayRef(rows_shape(x)) || t.scalar_type() != at::kFloat || t.device() != x.device())
    refuse(std::string(what) + " must be Float of shape " + text(rows_shape(x)) + " on " + x.device().str());
  return t.contiguous();
}

// (x, weight, target, bias, ignore_index, stats, stream): loss, lse or None
PyObject *items(const Arguments &a) {
  a.expect(7);
  const Tensor &x = a.tensor(0, "x");
  hctr_items_args r = {};
  r.dtype = type_of(x.scalar_type(), "x");
  const Matrix m = matrix_of(x, "x"), weight = weights_of(a.tensor(1, "weight"), x, m.width, "weight");
  const Tensor target = targets_of(a.tensor(2, "target"), x);
  r.rows = m.rows, r.width = m.width, r.items = weight.rows;
  r.x = m.at, r.weight = weight.at;
  bool any = false;
  const Bias bias = bias_of(a.maybe(3, "bias"), r.items, x, r.bias_dtype, any, "bias");
  r.bias = bias.at;
  r.target = (const int64_t *)pointer(target, "target"), r.ignore_index = a.whole(4);
  const Tensor loss = result(rows_shape(x), x, at::kFloat);
  Maybe lse;
  if (a.flag(5)) lse = result(rows_shape(x), x, at::kFloat), r.lse = (float *)lse->data_ptr();
  r.loss = (float *)loss.data_ptr();
  const Tensor space = with_space(r, hctr_linear_cross_entropy_workspace(&r), x);
  r.stream = a.stream(6);
  done(hctr_linear_cross_entropy(&r));
  return tuple(Maybe(loss), lse);
}

// (dloss, x, weight, target, lse, bias, ignore_index, need_x, need_weight, need_bias, stream): dx, dweight, dbias
PyObject *items_backward(const Arguments &a) {
  a.expect(11);
  const Tensor &x = a.tensor(1, "x"), &weight = a.tensor(2, "weight");
  hctr_items_grad_args r = {};
  r.dtype = type_of(x.scalar_type(), "x");
  const Matrix m = matrix_of(x, "x"), w = weights_of(weight, x, m.width, "weight");
  const Tensor target = targets_of(a.tensor(3, "target"), x), dloss = per_row(a.tensor(0, "dloss"), x, "dloss"), lse = per_row(a.tensor(4, "lse"), x, "lse");
  r.rows = m.rows, r.width = m.width, r.items = w.rows;
  r.x = m.at, r.weight = w.at;
  bool any = false;
  const Bias bias = bias_of(a.maybe(5, "bias"), r.items, x, r.bias_dtype, any, "bias");
  r.bias = bias.at;
  r.target = (const int64_t *)pointer(target, "target"), r.ignore_index = a.whole(6);
  r.dloss = (const float *)pointer(dloss, "dloss"), r.lse = (const float *)pointer(lse, "lse");
  Maybe dx, dweight, dbias;
  if (a.flag(7)) dx = result(x.sizes(), x, x.scalar_type());
  if (a.flag(8)) dweight = result(weight.sizes(), x, x.scalar_type());
  if (bias.t && a.flag(9)) dbias = result({(int64_t)r.items}, x, bias.t->scalar_type());
  r.dx = matrix(dx, r.width), r.dweight = matrix(dweight, r.width), r.dbias = pointer(dbias, "dbias");
  const Tensor space = with_space(r, hctr_linear_cross_entropy_backward_workspace(&r), x);
  r.stream = a.stream(10);
  done(hctr_linear_cross_entropy_backward(&r));
  return tuple(dx, dweight, dbias);
}

// ---- many gradients ---------------------------------------------------------------------------------------------------
std::vector<Tensor> tensors_of(const Arguments &a, PyObject *list, const char *what, bool read) {
  if (!PyList_Check(list)) refuse(std::string(what) + " must be a list");
  std::vector<Tensor> all;
  all.reserve(PyList_GET_SIZE(list));
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); i++) {
    PyObject *o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) refuse(std::string(what) + " must be tensors");
    const Tensor &t = THPVariable_Unpack(o);
    const Tensor &v = read ? a.as_read(t) : t;
    if (!v.is_cuda()) refuse(std::string(what) + " must be on the GPU");
    if (v.device() != (all.empty() ? v : all[0]).device()) refuse(std::string(what) + " must be on one device");
    all.push_back(v);
  }
  return all;
}
hctr_gradient gradient_of(const Tensor &t, const char *what) {
  hctr_gradient g = {};
  g.count = (size_t)t.numel(), g.dtype = type_of(t.scalar_type(), what);
  g.values = g.count ? t.data_ptr() : nullptr;
  if (g.count && !g.values) refuse(std::string(what) + " has no memory");
  return g;
}
// (values one behind the other, in whatever order)
Tensor dense(const Tensor &t) { return t.is_non_overlapping_and_dense() ? t : t.contiguous(); }

// (gradients, stream): norm
PyObject *gradient_norm(const Arguments &a) {
  a.expect(2);
  std::vector<Tensor> given = tensors_of(a, a.given[0], "gradients", true);
  if (given.empty()) refuse("there are no gradients");
  std::vector<hctr_gradient> list;
  for (Tensor &t : given) {
    t = dense(t);
    list.push_back(gradient_of(t, "a gradient"));
  }
  const Tensor norm = result({}, given[0], at::kFloat);
  hctr_clip_args r = {};
  r.gradients = list.data(), r.count = list.size(), r.norm = (float *)norm.data_ptr();
  const Tensor space = with_space(r, hctr_gradient_workspace(&r), norm);
  r.stream = a.stream(1);
  done(hctr_gradient_norm(&r));
  return wrap(norm);
}

// (gradients, into, max_norm, norm or None, whether results may not want gradients, stream): norm
PyObject *clip_gradients(const Arguments &a) {
  a.expect(6);
  std::vector<Tensor> given = tensors_of(a, a.given[0], "gradients", true), into = tensors_of(a, a.given[1], "into", false);
  if (given.empty()) refuse("there are no gradients");
  if (given.size() != into.size()) refuse("there must be as many results as gradients");
  if (given[0].device() != into[0].device()) refuse("into must be on the device of the gradients");
  const Maybe norm = a.maybe(3, "norm");
  const bool leaves = a.flag(4);
  std::vector<hctr_gradient> list;
  for (size_t i = 0; i < given.size(); i++) {
    Tensor &t = given[i];
    const Tensor &o = into[i];
    if (o.sizes() != t.sizes() || o.scalar_type() != t.scalar_type())
      refuse("a result must be of its gradient's type and shape, " + std::string(c10::toString(t.scalar_type())) + " " + text(t.sizes()));
    if (!o.is_non_overlapping_and_dense() || o.is_neg()) refuse("a result must hold its values one behind the other");
    if (leaves && o.requires_grad()) refuse("a result is written in place, and wants a gradient: call this under torch.no_grad()");
    if (!t.is_non_overlapping_and_dense() || t.strides() != o.strides()) t = at::empty_like(o).copy_(t);
    hctr_gradient g = gradient_of(t, "a gradient");
    g.into = g.count ? o.data_ptr() : nullptr;
    if (g.count && !g.into) refuse("a result has no memory");
    list.push_back(g);
  }
  hctr_clip_args r = {};
  r.gradients = list.data(), r.count = list.size();
  Tensor out;
  if (norm) {
    if (norm->numel() != 1 || norm->scalar_type() != at::kFloat || norm->device() != given[0].device())
      refuse("norm must be one float32 on " + given[0].device().str());
    out = *norm;
    r.given = (const float *)pointer(norm, "norm");
  } else {
    out = result({}, given[0], at::kFloat);
    r.norm = (float *)out.data_ptr();
  }
  r.max_norm = (float)a.number(2);
  Tensor space;
  if (!norm) space = with_space(r, hctr_gradient_workspace(&r), given[0]);
  r.stream = a.stream(5);
  done(hctr_clip_gradients(&r));
  for (const Tensor &o : into)
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  return wrap(out);
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
                         {"gated", method<gated>(), METH_FASTCALL, nullptr},
                         {"gated_backward", method<gated_backward>(), METH_FASTCALL, nullptr},
                         {"items", method<items>(), METH_FASTCALL, nullptr},
                         {"items_backward", method<items_backward>(), METH_FASTCALL, nullptr},
                         {"gradient_norm", method<gradient_norm>(), METH_FASTCALL, nullptr},
                         {"clip_gradients", method<clip_gradients>(), METH_FASTCALL, nullptr},
                         {"unseen_on", unseen_on, METH_O, nullptr},
                         {"traced", traced, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hetuctr_nn", "The dense operators on torch tensors; use hetuctr_amd.nn.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_hetuctr_nn() { return PyModule_Create(&module); }
