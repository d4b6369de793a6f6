// The gated linear layer and its gradient: argument checks, workspaces, the launches.
#include "gated.h"

#include <algorithm>

#include "dense.h"
#include "few_rows.h"

namespace hctr {
namespace {

Operand operand(const Layout &l, size_t rows) { return {{l.at, nullptr}, l.stride, (uint32_t)rows, 0, 0}; }

struct ForwardPlan {
  bool few;
  Shape shape;
  size_t x, gate, up, partial, bytes;
};
ForwardPlan plan_of(const hctr_gated_args &a) {
  ForwardPlan p = {};
  if (!a.rows) return p;
  p.few = a.rows <= kFewRows;
  if (p.few) return p;
  const size_t size = size_of(a.dtype);
  p.shape = shape_of(a.rows, a.hidden, a.width, (int)size, true, true);
  p.x = laid_out_bytes(a.x, a.rows, a.width, size);
  p.gate = laid_out_bytes(a.gate_weight, a.hidden, a.width, size);
  p.up = laid_out_bytes(a.up_weight, a.hidden, a.width, size);
  // (the two weights' tiles are counted with one stride)
  if (!p.gate != !p.up || (!p.gate && a.hidden > 1 && a.gate_weight.stride != a.up_weight.stride))
    p.gate = p.up = up(a.hidden * up(a.width * size, 16), 256);
  if (p.shape.splits > 1) p.partial = 2 * parts_bytes(a.rows, a.hidden, p.shape.splits);
  p.bytes = p.x + p.gate + p.up + p.partial;
  return p;
}

void check(const hctr_gated_args &a) {
  check_dtype(a.dtype, "gated linear");
  check_sizes(a.rows, a.width, a.hidden, 1u << 20, "gated linear", "hidden must be in 1..2^20");
  HCTR_CHECK(a.activation >= HCTR_SILU && a.activation <= HCTR_SIGMOID, "gated linear: unknown activation");
  HCTR_CHECK(!(a.gate_bias || a.up_bias) || a.bias_dtype == HCTR_F32 || a.bias_dtype == a.dtype, "gated linear: the biases are of the matrices' type or float");
}

template <typename T> void forward(const hctr_gated_args &a) {
  const ForwardPlan plan = plan_of(a);
  const hipStream_t s = (hipStream_t)a.stream;
  const size_t size = sizeof(T);
  GatedForward p = {};
  p.rows = (uint32_t)a.rows, p.width = (uint32_t)a.width, p.hidden = (uint32_t)a.hidden;
  p.gate_bias = a.gate_bias, p.up_bias = a.up_bias, p.narrow = a.bias_dtype != HCTR_F32;
  p.activation = a.activation;
  p.h = a.h.data, p.gate = a.gate.data, p.up = a.up.data;
  p.h_stride = a.h.stride, p.gate_stride = a.gate.stride, p.up_stride = a.up.stride;
  if (plan.few) {
    p.loose_x = a.x.data, p.loose_gate = a.gate_weight.data, p.loose_up = a.up_weight.data;
    p.loose_stride = a.x.stride, p.loose_gate_stride = a.gate_weight.stride, p.loose_up_stride = a.up_weight.stride;
    return launch_gated_few<T>(p, s);
  }
  char *space = (char *)a.workspace;
  p.x = operand(laid_out(a.x, a.rows, a.width, a.dtype, space, s), a.rows);
  if (plan.gate) {
    const size_t stride = up(a.width * size, 16);
    for (int i = 0; i < 2; i++) {
      launch_copy_rows<T>(i ? a.up_weight : a.gate_weight, a.hidden, a.width, space, stride, s);
      p.weights.base[i] = space;
      space += plan.gate;
    }
    p.weights.stride = (int64_t)stride;
  } else {
    p.weights = {{(const char *)a.gate_weight.data, (const char *)a.up_weight.data}, a.hidden > 1 ? a.gate_weight.stride * (int64_t)size : (int64_t)(a.width * size), 0, 0, 0};
  }
  p.weights.rows = p.hidden;
  p.splits = plan.shape.splits;
  p.partial = p.splits > 1 ? (float *)space : nullptr;
  p.band = 8;
  launch_gated<T>(p, plan.shape.tile, s);
}

struct BackwardPlan {
  size_t padded, row_blocks, rows_each;
  Shape dx, dweight;
  size_t slopes, sums, sizes, x, gate, up, parts, bytes;
  bool weights;
};
BackwardPlan plan_of(const hctr_gated_grad_args &a) {
  BackwardPlan p = {};
  const size_t size = size_of(a.dtype), padded = up(a.hidden, kStepBytes / size);
  p.padded = padded;
  p.weights = a.dgate_weight.data || a.dup_weight.data;
  p.slopes = up(a.rows * 2 * padded * size, 256);
  // blocks for about eight rounds of the card, of 8 to 256 rows each
  const size_t across = div_up(padded, slope_columns((int)size));
  p.rows_each = std::min<size_t>(256, std::max<size_t>(8, up(a.rows * across / 8192 + 1, 8)));
  p.rows_each = std::max(p.rows_each, up((a.rows + 65534) / 65535, 8));
  p.row_blocks = div_up(a.rows, p.rows_each);
  if (a.dgate_bias || a.dup_bias) p.sums = up(p.row_blocks * 2 * padded * sizeof(float), 256);
  if (a.dtype == HCTR_F16 && a.rows && (a.dx.data || p.weights)) p.sizes = up((kGuesses + 2 + p.row_blocks * across) * sizeof(float), 256);
  if (a.dx.data && a.rows) {
    p.dx = shape_of(a.rows, a.width, 2 * padded, (int)size, false, true);
    if (p.dx.splits > 1) p.parts = parts_bytes(a.rows, a.width, p.dx.splits);
    p.gate = laid_out_bytes(a.gate_weight, a.hidden, a.width, size);
    p.up = laid_out_bytes(a.up_weight, a.hidden, a.width, size);
    if (!p.gate != !p.up || (!p.gate && a.hidden > 1 && a.gate_weight.stride != a.up_weight.stride))
      p.gate = p.up = up(a.hidden * up(a.width * size, 16), 256);
  }
  if (p.weights) {
    const size_t rows = a.dgate_weight.data && a.dup_weight.data ? 2 * padded : padded;
    p.dweight = shape_of(rows, a.width, a.rows, (int)size, false, true);
    if (p.dweight.splits > 1) p.parts = std::max(p.parts, parts_bytes(rows, a.width, p.dweight.splits));
    p.x = laid_out_bytes(a.x, a.rows, a.width, size);
  }
  p.parts = up(p.parts, 256);
  p.bytes = p.slopes + p.sums + p.sizes + p.parts + p.x + p.gate + p.up;
  return p;
}

template <typename T> void backward(const hctr_gated_grad_args &a) {
  const BackwardPlan plan = plan_of(a);
  const hipStream_t s = (hipStream_t)a.stream;
  const size_t size = sizeof(T), padded = plan.padded;
  char *space = (char *)a.workspace, *slopes = space, *parts = slopes + plan.slopes;
  float *sums = (float *)(parts + plan.parts), *scale = plan.sizes ? (float *)((char *)sums + plan.sums) : nullptr;
  const float *back = scale ? scale + 1 : nullptr;
  space = (char *)sums + plan.sums + plan.sizes;

  GatedSlopes p = {};
  p.dh = a.dh.data, p.gate = a.gate.data, p.up = a.up.data;
  p.dh_stride = a.dh.stride, p.gate_stride = a.gate.stride, p.up_stride = a.up.stride;
  p.slopes = slopes, p.sums = plan.sums ? sums : nullptr;
  p.scale = scale;
  if (scale) {
    // (us of the gradient, 65536 rows through 3328 x 512 twice, slopes of 1e-3: 1748 without a guess, as they are all made twice; 1310 with one.  Where there are
    // few slopes a launch takes longer than making them again.)
    p.guess = (uint64_t)a.rows * a.hidden >= (1u << 22) ? scale + 2 : nullptr;
    p.sizes = scale + 2 + kGuesses;
  }
  p.rows = (uint32_t)a.rows, p.hidden = (uint32_t)a.hidden, p.padded = (uint32_t)padded, p.rows_each = (uint32_t)plan.rows_each;
  p.activation = a.activation;
  if (a.rows) launch_slopes<T>(p, s);
  if (a.dgate_bias || a.dup_bias)
    launch_column_sums({sums, (uint32_t)plan.row_blocks, (uint32_t)(2 * padded), (uint32_t)padded, (uint32_t)a.hidden, nullptr, 1, nullptr, {a.dgate_bias, a.dup_bias}},
                       a.bias_dtype, s);
  const Operand by_row = {{slopes, nullptr}, (int64_t)(2 * padded * size), (uint32_t)a.rows, 0, 0};
  if (a.dx.data && a.rows) {
    ProductArgs q = {};
    q.a = by_row;
    q.b.rows = (uint32_t)a.width, q.b.behind_from = (uint32_t)padded, q.b.behind_k = (uint32_t)a.hidden;
    if (plan.gate) {
      const size_t stride = up(a.width * size, 16);
      for (int i = 0; i < 2; i++) {
        launch_copy_rows<T>(i ? a.up_weight : a.gate_weight, a.hidden, a.width, space, stride, s);
        q.b.base[i] = space;
        space += plan.gate;
      }
      q.b.stride = (int64_t)stride;
    } else {
      q.b.base[0] = (const char *)a.gate_weight.data, q.b.base[1] = (const char *)a.up_weight.data;
      q.b.stride = a.hidden > 1 ? a.gate_weight.stride * (int64_t)size : (int64_t)(a.width * size);
    }
    q.rows = (uint32_t)a.rows, q.columns = (uint32_t)a.width, q.k = (uint32_t)(2 * padded);
    q.splits = plan.dx.splits, q.band = 8;
    q.partial = q.splits > 1 ? (float *)parts : nullptr;
    q.result = {{a.dx.data, nullptr}, {a.dx.stride, 0}, q.rows, q.columns, ~0u, back, nullptr};
    launch_forward_product<T>(q, plan.dx.tile, s);
    if (q.partial) launch_join<T>(q, s);
  }
  if (plan.weights) {
    const bool gate = a.dgate_weight.data, both = gate && a.dup_weight.data;
    ProductArgs q = {};
    q.a = by_row;
    q.a.rows = (uint32_t)(both ? 2 * padded : padded);
    if (!gate) q.a.base[0] += padded * size;
    q.b = operand(laid_out(a.x, a.rows, a.width, a.dtype, space, s), a.width);
    q.rows = q.a.rows, q.columns = (uint32_t)a.width, q.k = (uint32_t)a.rows;
    q.splits = plan.dweight.splits, q.band = 8;
    q.partial = q.splits > 1 ? (float *)parts : nullptr;
    const hctr_matrix &first = gate ? a.dgate_weight : a.dup_weight, &second = a.dup_weight;
    q.result = {{first.data, both ? second.data : nullptr}, {first.stride, second.stride}, (uint32_t)a.hidden, q.columns, (uint32_t)padded, back,
                nullptr};
    launch_across_product<T>(q, plan.dweight.tile, s);
    if (q.partial) launch_join<T>(q, s);
  }
}

void check(const hctr_gated_grad_args &a) {
  check_dtype(a.dtype, "gated linear");
  check_sizes(a.rows, a.width, a.hidden, 1u << 20, "gated linear", "hidden must be in 1..2^20");
  HCTR_CHECK(a.activation >= HCTR_SILU && a.activation <= HCTR_SIGMOID, "gated linear: unknown activation");
  HCTR_CHECK(!(a.dgate_bias || a.dup_bias) || a.bias_dtype == HCTR_F32 || a.bias_dtype == a.dtype, "gated linear: the biases are of the matrices' type or float");
}

} // namespace

size_t gated_linear_workspace(const hctr_gated_args &a) {
  check(a);
  return plan_of(a).bytes;
}
size_t gated_linear_backward_workspace(const hctr_gated_grad_args &a) {
  check(a);
  return plan_of(a).bytes;
}

void gated_linear(const hctr_gated_args &a) {
  check(a);
  if (!a.rows) return;
  check_matrix(a.x, a.rows, a.width, false, "gated linear: x");
  check_matrix(a.gate_weight, a.hidden, a.width, false, "gated linear: gate_weight");
  check_matrix(a.up_weight, a.hidden, a.width, false, "gated linear: up_weight");
  check_matrix(a.h, a.rows, a.hidden, true, "gated linear: h");
  if (a.gate.data) check_matrix(a.gate, a.rows, a.hidden, true, "gated linear: gate");
  if (a.up.data) check_matrix(a.up, a.rows, a.hidden, true, "gated linear: up");
  check_space(a.workspace, a.workspace_bytes, plan_of(a).bytes, "gated linear");
  if (a.dtype == HCTR_F32) forward<float>(a);
  else if (a.dtype == HCTR_BF16) forward<bf16_t>(a);
  else forward<f16_t>(a);
}

void gated_linear_backward(const hctr_gated_grad_args &a) {
  check(a);
  const bool weights = a.dgate_weight.data || a.dup_weight.data;
  if (a.rows) {
    check_matrix(a.dh, a.rows, a.hidden, false, "gated linear: dh");
    check_matrix(a.gate, a.rows, a.hidden, false, "gated linear: gate");
    check_matrix(a.up, a.rows, a.hidden, false, "gated linear: up");
    if (weights) check_matrix(a.x, a.rows, a.width, false, "gated linear: x");
    if (a.dx.data) {
      check_matrix(a.gate_weight, a.hidden, a.width, false, "gated linear: gate_weight");
      check_matrix(a.up_weight, a.hidden, a.width, false, "gated linear: up_weight");
      check_matrix(a.dx, a.rows, a.width, true, "gated linear: dx");
    }
  }
  if (a.dgate_weight.data) check_matrix(a.dgate_weight, a.hidden, a.width, true, "gated linear: dgate_weight");
  if (a.dup_weight.data) check_matrix(a.dup_weight, a.hidden, a.width, true, "gated linear: dup_weight");
  check_space(a.workspace, a.workspace_bytes, plan_of(a).bytes, "gated linear");
  if (a.dtype == HCTR_F32) backward<float>(a);
  else if (a.dtype == HCTR_BF16) backward<bf16_t>(a);
  else backward<f16_t>(a);
}

} // namespace hctr
