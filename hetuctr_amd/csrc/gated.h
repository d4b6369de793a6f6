// The gated linear layer, h = f(x gate^T) * (x up^T), and its gradient.
#pragma once
#include "products.h"

namespace hctr {

struct GatedForward {
  Operand x, weights; // the weights paired
  const void *loose_x, *loose_gate, *loose_up; // of few rows: as they are given, strides in elements
  int64_t loose_stride, loose_gate_stride, loose_up_stride;
  uint32_t rows, width, hidden, row_tiles, column_tiles, band, splits;
  float *partial; // [split][rows][2 * hidden, up to multiples of 4 each], or null
  const void *gate_bias, *up_bias;
  bool narrow; // the biases are of the matrices' type
  int activation;
  void *h, *gate, *up; // gate, up: may be null
  int64_t h_stride, gate_stride, up_stride;
};
template <typename T> void launch_gated(GatedForward &p, int tile, hipStream_t s);
template <typename T> void launch_gated_few(const GatedForward &p, hipStream_t s);

struct GatedSlopes {
  const void *dh, *gate, *up;
  int64_t dh_stride, gate_stride, up_stride;
  void *slopes;         // [rows][2 * padded]: dgate, dup, zeros behind each
  float *sums;          // [blocks][2 * padded] sums over a block's rows, or null
  float *sizes;         // half: [blocks along the rows][blocks along the columns] the largest |dgate|, |dup|; or null: not scaled
  float *guess;         // half: [kGuesses] the largest that some blocks found in some of the rows; or null: they are not scaled at first
  float *scale;         // half: [2] what dgate and dup were multiplied by before they were rounded, and 1 / that
  uint32_t rows, hidden, padded, rows_each; // rows of a block
  int activation;
};
constexpr uint32_t kGuesses = 256;
inline uint32_t slope_columns(int size) { return 32 * (16 / size); } // of a block
template <typename T> void launch_slopes(const GatedSlopes &p, hipStream_t s);

// The entry points of the C ABI behind their guard
void gated_linear(const hctr_gated_args &a);
void gated_linear_backward(const hctr_gated_grad_args &a);
size_t gated_linear_workspace(const hctr_gated_args &a);
size_t gated_linear_backward_workspace(const hctr_gated_grad_args &a);

} // namespace hctr
