// Softmax cross entropy of x weight^T + bias over many items, and its gradient.
#pragma once
#include "products.h"

namespace hctr {

// What is known of the rows that take part, which are numbered anew, in their order; all in device memory
struct Taken {
  uint32_t *count;
  float *scale;      // [2]: what d is multiplied by before it is rounded to 16 bits, and 1 / that
  uint32_t *row_of;  // [rows] where each one lies among all rows
  uint32_t *target;  // its item; kNoItem: that is none
  float *dloss, *lse; // of the gradient
};
constexpr uint32_t kNoItem = 0xffffffffu;

// Rows that take part are copied, with what belongs to them, in whole pieces of 16 bytes; the results of the others are set to zero.
struct TakeRows {
  const void *x;
  int64_t x_stride;
  const int64_t *target;
  int64_t ignored;
  uint32_t rows, width, items;
  const uint2 *chunks; // [chunks of kChunk rows]: how many take part, and the largest |dloss|; or null: there is one chunk
  void *to;            // x of those that take part
  uint32_t to_stride;  // elements
  Taken taken;
  const float *dloss, *lse_in; // gradient
  float *loss, *lse;           // forward; may be null
  void *dx;                    // gradient; may be null
  int64_t dx_stride;
  bool scaled;
};
constexpr uint32_t kChunk = 1024;
void launch_count_rows(const int64_t *target, int64_t ignored, const float *dloss, uint32_t rows, uint2 *chunks, hipStream_t s);
template <typename T> void launch_take_rows(const TakeRows &p, hipStream_t s);

// The logits of a tile, and what becomes of them
struct ItemsProduct {
  Operand x, weight;
  const void *loose_weight; // of few rows: as it is given, stride in elements
  int64_t loose_stride;
  const void *few_x;
  uint32_t few_stride;
  uint32_t rows, width, items, first; // items first .. first + items - 1 of all
  uint32_t row_tiles, column_tiles, band;
  const void *bias; // of item `first`
  bool narrow;
  Taken taken;
  float2 *parts; // forward: [column tiles][rows]: the largest logit and the sum of exponentials less it
  float *hit;    // [rows] the target's logit
  void *d;       // gradient: [rows][d_stride]
  uint32_t d_stride;
  float *sums;   // [row tiles][d_stride] sums over a tile's rows, or null
};
template <typename T> void launch_items_forward(ItemsProduct &p, int tile, hipStream_t s);  // tile 0: few rows
template <typename T> void launch_items_gradient(ItemsProduct &p, int tile, hipStream_t s);
constexpr int kFewItems = 32; // a tile's items where rows are few

// The entry points of the C ABI behind their guard
void linear_cross_entropy(const hctr_items_args &a);
void linear_cross_entropy_backward(const hctr_items_grad_args &a);
size_t linear_cross_entropy_workspace(const hctr_items_args &a);
size_t linear_cross_entropy_backward_workspace(const hctr_items_grad_args &a);

} // namespace hctr
