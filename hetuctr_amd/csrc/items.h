// Softmax cross entropy of x weight^T + bias over many items, and its gradient.
#pragma once
#include "products.h"

namespace hctr {

// What is known of the rows that take part, which are numbered anew, in their order, and of the items; all in device memory
struct Taken {
  uint32_t *count;
  float *scale;       // [2]: what d is multiplied by before it is rounded to 16 bits, and 1 / that
  uint32_t *row_of;   // [rows] where each one lies among all rows
  uint32_t *target;   // its item; kNoItem: that is none
  float *dloss, *lse; // of the gradient
  float *hits;        // of the forward pass, in lse's place: a row's logit of its target, in units of log 2
  float *bias;        // [items] in units of log 2
};
constexpr uint32_t kNoItem = 0xffffffffu;
// behind the last row of `target`, `dloss` and `lse` (kNoItem, 0, infinity) and the last item of `bias` (-infinity) follow what makes d zero,
// up to the next multiple of
constexpr uint32_t kFilled = 256;

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
  const void *bias;
  bool narrow; // the bias is of the matrices' type
};
constexpr uint32_t kChunk = 1024;
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
  uint32_t column_from, columns_here; // the tiles of a launch (few rows: from where on)
  Taken taken;
  float2 *parts; // forward: [column tiles][rows]: the largest logit and the sum of exponentials less it, both in units of log 2
  void *d;       // gradient: [rows][d_stride]
  uint32_t d_stride;
  float *sums;   // [row tiles][d_stride] sums over a tile's rows, or null
};
template <typename T> void launch_items_forward(ItemsProduct &p, int tile, hipStream_t s);  // tile 0: few rows
template <typename T> void launch_items_gradient(ItemsProduct &p, int tile, hipStream_t s);
// Narrow matrices of 16-bit values: rows of up to kNarrow columns.  A block owns rows of one matrix, whose values it keeps in registers, and
// goes through a range of the rows of the other.
constexpr size_t kNarrow = 128;
// Blocks that share a CU: three where the registers hold them (us, 4096 rows, a million items: forward of 64 columns 955 -> 889, of 32
// 844 -> 777, dx of 32 985 -> 895, the weights' gradient 987 -> 985; forward of 128 would spill, 1373 -> 1403).
constexpr int narrow_share(size_t width, bool gradient) { return width <= 64 && (!gradient || width <= 32) ? 3 : 2; }
struct ItemsNarrow {
  const char *x, *weight;
  int64_t x_stride, weight_stride; // bytes
  uint32_t rows, width, items;
  Taken taken;
  uint32_t ranges, owners; // blocks along the rows that are gone through, and along those that are owned
  float2 *parts;           // forward: [range][rows]
  float *partial;          // gradient: [range][owned rows][width up to a multiple of 4], or null: to `result`
  Result result;
  float *sums; // of the weight's gradient: [range][items] sums over the rows, or null
};
uint32_t narrow_ranges(size_t owned, size_t through, size_t width, bool gradient);
template <typename T> void launch_narrow_forward(ItemsNarrow &p, hipStream_t s);
template <typename T> void launch_narrow_dx(ItemsNarrow &p, hipStream_t s);
template <typename T> void launch_narrow_dweight(ItemsNarrow &p, hipStream_t s);

// The entry points of the C ABI behind their guard
void linear_cross_entropy(const hctr_items_args &a);
void linear_cross_entropy_backward(const hctr_items_grad_args &a);
size_t linear_cross_entropy_workspace(const hctr_items_args &a);
size_t linear_cross_entropy_backward_workspace(const hctr_items_grad_args &a);

} // namespace hctr
