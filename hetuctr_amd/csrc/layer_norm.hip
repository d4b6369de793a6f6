// Layer normalisation and its gradient: argument checks, the choice of the kernels, the sums of the weight's gradient.
#include "layer_norm.h"

#include <algorithm>

namespace hctr {
namespace {

// The blocks' rows of sums (dweight's columns, then dbias's), added up: COLUMNS neighbouring columns per block, whose threads share
// out the rows and join their sums through LDS, in an order that depends on nothing but the sizes.  A thread has eight loads under
// way: what it waits for is the memory, the rows having been written by other XCDs.  With few columns a block takes 16 of them,
// to have more threads per column; with many 32, whole cache lines.  4 to 5 us, of which the launch and two trips to memory are most:
// us with 32, 16 and 8 columns, 768 rows of 2 x 128 5.0, 4.1, 3.9; 1024 of 2 x 37 5.0, 4.3, 4.7; 256 of 2 x 8192 4.6, 7.2, 12.5.
constexpr int kSumThreads = 1024;
template <typename W, int COLUMNS>
__global__ __launch_bounds__(kSumThreads) void sum_partial(const float *__restrict__ partial, uint32_t blocks, uint32_t width, W *dweight, W *dbias) {
  constexpr uint32_t ROWS = kSumThreads / COLUMNS, LOADS = 8;
  __shared__ float sums[ROWS][COLUMNS + 1];
  const uint32_t x = threadIdx.x % COLUMNS, y = threadIdx.x / COLUMNS;
  const uint64_t c = (uint64_t)blockIdx.x * COLUMNS + x, columns = 2 * (uint64_t)width;
  float sum = 0.f;
  for (uint32_t i = y; i < blocks; i += ROWS * LOADS) {
    float v[LOADS];
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) v[k] = c < columns && i + k * ROWS < blocks ? partial[(i + k * ROWS) * columns + c] : 0.f;
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) sum += v[k];
  }
  sums[y][x] = sum;
  __syncthreads();
  if (y || c >= columns) return;
  sum = 0.f;
#pragma unroll
  for (uint32_t i = 0; i < ROWS; i++) sum += sums[i][x];
  if (c < width) {
    if (dweight) dweight[c] = (W)sum;
  } else if (dbias) {
    dbias[c - width] = (W)sum;
  }
}

template <typename W> void launch_sum(const hctr_norm_grad_args &a, unsigned blocks, hipStream_t s) {
  const auto launch = [&](auto kernel, unsigned columns) {
    hipLaunchKernelGGL(kernel, dim3(div_up(2 * a.width, columns)), dim3(kSumThreads), 0, s, (const float *)a.workspace, blocks, (uint32_t)a.width,
                       (W *)a.dweight, (W *)a.dbias);
  };
  if (a.width <= 2048) launch(sum_partial<W, 16>, 16);
  else launch(sum_partial<W, 32>, 32);
  HCTR_HIP(hipGetLastError());
}

} // namespace

// Few rows: weight and bias get blocks of their own, one launch does it all, and no workspace is needed.  A call's time in us with
// two launches and with one, dropped (the draws, made again for every column, are what many rows cost): 128 columns, 1 to 512
// rows 11.0, 6.8, 1024 rows 11.1, 10.3, 2048 rows 11.0, 18.3; 1024 columns, 512 rows 11.0, 6.9, 1024 rows 11.1, 18.2; 4096 columns,
// 128 rows 11.1, 6.9, 512 rows 11.6, 20.7; 16384 columns, 1 row 10.8, 26.8.
static bool few(size_t rows, size_t width) { return rows <= 512 && width <= 4096 && rows * width <= (1u << 19); }

// The most that norm_grad_blocks says for any form and pair of types.
size_t layer_norm_workspace(size_t rows, size_t width) {
  if (!rows || !width || width >= (1u << 31) || few(rows, width)) return 0;
  const uint32_t w = (uint32_t)width;
  return (size_t)std::max(norm_grad_blocks(rows, w, kVec<float>, 6), norm_grad_blocks(rows, w, kVec<bf16_t>, 4)) * 2 * width * sizeof(float);
}

void check_types(int stream, int act, int affine, bool has_affine) {
  const auto known = [](int t) { return t == HCTR_F32 || t == HCTR_BF16 || t == HCTR_F16; };
  HCTR_CHECK(known(stream) && known(act), "layer norm: unknown type");
  HCTR_CHECK(stream == act || stream == HCTR_F32, "layer norm: what is normalised is of the activations' type or float");
  HCTR_CHECK(!has_affine || affine == HCTR_F32 || affine == act, "layer norm: weight and bias are of the activations' type or float");
}

void layer_norm(const hctr_norm_args &a, bool add) {
  HCTR_CHECK(a.width >= 1 && a.width < (1u << 31), "layer norm: the width must be in 1..2^31 - 1");
  HCTR_CHECK(a.eps >= 0.f, "layer norm: eps must not be negative");
  check_types(a.stream_dtype, a.act_dtype, a.affine_dtype, a.weight || a.bias);
  NormForward p = {};
  const bool on = make_dropping(a.drop, a.width, p.drop);
  if (!a.rows) return;
  check_matrix(a.x, a.rows, a.width, false, "layer norm: x");
  check_matrix(a.y, a.rows, a.width, true, "layer norm: y");
  if (add) {
    check_matrix(a.residual, a.rows, a.width, false, "layer norm: residual");
    check_matrix(a.sum, a.rows, a.width, true, "layer norm: sum");
  }
  p.rows = a.rows;
  p.width = (uint32_t)a.width;
  p.eps = a.eps;
  p.inv_width = (float)(1.0 / (double)a.width);
  p.x = a.x.data, p.x_stride = a.x.stride;
  p.y = a.y.data, p.y_stride = a.y.stride;
  if (add) {
    p.residual = a.residual.data, p.residual_stride = a.residual.stride;
    p.sum = a.sum.data, p.sum_stride = a.sum.stride;
  }
  p.weight = a.weight, p.bias = a.bias;
  p.narrow = a.affine_dtype != HCTR_F32;
  p.mean = a.mean, p.rstd = a.rstd;
  const hipStream_t s = (hipStream_t)a.stream;
  if (a.stream_dtype == HCTR_BF16) launch_norm<bf16_t, bf16_t>(p, add, on, s);
  else if (a.stream_dtype == HCTR_F16) launch_norm<f16_t, f16_t>(p, add, on, s);
  else if (a.act_dtype == HCTR_BF16) launch_norm<float, bf16_t>(p, add, on, s);
  else if (a.act_dtype == HCTR_F16) launch_norm<float, f16_t>(p, add, on, s);
  else launch_norm<float, float>(p, add, on, s);
}

void layer_norm_backward(const hctr_norm_grad_args &a, bool add) {
  HCTR_CHECK(a.width >= 1 && a.width < (1u << 31), "layer norm: the width must be in 1..2^31 - 1");
  const bool columns = a.dweight || a.dbias;
  check_types(a.stream_dtype, a.act_dtype, a.affine_dtype, a.weight || columns);
  NormBackward p = {};
  const bool on = make_dropping(a.drop, a.width, p.drop);
  const hipStream_t s = (hipStream_t)a.stream;
  if (a.rows) {
    check_matrix(a.dy, a.rows, a.width, false, "layer norm: dy");
    check_matrix(a.s, a.rows, a.width, false, "layer norm: s");
    HCTR_CHECK(a.mean && a.rstd, "layer norm: mean and rstd of the forward pass are needed");
    if (!add || a.dx.data) check_matrix(a.dx, a.rows, a.width, true, "layer norm: dx");
    if (add && a.dresidual.data) check_matrix(a.dresidual, a.rows, a.width, true, "layer norm: dresidual");
    HCTR_CHECK(!columns || few(a.rows, a.width) || (a.workspace && (uintptr_t)a.workspace % 16 == 0 && a.workspace_bytes >= layer_norm_workspace(a.rows, a.width)),
               "layer norm: the workspace is missing, too small or not 16-byte aligned");
  }
  p.rows = a.rows;
  p.width = (uint32_t)a.width;
  p.inv_width = (float)(1.0 / (double)a.width);
  p.dy = a.dy.data, p.dy_stride = a.dy.stride;
  p.s = a.s.data, p.s_stride = a.s.stride;
  p.dx = a.dx.data, p.dx_stride = a.dx.stride;
  if (add) {
    p.ds = a.dsum.data, p.ds_stride = a.dsum.stride;
    p.dresidual = a.dresidual.data, p.dresidual_stride = a.dresidual.stride;
  }
  p.mean = a.mean, p.rstd = a.rstd;
  p.weight = a.weight;
  p.narrow = a.affine_dtype != HCTR_F32;
  const bool alone = columns && a.rows && few(a.rows, a.width); // one launch does it all
  if (alone) p.dweight = a.dweight, p.dbias = a.dbias;
  else if (columns) p.partial = (float *)a.workspace;
  unsigned blocks = 0;
  if (a.rows) {
    if (a.stream_dtype == HCTR_BF16) blocks = launch_norm_grad<bf16_t, bf16_t>(p, add, on, s);
    else if (a.stream_dtype == HCTR_F16) blocks = launch_norm_grad<f16_t, f16_t>(p, add, on, s);
    else if (a.act_dtype == HCTR_BF16) blocks = launch_norm_grad<float, bf16_t>(p, add, on, s);
    else if (a.act_dtype == HCTR_F16) blocks = launch_norm_grad<float, f16_t>(p, add, on, s);
    else blocks = launch_norm_grad<float, float>(p, add, on, s);
  }
  if (!columns || alone) return;
  if (a.affine_dtype == HCTR_F32) launch_sum<float>(a, blocks, s);
  else if (a.affine_dtype == HCTR_BF16) launch_sum<bf16_t>(a, blocks, s);
  else launch_sum<f16_t>(a, blocks, s);
}

} // namespace hctr
