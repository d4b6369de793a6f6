// The choice of tiles for a product, matrices laid out for tiles, sums over rows.
#include <algorithm>

#include "products.h"

namespace hctr {

// The tile and the number of parts along k that a product should take least time with.  Of each tile up to `most` share a CU, and take
// us[n - 1] for a step of 128 bytes of k while n of them do; every tile costs what it takes to begin and to end.  Parts are written and
// read again as floats, by a launch more.
Shape shape_of(size_t rows, size_t columns, size_t k, int size, bool paired, bool may_split) {
  struct Kind {
    int tile, most;
    double us[2];
  };
  static constexpr Kind kNarrowTypes[] = {{256, 1, {1.8}}, {128, 2, {0.8, 1.05}}, {64, 2, {0.4, 0.5}}};
  static constexpr Kind kFloats[] = {{256, 1, {5.9}}, {128, 2, {1.95, 3.2}}, {64, 2, {1.15, 1.25}}};
  const double ends = 4.0;
  const size_t cus = 256, steps = (k * size + kStepBytes - 1) / kStepBytes, wide = paired ? 2 * columns : columns;
  Shape best = {128, 1};
  double least = 1e30;
  for (const Kind &kind : size == 2 ? kNarrowTypes : kFloats) {
    const size_t tiles = ((rows + kind.tile - 1) / kind.tile) * ((wide + kind.tile - 1) / kind.tile);
    for (uint32_t splits = 1; splits <= (may_split ? 32u : 1u) && (splits == 1 || steps / splits >= 4); splits++) {
      const size_t each = (steps + splits - 1) / splits, turns = (tiles * splits + cus - 1) / cus; // tiles that a CU has to do
      double t = turns / kind.most * (each * kind.us[kind.most - 1] + ends);
      if (turns % kind.most) t += each * kind.us[turns % kind.most - 1] + ends;
      if (splits > 1) t += 4.0 + 0.5e-6 * parts_bytes(rows, wide, splits);
      if (t < least) least = t, best = {kind.tile, splits};
    }
  }
  return best;
}

Layout laid_out(const hctr_matrix &m, size_t rows, size_t width, int dtype, char *&space, hipStream_t s) {
  const size_t size = size_of(dtype);
  if (!rows || fits(m, rows, width, size)) return {(const char *)m.data, rows > 1 ? m.stride * (int64_t)size : (int64_t)(width * size)};
  const size_t stride = up(width * size, 16);
  const Layout l = {space, (int64_t)stride};
  if (dtype == HCTR_F32) launch_copy_rows<float>(m, rows, width, space, stride, s);
  else if (dtype == HCTR_BF16) launch_copy_rows<bf16_t>(m, rows, width, space, stride, s);
  else launch_copy_rows<f16_t>(m, rows, width, space, stride, s);
  space += laid_out_bytes(m, rows, width, size);
  return l;
}

namespace {

// 16 neighbouring columns per block, whose threads share out the rows, eight loads under way, and join their sums through LDS, in
// an order that depends on the sizes alone.
constexpr int kSumThreads = 512, kSumColumns = 16;
template <typename W> __global__ __launch_bounds__(kSumThreads) void column_sums(ColumnSums p) {
  constexpr uint32_t ROWS = kSumThreads / kSumColumns, LOADS = 8;
  __shared__ float sums[ROWS][kSumColumns + 1];
  const uint32_t x = threadIdx.x % kSumColumns, y = threadIdx.x / kSumColumns, c = blockIdx.x * kSumColumns + x;
  const uint32_t rows = p.rows_there ? min(p.rows, (*p.rows_there + p.per - 1) / p.per) : p.rows;
  float sum = 0.f;
  for (uint32_t i = y; i < rows; i += ROWS * LOADS) {
    float v[LOADS];
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) v[k] = c < p.columns && i + k * ROWS < rows ? p.partial[(uint64_t)(i + k * ROWS) * p.columns + c] : 0.f;
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) sum += v[k];
  }
  sums[y][x] = sum;
  __syncthreads();
  if (y || c >= p.columns) return;
  sum = 0.f;
#pragma unroll
  for (uint32_t i = 0; i < ROWS; i++) sum += sums[i][x];
  if (p.scale) sum *= *p.scale;
  const bool second = c >= p.second_from;
  const uint32_t at = c - (second ? p.second_from : 0);
  W *to = (W *)(second ? p.out[1] : p.out[0]);
  if (to && at < p.count) to[at] = (W)sum;
}

// few rows: a thread per column
template <typename W> __global__ __launch_bounds__(256) void few_sums(ColumnSums p) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.columns) return;
  const uint32_t rows = p.rows_there ? min(p.rows, (*p.rows_there + p.per - 1) / p.per) : p.rows;
  float sum = 0.f;
  for (uint32_t i = 0; i < rows; i++) sum += p.partial[(uint64_t)i * p.columns + c];
  if (p.scale) sum *= *p.scale;
  const bool second = c >= p.second_from;
  const uint32_t at = c - (second ? p.second_from : 0);
  W *to = (W *)(second ? p.out[1] : p.out[0]);
  if (to && at < p.count) to[at] = (W)sum;
}

} // namespace

void launch_column_sums(const ColumnSums &c, int dtype, hipStream_t s) {
  if (c.rows <= 4) {
    const dim3 blocks(div_up(c.columns, 256)), threads(256);
    if (dtype == HCTR_F32) hipLaunchKernelGGL((few_sums<float>), blocks, threads, 0, s, c);
    else if (dtype == HCTR_BF16) hipLaunchKernelGGL((few_sums<bf16_t>), blocks, threads, 0, s, c);
    else hipLaunchKernelGGL((few_sums<f16_t>), blocks, threads, 0, s, c);
    HCTR_HIP(hipGetLastError());
    return;
  }
  const dim3 blocks(div_up(c.columns, kSumColumns)), threads(kSumThreads);
  if (dtype == HCTR_F32) hipLaunchKernelGGL((column_sums<float>), blocks, threads, 0, s, c);
  else if (dtype == HCTR_BF16) hipLaunchKernelGGL((column_sums<bf16_t>), blocks, threads, 0, s, c);
  else hipLaunchKernelGGL((column_sums<f16_t>), blocks, threads, 0, s, c);
  HCTR_HIP(hipGetLastError());
}

} // namespace hctr
