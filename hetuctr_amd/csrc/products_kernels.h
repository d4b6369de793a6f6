// The kernels of products.h for one type; products_*.hip build them side by side.
#pragma once
#include "products.h"

namespace hctr {

template <typename T, Lies LA, Lies LB, Second SB, int TILE>
__global__ __launch_bounds__((Product<T, LA, LB, SB, TILE, TILE>::kThreads), (Product<T, LA, LB, SB, TILE, TILE>::kWavesEach)) void product(ProductArgs p) {
  typedef Product<T, LA, LB, SB, TILE, TILE> P;
  __shared__ __attribute__((aligned(1024))) char tiles[P::kLdsBytes];
  // (the tiles of rows that are there are shared out among the XCDs, not those of all rows: 8192 rows of which a quarter takes no part, and 65537
  // items of 4096 values, us 9919 and 9417 for the gradient of their cross entropy)
  const uint32_t rows = p.rows_there ? min(p.rows, *p.rows_there) : p.rows, row_tiles = (rows + TILE - 1) / TILE, live = row_tiles * p.column_tiles;
  if (blockIdx.x >= live) return;
  uint32_t row, column;
  tile_of(blockIdx.x, live, row_tiles, p.column_tiles, p.band, row, column);
  const uint32_t row0 = row * TILE, column0 = column * TILE;
  const uint32_t k = p.k_there ? min(p.k, *p.k_there) : p.k;
  const uint32_t steps = (k + kStep<T> - 1) / kStep<T>, each = (steps + p.splits - 1) / p.splits;
  const uint32_t k0 = blockIdx.y * each * kStep<T>, k1 = min(k, k0 + each * kStep<T>);
  typename P::Sums sum;
  P::run(p.a, p.b, row0, column0, k0, k1, (uint32_t)(uintptr_t)(lds_char *)tiles, sum);
  const uint32_t l = lane_id(), columns = (p.columns + 3) / 4 * 4;
  const float scale = !p.partial && p.result.scale ? *p.result.scale : 1.f;
  if constexpr (sizeof(T) == 2) {
    if (!p.partial) {
      typedef Staged<T, TILE, TILE> S;
      const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)tiles;
      __syncthreads(); // the tiles are read
#pragma unroll
      for (int i = 0; i < P::kRowTiles; i++)
#pragma unroll
        for (int j = 0; j < P::kColumnTiles; j++) S::put(lds, P::wave_row() + i * 16 + l % 16, P::wave_column() + j * 16 + l / 16 * 4, sum[i][j] * scale);
      __syncthreads();
      S::template each<P::kThreads>(lds, [&](uint32_t r, uint32_t c, auto x) {
        if (row0 + r >= rows || column0 + c >= p.columns) return;
        if (T *to = row_of<T>(p.result, row0 + r)) write<8>(to, column0 + c, p.columns, x);
      });
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < P::kRowTiles; i++) {
    const uint32_t r = row0 + P::wave_row() + i * 16 + l % 16;
    if (r >= rows) continue;
    float *part = p.partial + ((uint64_t)blockIdx.y * p.rows + r) * columns;
#pragma unroll
    for (int j = 0; j < P::kColumnTiles; j++) {
      const uint32_t c = column0 + P::wave_column() + j * 16 + l / 16 * 4;
      if (c >= p.columns) continue;
      if (!p.partial) {
        if (T *to = row_of<T>(p.result, r)) write4<T>(to, c, p.columns, sum[i][j] * scale);
      } else {
        f32x4 *to = (f32x4 *)(part + c);
        *to = p.add ? *to + sum[i][j] : sum[i][j];
      }
    }
  }
}

template <typename T> __global__ __launch_bounds__(256) void join_parts(const float *partial, uint32_t splits, uint32_t rows, uint32_t columns, const uint32_t *rows_there, Result result) {
  const uint32_t quads = (columns + 3) / 4, there = rows_there ? min(rows, *rows_there) : rows;
  const float scale = result.scale ? *result.scale : 1.f;
  const uint64_t total = (uint64_t)there * quads, apart = (uint64_t)rows * quads;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const f32x4 *from = (const f32x4 *)partial + i;
    f32x4 sum = from[0];
    for (uint32_t s = 1; s < splits; s++) sum += from[s * apart];
    const uint64_t r = total >> 32 ? i / quads : (uint32_t)i / quads;
    if (T *to = row_of<T>(result, (uint32_t)r)) write4<T>(to, (uint32_t)(i - r * quads) * 4, columns, sum * scale);
  }
}

template <typename T, Lies LA, Lies LB, Second SB> void launch_product(ProductArgs &p, int tile, hipStream_t s) {
  p.row_tiles = div_up(p.rows, tile), p.column_tiles = div_up(p.columns, tile);
  const dim3 blocks(p.row_tiles * p.column_tiles, p.splits), threads(tile_threads(p.row_tiles, p.column_tiles, tile, "product"));
  if (tile == 256) hipLaunchKernelGGL((product<T, LA, LB, SB, 256>), blocks, threads, 0, s, p);
  else if (tile == 128) hipLaunchKernelGGL((product<T, LA, LB, SB, 128>), blocks, threads, 0, s, p);
  else hipLaunchKernelGGL((product<T, LA, LB, SB, 64>), blocks, threads, 0, s, p);
  HCTR_HIP(hipGetLastError());
}
template <typename T> void launch_forward_product(ProductArgs &p, int tile, hipStream_t s) {
  launch_product<T, Lies::kAlong, Lies::kAcross, Second::kBehind>(p, tile, s);
}
template <typename T> void launch_across_product(ProductArgs &p, int tile, hipStream_t s) {
  launch_product<T, Lies::kAcross, Lies::kAcross, Second::kNone>(p, tile, s);
}
template <typename T> void launch_join(const ProductArgs &p, hipStream_t s) {
  const uint64_t quads = (uint64_t)p.rows * ((p.columns + 3) / 4);
  hipLaunchKernelGGL((join_parts<T>), dim3((unsigned)min((quads + 255) / 256, (uint64_t)16384)), dim3(256), 0, s, p.partial, p.splits, p.rows, p.columns, p.rows_there, p.result);
  HCTR_HIP(hipGetLastError());
}

// rows of `width` values, the last piece of 16 bytes filled up with zeros
template <typename T> __global__ __launch_bounds__(256) void copy_rows(const T *from, int64_t from_stride, T *to, int64_t to_stride, uint64_t pieces, uint32_t per_row, uint32_t width) {
  constexpr int V = kVec<T>;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = pieces >> 32 ? i / per_row : (uint32_t)i / per_row;
    const uint32_t c = (uint32_t)(i - r * per_row) * V;
    *(typename Packed<T, V>::type *)(to + (int64_t)r * to_stride + c) = settled<V, Rows::kLong>(load_raw<V, Rows::kLong>(from + (int64_t)r * from_stride, c, width), c, width);
  }
}
template <typename T> void launch_copy_rows(const hctr_matrix &m, size_t rows, size_t width, char *to, size_t to_stride, hipStream_t s) {
  const uint32_t per_row = div_up(width, kVec<T>);
  const uint64_t pieces = (uint64_t)rows * per_row;
  hipLaunchKernelGGL((copy_rows<T>), dim3((unsigned)std::min<uint64_t>((pieces + 255) / 256, 1u << 20)), dim3(256), 0, s, (const T *)m.data, m.stride, (T *)to,
                     (int64_t)(to_stride / sizeof(T)), pieces, per_row, (uint32_t)width);
  HCTR_HIP(hipGetLastError());
}

} // namespace hctr
