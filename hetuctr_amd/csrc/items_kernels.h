// The kernels of items.h for one type; items_*.hip build them side by side.
#pragma once
#include <algorithm>

#include "few_rows.h"
#include "items.h"
#include "items_tail.h"
#include "launch_cut.h"

namespace hctr {

// logits of N times four items
template <int N> __device__ __forceinline__ Tail tail_of(const f32x4 (&v)[N]) {
  float most = kLowest;
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int e = 0; e < 4; e += 2) most = fmaxf(fmaxf(most, v[j][e]), v[j][e + 1]);
  Tail t = {most, 0.f};
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int e = 0; e < 4; e++) t.sum += __builtin_amdgcn_exp2f(v[j][e] - most);
  return t; // (a NaN is not the largest, but makes the sum one)
}

__device__ __forceinline__ f32x4 bias4(const ItemsProduct &p, uint32_t c) { return *(const f32x4 *)(p.taken.bias + p.first + c); }
__device__ __forceinline__ f32x4 logit4(f32x4 sum, f32x4 bias) {
#pragma unroll
  for (int e = 0; e < 4; e++) sum[e] = __builtin_fmaf(sum[e], kLog2E, bias[e]);
  return sum;
}

// d of a row's item, before the target's part; the sum over k less lse is rounded once, whatever the two are
__device__ __forceinline__ float chance(float sum, float lse, float bias) { return __builtin_amdgcn_exp2f(__builtin_fmaf(sum - lse, kLog2E, bias)); }
__device__ __forceinline__ f32x4 slope4(f32x4 sum, f32x4 bias, float lse, float scale, uint32_t hit) {
  f32x4 d;
#pragma unroll
  for (int e = 0; e < 4; e++) d[e] = (chance(sum[e], lse, bias[e]) - (hit == (uint32_t)e ? 1.f : 0.f)) * scale;
  return d;
}

// A tile of logits.  Forward: the rows' tails over the tile's items, in registers, then over the lanes that share a row, then over the waves.
// Gradient: d, rounded to the type, since the matrix cores take both operands of the products behind it in one, and its sums over the tile's
// rows for the bias, from before that.  An exponential and four to six instructions a logit stand behind
// width / 32 products of 16 x 16 x 32: from some hundred columns on the matrix cores bound it (6144 rows and 65537 items of 4096 bfloat16:
// gradient 3.1 ms, 1.06 PFLOP/s).
template <typename T, int TILE, bool GRADIENT>
__global__ __launch_bounds__((Product<T, Lies::kAlong, Lies::kAlong, Second::kNone, TILE, TILE>::kThreads), (Product<T, Lies::kAlong, Lies::kAlong, Second::kNone, TILE, TILE>::kWavesEach)) void items_product(ItemsProduct p) {
  typedef Product<T, Lies::kAlong, Lies::kAlong, Second::kNone, TILE, TILE> P;
  __shared__ __attribute__((aligned(1024))) char tiles[P::kLdsBytes];
  // (the tiles of rows that are there are shared out among the XCDs, not those of all rows)
  const uint32_t rows = *p.taken.count, row_tiles = (rows + TILE - 1) / TILE, live = row_tiles * p.columns_here;
  if (blockIdx.x >= live) return;
  uint32_t row, column;
  tile_of(blockIdx.x, live, row_tiles, p.columns_here, p.band, row, column);
  column += p.column_from;
  const uint32_t row0 = row * TILE, column0 = column * TILE;
  typename P::Sums sum;
  P::run(p.x, p.weight, row0, column0, 0, p.width, (uint32_t)(uintptr_t)(lds_char *)tiles, sum);
  const uint32_t l = lane_id(), wave_column = P::wave_column();
  f32x4 bias[P::kColumnTiles];
#pragma unroll
  for (int j = 0; j < P::kColumnTiles; j++) bias[j] = bias4(p, column0 + wave_column + j * 16 + l / 16 * 4);
  __syncthreads(); // the tiles are read
  if constexpr (!GRADIENT) {
    constexpr int ACROSS = TILE / 64;
    Tail *tails = (Tail *)tiles; // [ACROSS][TILE]
    // (all loaded before any hit is written, which might change them for all that the compiler knows)
    uint32_t aims[P::kRowTiles]; // the targets' places among the wave's columns
#pragma unroll
    for (int i = 0; i < P::kRowTiles; i++) {
      const uint32_t r = row0 + P::wave_row() + i * 16 + l % 16;
      aims[i] = (r < rows ? p.taken.target[r] : kNoItem) - (column0 + wave_column);
    }
#pragma unroll
    for (int i = 0; i < P::kRowTiles; i++) {
      const uint32_t in = P::wave_row() + i * 16 + l % 16;
#pragma unroll
      for (int j = 0; j < P::kColumnTiles; j++) sum[i][j] = logit4(sum[i][j], bias[j]);
      Tail t = tail_of(sum[i]);
      t = join_lanes(t, 16);
      t = join_lanes(t, 32);
      if (l < 16) tails[wave_column / 64 * TILE + in] = t;
      const uint32_t aim = aims[i];
      if (__ballot(aim < 64))
#pragma unroll
        for (int j = 0; j < P::kColumnTiles; j++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (aim == j * 16 + l / 16 * 4 + e) p.taken.hits[row0 + in] = sum[i][j][e];
    }
    __syncthreads();
    const uint32_t r = threadIdx.x;
    if (r < TILE && row0 + r < rows) {
      Tail t = tails[r];
#pragma unroll
      for (int w = 1; w < ACROSS; w++) t = join(t, tails[w * TILE + r]);
      p.parts[(uint64_t)column * p.rows + row0 + r] = make_float2(t.most, t.sum);
    }
  } else {
    const float scale = p.taken.scale[0];
    f32x4 down[P::kColumnTiles] = {};
    typedef std::conditional_t<sizeof(T) == 2, T, bf16_t> Narrow; // (floats are not staged)
    typedef Staged<Narrow, TILE, TILE> S;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)tiles;
#pragma unroll
    for (int i = 0; i < P::kRowTiles; i++) {
      const uint32_t in = P::wave_row() + i * 16 + l % 16, r = row0 + in;
      const bool there = r < rows;
      const float lse = there ? p.taken.lse[r] : 0.f, dloss = there ? p.taken.dloss[r] * scale : 0.f;
      const uint32_t target = there ? p.taken.target[r] - p.first : kNoItem;
#pragma unroll
      for (int j = 0; j < P::kColumnTiles; j++) {
        const uint32_t c = wave_column + j * 16 + l / 16 * 4;
        const f32x4 d = slope4(sum[i][j], bias[j], lse, dloss, target - (column0 + c));
        if (there) down[j] += d;
        if constexpr (sizeof(T) == 2) S::put(lds, in, c, d);
        else if (there && column0 + c < p.d_stride) write4<T>((T *)p.d + (uint64_t)r * p.d_stride, column0 + c, p.d_stride, d);
      }
    }
    if constexpr (sizeof(T) == 2) {
      __syncthreads();
      S::template each<P::kThreads>(lds, [&](uint32_t r, uint32_t c, auto x) {
        if (row0 + r < rows && column0 + c < p.d_stride) *(typename Packed<T, 8>::type *)((T *)p.d + (uint64_t)(row0 + r) * p.d_stride + column0 + c) = x;
      });
      if (p.sums) __syncthreads(); // the staged tile is read
    }
    if (p.sums) {
      f32x4 *joined = (f32x4 *)tiles; // [2][TILE / 4]
#pragma unroll
      for (int j = 0; j < P::kColumnTiles; j++) {
#pragma unroll
        for (int mask = 1; mask < 16; mask *= 2)
#pragma unroll
          for (int e = 0; e < 4; e++) down[j][e] += __shfl_xor(down[j][e], mask);
        if (l % 16 == 0) joined[(P::wave_row() ? TILE / 4 : 0) + (wave_column + j * 16) / 4 + l / 16] = down[j];
      }
      __syncthreads();
      const uint32_t c = threadIdx.x * 4;
      if (c < TILE && column0 + c < p.d_stride) *(f32x4 *)(p.sums + (uint64_t)row * p.d_stride + column0 + c) = joined[c / 4] + joined[TILE / 4 + c / 4];
    }
  }
}

template <typename T, int ROWS, int GROUPS, bool GRADIENT> __global__ __launch_bounds__((FewRows<T, ROWS, GROUPS>::kThreads)) void items_few(ItemsProduct p) {
  typedef FewRows<T, ROWS, GROUPS> F;
  constexpr uint32_t QUADS = F::kWeights / 4; // of a row
  __shared__ typename F::Sums sums[F::kSums];
  const uint32_t count = *p.taken.count, row0 = blockIdx.y * ROWS, column = p.column_from + blockIdx.x, column0 = column * F::kWeights;
  if (row0 >= count) return;
  const uint32_t rows = min(count - row0, (uint32_t)ROWS);
  const T *groups[F::kGroups];
  uint32_t left[F::kGroups];
  int64_t stride[F::kGroups];
#pragma unroll
  for (uint32_t j = 0; j < F::kGroups; j++) {
    const uint32_t c = min(column0 + j * 16, p.items - 1); // (behind the last item: that one again)
    groups[j] = (const T *)p.loose_weight + (int64_t)c * p.loose_stride;
    stride[j] = p.loose_stride;
    left[j] = p.items - c;
  }
  F::run((const T *)p.few_x + (uint64_t)row0 * p.few_stride, p.few_stride, rows, groups, left, stride, p.width, sums);
  // four items of a row a thread; the threads of a row are neighbours
  for (uint32_t t = threadIdx.x; t < ROWS * QUADS; t += F::kThreads) {
    const uint32_t r = t / QUADS, c = t % QUADS * 4;
    const f32x4 sum = *(const f32x4 *)&sums[0][r][c], bias = column0 + c < p.items ? bias4(p, column0 + c) : f32x4{-kInfinity, -kInfinity, -kInfinity, -kInfinity};
    if constexpr (!GRADIENT) {
      const f32x4 logit[1] = {logit4(sum, bias)};
      Tail tail = tail_of(logit);
#pragma unroll
      for (uint32_t mask = 1; mask < QUADS; mask *= 2) tail = join_lanes(tail, mask);
      if (c == 0 && r < rows) p.parts[(uint64_t)column * p.rows + row0 + r] = make_float2(tail.most, tail.sum);
      const uint32_t aim = (r < rows ? p.taken.target[row0 + r] : kNoItem) - (column0 + c);
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (aim == (uint32_t)e) p.taken.hits[row0 + r] = logit[0][e];
    } else {
      f32x4 d = {};
      if (r < rows) {
        d = slope4(sum, bias, p.taken.lse[row0 + r], p.taken.dloss[row0 + r] * p.taken.scale[0], p.taken.target[row0 + r] - p.first - (column0 + c));
        if (column0 + c < p.d_stride) write4<T>((T *)p.d + (uint64_t)(row0 + r) * p.d_stride, column0 + c, p.d_stride, d);
      }
      *(f32x4 *)&sums[0][r][c] = d;
    }
  }
  if (GRADIENT && p.sums) {
    __syncthreads();
    const uint32_t c = threadIdx.x * 4;
    if (c < F::kWeights && column0 + c < p.d_stride) {
      f32x4 all = {};
      for (uint32_t i = 0; i < rows; i++) all += *(const f32x4 *)&sums[0][i][c];
      *(f32x4 *)(p.sums + (uint64_t)blockIdx.y * p.d_stride + column0 + c) = all;
    }
  }
}

template <typename T, bool GRADIENT> void launch_items(ItemsProduct &p, int tile, hipStream_t s) {
  if (!tile) {
    const auto launch = [&](auto kernel, uint32_t rows, int groups) {
      p.column_tiles = div_up(p.items, 16 * groups);
      const uint32_t threads = FewRows<T, 16, 2>::kThreads, most = most_blocks(threads);
      for (p.column_from = 0; p.column_from < p.column_tiles; p.column_from += most) {
        hipLaunchKernelGGL(kernel, dim3(std::min(p.column_tiles - p.column_from, most), div_up(p.rows, rows)), dim3(threads), 0, s, p);
        HCTR_HIP(hipGetLastError());
      }
    };
    if (few_groups(p.rows, p.items) == 2) {
      if (p.rows <= 16) launch(items_few<T, 16, 2, GRADIENT>, 16, 2);
      else launch(items_few<T, 32, 2, GRADIENT>, 32, 2);
    } else {
      if (p.rows <= 16) launch(items_few<T, 16, 4, GRADIENT>, 16, 4);
      else launch(items_few<T, 32, 4, GRADIENT>, 32, 4);
    }
  } else {
    p.row_tiles = div_up(p.rows, tile), p.column_tiles = div_up(p.items, tile);
    // (a million rows and a million items are more tiles than a launch has)
    const uint32_t most = std::max<uint32_t>(1, most_blocks(512) / p.row_tiles);
    for (p.column_from = 0; p.column_from < p.column_tiles; p.column_from += p.columns_here) {
      p.columns_here = std::min(p.column_tiles - p.column_from, most);
      const dim3 blocks(p.row_tiles * p.columns_here);
      if (tile == 256) hipLaunchKernelGGL((items_product<T, 256, GRADIENT>), blocks, dim3(512), 0, s, p);
      else if (tile == 128) hipLaunchKernelGGL((items_product<T, 128, GRADIENT>), blocks, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((items_product<T, 64, GRADIENT>), blocks, dim3(128), 0, s, p);
      HCTR_HIP(hipGetLastError());
    }
  }
}
template <typename T> void launch_items_forward(ItemsProduct &p, int tile, hipStream_t s) { launch_items<T, false>(p, tile, s); }
template <typename T> void launch_items_gradient(ItemsProduct &p, int tile, hipStream_t s) { launch_items<T, true>(p, tile, s); }

// What brings the largest |dloss| to 2^13, where values of half precision are rounded to 11 bits down to 2^-27 of it.  That largest one
// becomes a power of two: where all rows have the same, as those of a mean do, the target's slope, p - 1 times it, is rounded with a
// p that is small and not with dloss, whose rounding would be the same in every row and add up (8192 rows of 1/6144 in bfloat16: dx and
// dweight are 0.0033 of their size off instead of 0.0017, of which 0.0017 are their own rounding).
constexpr float kScaled = 8192.f;
__device__ __forceinline__ float largest_of(uint32_t bits) { return bits ? fmaxf(__builtin_bit_cast(float, bits), 0x1p-100f) : kScaled; }

// A few rows a block: it finds how many of those before them take part from the chunks' counts and its own chunk's targets.
template <typename T, uint32_t kTakeRows> __global__ __launch_bounds__(256) void take_rows(TakeRows p) {
  constexpr int V = kVec<T>;
  __shared__ uint32_t words[5];
  __shared__ uint32_t place[kTakeRows];
  const uint32_t t = threadIdx.x, row_blocks = (p.rows + kTakeRows - 1) / kTakeRows;
  if (blockIdx.x >= row_blocks) {
    // a bias below -1e30 is as good as -infinity: a difference from it would say nothing about the rest of the logit
    const uint32_t c = (blockIdx.x - row_blocks) * kFilled + t;
    const float b = bias_at<T>(p.bias, p.narrow, c, p.items);
    p.taken.bias[c] = c >= p.items || b < -1e30f ? -kInfinity : b * kLog2E;
    return;
  }
  const uint32_t first = blockIdx.x * kTakeRows, chunk = first / kChunk;
  const uint32_t in = first % kChunk, chunk_rows = min(kChunk, p.rows - chunk * kChunk);
  // the rows of the chunk before this block's, and of the chunks before it; block 0 looks at all of them
  uint32_t before = 0, all = 0, most = 0;
  const bool head = blockIdx.x == 0;
  for (uint32_t i = t; i < (head ? chunk_rows : in); i += 256) {
    const uint32_t r = chunk * kChunk + i;
    const bool taken = p.target[r] != p.ignored;
    before += taken && i < in;
    all += taken;
    if (head && taken && p.scaled) most = max(most, size_bits(p.dloss[r]));
  }
  if (p.chunks) {
    const uint32_t chunks = (p.rows + kChunk - 1) / kChunk;
    if (head) all = most = 0;
    for (uint32_t i = t; i < (head ? chunks : chunk); i += 256) {
      const uint2 c = p.chunks[i];
      if (head) all += c.x, most = max(most, c.y);
      else before += c.x;
    }
  }
  if (head) before = 0;
  uint32_t total;
  block_exclusive_scan<256>(head ? all : before, words, total);
  if (head) {
    __shared__ uint32_t largest[4];
#pragma unroll
    for (int mask = 32; mask; mask /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, mask));
    if (lane_id() == 0) largest[t / kWave] = most;
    __syncthreads();
    if (t == 0) {
      *p.taken.count = total;
      const float one = p.scaled ? largest_of(max(max(largest[0], largest[1]), max(largest[2], largest[3]))) : kScaled;
      p.taken.scale[0] = kScaled / one, p.taken.scale[1] = one / kScaled;
    }
    if (p.dloss && total + t < (total + kFilled - 1) / kFilled * kFilled)
      p.taken.target[total + t] = kNoItem, p.taken.dloss[total + t] = 0.f, p.taken.lse[total + t] = kInfinity;
  }
  if (t < kTakeRows) {
    const uint32_t r = first + t;
    const int64_t target = r < p.rows ? p.target[r] : p.ignored;
    const bool taken = target != p.ignored;
    const uint32_t mask = (uint32_t)__ballot(taken) & ((1u << kTakeRows) - 1);
    const uint32_t to = (head ? 0 : total) + __popc(mask & ((1u << t) - 1));
    place[t] = taken ? to : kNoItem;
    if (taken) {
      p.taken.row_of[to] = r;
      p.taken.target[to] = target >= 0 && target < (int64_t)p.items ? (uint32_t)target : kNoItem;
      if (p.dloss) p.taken.dloss[to] = p.dloss[r], p.taken.lse[to] = p.lse_in[r];
    } else if (r < p.rows) {
      if (p.loss) p.loss[r] = 0.f;
      if (p.lse) p.lse[r] = 0.f;
    }
  }
  __syncthreads();
  // all rows' pieces in turn, several loads under way
  const uint32_t pieces = p.to_stride / V;
  constexpr int LOADS = 4;
  for (uint32_t from = t; from < kTakeRows * pieces; from += 256 * LOADS) {
    typename Packed<T, V>::type v[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; k++) {
      const uint32_t at = from + k * 256, i = at / pieces, c = (at - i * pieces) * V;
      if (i < kTakeRows && place[i] != kNoItem) v[k] = load_raw<V, Rows::kLong>((const T *)p.x + (int64_t)(first + i) * p.x_stride, c, p.width);
    }
#pragma unroll
    for (int k = 0; k < LOADS; k++) {
      const uint32_t at = from + k * 256, i = at / pieces, c = (at - i * pieces) * V;
      if (i >= kTakeRows || first + i >= p.rows) continue;
      if (place[i] != kNoItem) *(typename Packed<T, V>::type *)((T *)p.to + (uint64_t)place[i] * p.to_stride + c) = settled<V, Rows::kLong>(v[k], c, p.width);
      else if (p.dx) store_columns<V, Rows::kLong>((T *)p.dx + (int64_t)(first + i) * p.dx_stride, c, p.width, Floats<V>{});
    }
  }
}
template <typename T> void launch_take_rows(const TakeRows &p, hipStream_t s) {
  const auto launch = [&](auto kernel, uint32_t rows) { hipLaunchKernelGGL(kernel, dim3(div_up(p.rows, rows) + div_up(p.items, kFilled)), dim3(256), 0, s, p); };
  if (p.rows <= kChunk) launch(take_rows<T, 2>, 2);
  else launch(take_rows<T, 8>, 8);
  HCTR_HIP(hipGetLastError());
}

} // namespace hctr
