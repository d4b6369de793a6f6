// The kernels of gated.h for one type; gated_*.hip build them side by side.
#pragma once
#include "few_rows.h"
#include "gated.h"

namespace hctr {

// sigmoid(v) and 1 - sigmoid(v), neither by cancellation.  For 16-bit values by the machine's own exponential of two and reciprocal: its argument is off by
// half a unit of itself, so that the value is by |v| * 2^-24 of it, far below their rounding where it is not nothing; a third of the instructions
// (us, 8192 rows through 4096 x 16384 twice 1951 -> 1800, 65536 rows through 3328 x 512 469 -> 450).
struct Sigmoid {
  float s, rest;
};
template <typename T> __device__ __forceinline__ Sigmoid sigmoid(float v) {
  float e, large;
  if constexpr (sizeof(T) == 2) {
    e = __builtin_amdgcn_exp2f(fabsf(v) * -1.4426950408889634f);
    large = __builtin_amdgcn_rcpf(1.f + e);
  } else {
    e = expf(-fabsf(v));
    large = 1.f / (1.f + e);
  }
  const float small = e * large;
  return v >= 0.f || v != v ? Sigmoid{large, small} : Sigmoid{small, large};
}
// The normal distribution's integral up to v, and exp(-v^2 / 2).  For 16-bit values by one exponential, which the slope takes too: below zero the integral
// is that exponential times t P(t), t = 1 / (1 + 0.28 |v|), with P of degree eight by least squares, weighted anew until its largest relative error
// was smallest, 1.7e-7, over all v; the exponential's argument, rounded, adds v^2 2^-24 (us, against the library's erfcf and expf: 65536 rows through 3328 x 512 twice with three results 1026 -> 865,
// its gradient 1328 -> 1258; 8192 through 4096 x 16384 1905 -> 1791).
struct Normal {
  float whole, e;
};
template <typename T> __device__ __forceinline__ Normal normal(float v) {
  if constexpr (sizeof(T) == 2) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28f, fabsf(v), 1.f)), e = __builtin_amdgcn_exp2f(v * v * -0.72134752044448170f);
    float q = 0.0247199624463723f;
    for (float c : {-0.09359308485038127f, 0.0924280603918132f, -0.0064491364459287335f, 0.07277499335202713f, 0.08363079551306478f, 0.10308466407569232f,
                    0.11169980273233898f, 0.11170385755238264f})
      q = __builtin_fmaf(q, t, c);
    const float rest = q * t * e;
    return {v < 0.f ? rest : 1.f - rest, e};
  } else return {0.5f * erfcf(v * -0.70710678118654752f), expf(-0.5f * v * v)};
}

template <typename T> __device__ __forceinline__ float activated(int f, float v) {
  if (f == HCTR_SILU) return v * sigmoid<T>(v).s;
  if (f == HCTR_GELU) return v * normal<T>(v).whole;
  if (f == HCTR_RELU) return v > 0.f || v != v ? v : 0.f;
  return sigmoid<T>(v).s;
}
// f(v) and f'(v)
struct Slope {
  float value, slope;
};
template <typename T> __device__ __forceinline__ Slope slope_of(int f, float v) {
  if (f == HCTR_GELU) {
    const Normal n = normal<T>(v);
    return {v * n.whole, n.whole + v * 0.39894228040143268f * n.e};
  }
  if (f == HCTR_RELU) return {v > 0.f || v != v ? v : 0.f, v > 0.f ? 1.f : 0.f};
  const Sigmoid g = sigmoid<T>(v);
  if (f == HCTR_SILU) return {v * g.s, g.s + v * g.s * g.rest};
  return {g.s, g.s * g.rest};
}

// four neighbouring columns of both products, which get their biases, and of the result
template <typename T> __device__ __forceinline__ f32x4 gated4(const GatedForward &p, uint32_t column, f32x4 &gate, f32x4 &up) {
  f32x4 h;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    gate[e] += bias_at<T>(p.gate_bias, p.narrow, column + e, p.hidden);
    up[e] += bias_at<T>(p.up_bias, p.narrow, column + e, p.hidden);
    h[e] = activated<T>(p.activation, gate[e]) * up[e];
  }
  return h;
}
template <typename T> __device__ __forceinline__ void finish_gated(const GatedForward &p, uint32_t row, uint32_t column, f32x4 gate, f32x4 up) {
  const f32x4 h = gated4<T>(p, column, gate, up);
  write4<T>((T *)p.h + (int64_t)row * p.h_stride, column, p.hidden, h);
  if (p.gate) write4<T>((T *)p.gate + (int64_t)row * p.gate_stride, column, p.hidden, gate);
  if (p.up) write4<T>((T *)p.up + (int64_t)row * p.up_stride, column, p.hidden, up);
}

// Both products in one: the rows of the two matrices of weights alternate in a tile, 32 by 32, so that a wave holds the same columns of
// both, and makes h of them.  Bound by the matrix cores, at the clock that their power leaves (56 % of the cycles), and by the ends of tiles, which
// nothing overlaps where a tile has the CU for itself: 8192 rows, 4096 x 16384 twice in bfloat16 1800 us with three results (1.22 PFLOP/s).
template <typename T, int TILE> __global__ __launch_bounds__((Product<T, Lies::kAlong, Lies::kAlong, Second::kPaired, TILE, TILE>::kThreads), (Product<T, Lies::kAlong, Lies::kAlong, Second::kPaired, TILE, TILE>::kWavesEach))
void gated_product(GatedForward p) {
  typedef Product<T, Lies::kAlong, Lies::kAlong, Second::kPaired, TILE, TILE> P;
  __shared__ __attribute__((aligned(1024))) char tiles[P::kLdsBytes];
  uint32_t row, column;
  tile_of(blockIdx.x, gridDim.x, p.row_tiles, p.column_tiles, p.band, row, column);
  const uint32_t steps = (p.width + kStep<T> - 1) / kStep<T>, each = (steps + p.splits - 1) / p.splits;
  const uint32_t k0 = blockIdx.y * each * kStep<T>, k1 = min(p.width, k0 + each * kStep<T>);
  typename P::Sums sum;
  P::run(p.x, p.weights, row * TILE, column * TILE, k0, k1, (uint32_t)(uintptr_t)(lds_char *)tiles, sum);
  const uint32_t l = lane_id(), half = (p.hidden + 3) / 4 * 4;
  if constexpr (sizeof(T) == 2) {
    if (!p.partial) {
      typedef Staged<T, TILE, TILE / 2> S;
      const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)tiles;
      const auto out = [&](uint32_t from, void *to, int64_t stride) {
        S::template each<P::kThreads>(from, [&](uint32_t r, uint32_t c, auto x) {
          r += row * TILE, c += column * (TILE / 2);
          if (r < p.rows && c < p.hidden) write<8>((T *)to + (int64_t)r * stride, c, p.hidden, x);
        });
      };
      __syncthreads(); // the tiles are read
#pragma unroll
      for (int i = 0; i < P::kRowTiles; i++)
#pragma unroll
        for (int j = 0; j < P::kColumnTiles / 2; j++) {
          const uint32_t r = P::wave_row() + i * 16 + l % 16, c = P::wave_column() / 2 + j * 16 + l / 16 * 4;
          S::put(lds, r, c, gated4<T>(p, column * (TILE / 2) + c, sum[i][j], sum[i][j + P::kColumnTiles / 2]));
          if (p.gate) S::put(lds + S::kBytes, r, c, sum[i][j]);
        }
      __syncthreads();
      out(lds, p.h, p.h_stride);
      if (p.gate) out(lds + S::kBytes, p.gate, p.gate_stride);
      if (!p.up) return;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < P::kRowTiles; i++)
#pragma unroll
        for (int j = 0; j < P::kColumnTiles / 2; j++)
          S::put(lds, P::wave_row() + i * 16 + l % 16, P::wave_column() / 2 + j * 16 + l / 16 * 4, sum[i][j + P::kColumnTiles / 2]);
      __syncthreads();
      out(lds, p.up, p.up_stride);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < P::kRowTiles; i++) {
    const uint32_t r = row * TILE + P::wave_row() + i * 16 + l % 16;
    if (r >= p.rows) continue;
#pragma unroll
    for (int j = 0; j < P::kColumnTiles / 2; j++) {
      const uint32_t c = (column * TILE + P::wave_column()) / 2 + j * 16 + l / 16 * 4;
      if (c >= p.hidden) continue;
      if (!p.partial) {
        finish_gated<T>(p, r, c, sum[i][j], sum[i][j + P::kColumnTiles / 2]);
      } else {
        float *part = p.partial + ((uint64_t)blockIdx.y * p.rows + r) * (2 * half) + c;
        *(f32x4 *)part = sum[i][j];
        *(f32x4 *)(part + half) = sum[i][j + P::kColumnTiles / 2];
      }
    }
  }
}

template <typename T> __global__ __launch_bounds__(256) void gated_join(GatedForward p) {
  const uint32_t quads = (p.hidden + 3) / 4;
  const uint64_t total = (uint64_t)p.rows * quads;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = total >> 32 ? i / quads : (uint32_t)i / quads;
    const uint32_t c = (uint32_t)(i - r * quads);
    const f32x4 *from = (const f32x4 *)p.partial + r * (2 * quads) + c;
    f32x4 gate = from[0], up = from[quads];
    for (uint32_t s = 1; s < p.splits; s++) {
      from += (uint64_t)p.rows * (2 * quads);
      gate += from[0], up += from[quads];
    }
    finish_gated<T>(p, (uint32_t)r, c * 4, gate, up);
  }
}

template <typename T, int ROWS, int GROUPS> __global__ __launch_bounds__((FewRows<T, ROWS, GROUPS>::kThreads)) void gated_few(GatedForward p) {
  typedef FewRows<T, ROWS, GROUPS> F;
  constexpr uint32_t HALF = F::kGroups / 2, COLUMNS = HALF * 16;
  __shared__ typename F::Sums sums[F::kSums];
  const uint32_t column0 = blockIdx.x * COLUMNS;
  const T *groups[F::kGroups];
  uint32_t left[F::kGroups];
  int64_t stride[F::kGroups];
#pragma unroll
  for (uint32_t j = 0; j < HALF; j++) {
    const uint32_t c = min(column0 + j * 16, p.hidden - 1); // (behind the last column: that one again)
    groups[j] = (const T *)p.loose_gate + (int64_t)c * p.loose_gate_stride, groups[j + HALF] = (const T *)p.loose_up + (int64_t)c * p.loose_up_stride;
    stride[j] = p.loose_gate_stride, stride[j + HALF] = p.loose_up_stride;
    left[j] = left[j + HALF] = p.hidden - c;
  }
  F::run((const T *)p.loose_x, p.loose_stride, p.rows, groups, left, stride, p.width, sums);
  for (uint32_t t = threadIdx.x; t < p.rows * (COLUMNS / 4); t += F::kThreads) {
    const uint32_t r = t / (COLUMNS / 4), c = t % (COLUMNS / 4) * 4;
    if (column0 + c < p.hidden) finish_gated<T>(p, r, column0 + c, *(const f32x4 *)&sums[0][r][c], *(const f32x4 *)&sums[0][r][c + COLUMNS]);
  }
}

// dgate and dup of columns c .. c + V - 1 of a row
template <typename T, int V> __device__ __forceinline__ void slopes_at(const GatedSlopes &p, uint32_t r, uint32_t c, Floats<V> (&d)[2]) {
  const Floats<V> dh = load_columns<V, Rows::kLong, true>((const T *)p.dh + (int64_t)r * p.dh_stride, c, p.hidden);
  const Floats<V> gate = load_columns<V, Rows::kLong, true>((const T *)p.gate + (int64_t)r * p.gate_stride, c, p.hidden);
  const Floats<V> up = load_columns<V, Rows::kLong, true>((const T *)p.up + (int64_t)r * p.up_stride, c, p.hidden);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const Slope s = slope_of<T>(p.activation, gate.v[e]);
    d[0].v[e] = c + e < p.hidden ? dh.v[e] * up.v[e] * s.slope : 0.f;
    d[1].v[e] = c + e < p.hidden ? dh.v[e] * s.value : 0.f;
  }
}
// the largest of them, leaving out what is not finite
template <int V> __device__ __forceinline__ float largest(const Floats<V> (&d)[2], float most) {
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int e = 0; e < V; e++) most = fmaxf(most, fabsf(d[i].v[e]) < __builtin_inff() ? fabsf(d[i].v[e]) : 0.f);
  return most;
}
// the largest of a block's values, which are not negative, the same in all threads
__device__ __forceinline__ float block_most(float v) {
  __shared__ float waves[256 / kWave];
#pragma unroll
  for (int mask = 32; mask; mask /= 2) v = fmaxf(v, __shfl_xor(v, mask));
  __syncthreads(); // what was there before is read
  if (lane_id() == 0) waves[threadIdx.x / kWave] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 256 / kWave; i++) v = fmaxf(v, waves[i]);
  return v;
}

// dgate and dup, as the operands of the products: rounded to the type, since the matrix cores take both of a product's in one.  Eight threads share
// out the rows of 32 pieces, block `across` along the columns, `down` along the rows.  SUMS: the sums over a block's rows, of what was neither
// scaled nor rounded.  Returns, if SIZE, the largest that the thread made, before it was scaled.
template <typename T, bool SUMS, bool SIZE> __device__ __forceinline__ float slopes_of(const GatedSlopes &p, uint32_t across, uint32_t down, float scale) {
  constexpr int V = kVec<T>, LANES = 32, GROUPS = 8;
  __shared__ float joined[SUMS ? GROUPS : 1][2][LANES * V];
  const uint32_t x = threadIdx.x % LANES, y = threadIdx.x / LANES, c = (across * LANES + x) * V;
  const uint32_t first = down * p.rows_each, last = min(p.rows, first + p.rows_each);
  Floats<V> sums[2] = {};
  float most = 0.f;
  if (c < p.padded)
    for (uint32_t r = first + y; r < last; r += GROUPS) {
      Floats<V> d[2];
      slopes_at<T>(p, r, c, d);
      if (SIZE) most = largest(d, most);
      T *to = (T *)p.slopes + (uint64_t)r * (2 * p.padded) + c;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (SUMS)
#pragma unroll
          for (int e = 0; e < V; e++) sums[i].v[e] += d[i].v[e];
#pragma unroll
        for (int e = 0; e < V; e++) d[i].v[e] *= scale;
        *(typename Packed<T, V>::type *)(to + i * p.padded) = rounded<T>(d[i]);
      }
    }
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < V; e++) joined[y][i][e * LANES + x] = sums[i].v[e];
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < 2 * LANES * V; t += 256) {
      const uint32_t i = t / (LANES * V), at = t % (LANES * V), column = across * LANES * V + at;
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < GROUPS; g++) sum += joined[g][i][at % V * LANES + at / V];
      if (column < p.padded) p.sums[(uint64_t)down * (2 * p.padded) + i * p.padded + column] = sum;
    }
  }
  return most;
}

// Half precision does not hold every slope: beyond 65504 they are infinite, and below 2^-14 they lose bits.  So they are multiplied by a power of
// two, by which the products' sums are divided, where that keeps the largest of them in 1 .. 2^15: then those above 2^-14 of it have
// all their bits, and none is off by more than 2^-25 of it.  The power is that which takes the largest of some rows to 2^8 .. 2^9, one if there
// are few; a launch behind finds the largest of all, and makes them again, it being in 2^13 .. 2^14, where it was not in that range.
__device__ __forceinline__ int power_to(int to, float most) { return most > 0.f ? min(to - ilogbf(most), 126) : 0; } // (a factor that is a float, and so is 1 / it)
__device__ __forceinline__ int guessed_power(const GatedSlopes &p) { return p.guess ? power_to(8, block_most(p.guess[threadIdx.x])) : 0; }

template <typename T> __global__ __launch_bounds__(256) void gated_guess(GatedSlopes p, uint32_t some) {
  constexpr uint32_t V = kVec<T>;
  const uint32_t pieces = (p.hidden + V - 1) / V;
  float most = 0.f;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < some * pieces; i += kGuesses * 256) {
    Floats<V> d[2];
    slopes_at<T>(p, (uint32_t)((uint64_t)(i / pieces) * p.rows / some), i % pieces * V, d);
    most = largest(d, most);
  }
  most = block_most(most);
  if (threadIdx.x == 0) p.guess[blockIdx.x] = most;
}

// Bound by memory: 8192 x 16384 in bfloat16, three matrices read and two written, 217 us, 6.2 TB/s.
template <typename T, bool SUMS> __global__ __launch_bounds__(256) void gated_slopes(GatedSlopes p) {
  if constexpr (std::is_same_v<T, f16_t>) {
    const float most = block_most(slopes_of<T, SUMS, true>(p, blockIdx.x, blockIdx.y, ldexpf(1.f, guessed_power(p))));
    if (p.sizes && threadIdx.x == 0) p.sizes[blockIdx.y * gridDim.x + blockIdx.x] = most;
  } else {
    slopes_of<T, SUMS, false>(p, blockIdx.x, blockIdx.y, 1.f);
  }
}

template <typename T> __global__ __launch_bounds__(256) void gated_rescale(GatedSlopes p, uint32_t across, uint32_t blocks) {
  float most = 0.f;
  for (uint32_t i = threadIdx.x; i < blocks; i += 256) most = fmaxf(most, p.sizes[i]);
  most = block_most(most);
  int by = guessed_power(p);
  const float was = ldexpf(most, by);
  const bool fits = most == 0.f || (was >= 1.f && was < 32768.f);
  if (!fits) by = power_to(13, most);
  const float scale = ldexpf(1.f, by);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.scale[0] = scale, p.scale[1] = ldexpf(1.f, -by);
  if (fits) return;
  for (uint32_t i = blockIdx.x; i < blocks; i += gridDim.x) slopes_of<T, false, false>(p, i % across, i / across, scale);
}

template <typename T> void launch_gated(GatedForward &p, int tile, hipStream_t s) {
  p.row_tiles = div_up(p.rows, tile), p.column_tiles = div_up(p.hidden, tile / 2);
  const dim3 blocks(p.row_tiles * p.column_tiles, p.splits), threads(tile_threads(p.row_tiles, p.column_tiles, tile, "gated linear"));
  if (tile == 256) hipLaunchKernelGGL((gated_product<T, 256>), blocks, threads, 0, s, p);
  else if (tile == 128) hipLaunchKernelGGL((gated_product<T, 128>), blocks, threads, 0, s, p);
  else hipLaunchKernelGGL((gated_product<T, 64>), blocks, threads, 0, s, p);
  HCTR_HIP(hipGetLastError());
  if (p.partial) {
    const uint64_t quads = (uint64_t)p.rows * ((p.hidden + 3) / 4);
    hipLaunchKernelGGL((gated_join<T>), dim3((unsigned)min((quads + 255) / 256, (uint64_t)16384)), dim3(256), 0, s, p);
    HCTR_HIP(hipGetLastError());
  }
}
template <typename T> void launch_gated_few(const GatedForward &p, hipStream_t s) {
  const auto launch = [&](auto kernel, int groups) {
    hipLaunchKernelGGL(kernel, dim3(div_up(p.hidden, 8 * groups)), dim3(FewRows<T, 16, 2>::kThreads), 0, s, p);
  };
  if (few_groups(p.rows, 2 * (size_t)p.hidden) == 2) {
    if (p.rows <= 16) launch(gated_few<T, 16, 2>, 2);
    else launch(gated_few<T, 32, 2>, 2);
  } else {
    if (p.rows <= 16) launch(gated_few<T, 16, 4>, 4);
    else launch(gated_few<T, 32, 4>, 4);
  }
  HCTR_HIP(hipGetLastError());
}
template <typename T> void launch_slopes(const GatedSlopes &p, hipStream_t s) {
  const dim3 blocks(div_up(p.padded, slope_columns(sizeof(T))), div_up(p.rows, p.rows_each));
  if constexpr (std::is_same_v<T, f16_t>)
    if (p.guess) {
      hipLaunchKernelGGL((gated_guess<T>), dim3(kGuesses), dim3(256), 0, s, p, min(p.rows, 64u));
      HCTR_HIP(hipGetLastError());
    }
  if (p.sums) hipLaunchKernelGGL((gated_slopes<T, true>), blocks, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((gated_slopes<T, false>), blocks, dim3(256), 0, s, p);
  HCTR_HIP(hipGetLastError());
  if constexpr (std::is_same_v<T, f16_t>)
    if (p.sizes) {
      hipLaunchKernelGGL((gated_rescale<T>), dim3(min(blocks.x * blocks.y, 2048u)), dim3(256), 0, s, p, blocks.x, blocks.x * blocks.y);
      HCTR_HIP(hipGetLastError());
    }
}

} // namespace hctr
