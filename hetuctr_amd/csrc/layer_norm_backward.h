// The kernels of the gradient of layer normalisation: of the rows, and of weight and bias.
//
// The rows' gradients need two sums over each row.  Those of weight and bias are sums over all rows: every block adds up the rows
// that it works on, writes one row of partial sums, and a second kernel adds those up in the order of the blocks, so that the
// result does not depend on which block is done first.
#pragma once
#include "layer_norm.h"

namespace hctr {
namespace {

// One block per row at a time, which it reads twice; its sums for weight and bias lie in its row of `partial` from the first row
// on: rows of any width.  It reads the row twice, and reads and writes the sums, 8 bytes a column each way, for every row: 1.2e8 floats in
// rows of 20000 704 us (2.0 TB/s of what the operator has to move), bfloat16 503 (1.4).
template <typename S, typename A, bool ADD, bool DROP>
__global__ __launch_bounds__(kWideGradBlock) void grad_wide(NormBackward a) {
  constexpr int V = kVec<S>;
  __shared__ float smem[kWideGradBlock / kWave];
  const uint64_t step = DROP ? step_of(a.drop) : 0;
  float *dweight = a.partial ? a.partial + (uint64_t)blockIdx.x * 2 * a.width : nullptr, *dbias = dweight + a.width;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float mean = a.mean[r], rstd = a.rstd[r];
    const auto gradient = [&](uint32_t c) { // of y, before what was dropped behind the normalisation
      Floats<V> f = load_columns<V, Rows::kLong>((const A *)a.dy + (int64_t)r * a.dy_stride, c, a.width);
      if constexpr (DROP && !ADD) drop_columns(f, a.drop, step, r * a.drop.quads + c / 4);
      return f;
    };
    const auto normal = [&](uint32_t c) {
      Floats<V> f = load_columns<V, Rows::kLong>((const S *)a.s + (int64_t)r * a.s_stride, c, a.width);
#pragma unroll
      for (int j = 0; j < V; j++) f.v[j] = (f.v[j] - mean) * rstd;
      return f;
    };
    float sum_g = 0.f, sum_gh = 0.f;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kWideGradBlock * V) {
      const Floats<V> g = gradient(c), h = normal(c);
      Floats<V> w[1];
      load_affine<V, A, Rows::kLong>(w, a.weight, a.narrow, c, 0, a.width, 1.f);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float gw = g.v[j] * w[0].v[j];
        if (c + j < a.width) {
          sum_g += gw;
          sum_gh = fmaf(gw, h.v[j], sum_gh);
        }
      }
      if (dweight) {
        const bool begin = r == blockIdx.x;
        Floats<V> sw = g, sb = g;
        const Floats<V> ow = begin ? Floats<V>{} : load_columns<V, Rows::kLong>((const float *)dweight, c, a.width);
        const Floats<V> ob = begin ? Floats<V>{} : load_columns<V, Rows::kLong>((const float *)dbias, c, a.width);
#pragma unroll
        for (int j = 0; j < V; j++) {
          sw.v[j] = fmaf(g.v[j], h.v[j], ow.v[j]);
          sb.v[j] += ob.v[j];
        }
        store_columns<V, Rows::kLong>(dweight, c, a.width, sw);
        store_columns<V, Rows::kLong>(dbias, c, a.width, sb);
      }
    }
    const float mean_g = block_sum<kWideGradBlock>(sum_g, smem) * a.inv_width, mean_gh = block_sum<kWideGradBlock>(sum_gh, smem) * a.inv_width;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kWideGradBlock * V) {
      const Floats<V> g = gradient(c), h = normal(c);
      Floats<V> w[1];
      load_affine<V, A, Rows::kLong>(w, a.weight, a.narrow, c, 0, a.width, 1.f);
      Floats<V> d;
#pragma unroll
      for (int j = 0; j < V; j++) d.v[j] = rstd * (fmaf(g.v[j], w[0].v[j], -mean_g) - h.v[j] * mean_gh);
      if constexpr (ADD) {
        if (a.ds) {
          const Floats<V> more = load_columns<V, Rows::kLong>((const S *)a.ds + (int64_t)r * a.ds_stride, c, a.width);
#pragma unroll
          for (int j = 0; j < V; j++) d.v[j] += more.v[j];
        }
        if (a.dresidual) store_columns<V, Rows::kLong>((S *)a.dresidual + (int64_t)r * a.dresidual_stride, c, a.width, d);
        if (a.dx) {
          if constexpr (DROP) drop_columns(d, a.drop, step, r * a.drop.quads + c / 4);
          store_columns<V, Rows::kLong>((A *)a.dx + (int64_t)r * a.dx_stride, c, a.width, d);
        }
      } else {
        store_columns<V, Rows::kLong>((S *)a.dx + (int64_t)r * a.dx_stride, c, a.width, d);
      }
    }
  }
}

// The gradients of weight and bias, of few rows: kColumns columns per block, whose threads share out the rows, read them for
// themselves beside the blocks of rows, and join their sums through LDS.  Nothing has to be written in between, and no second
// launch adds it up.
constexpr uint32_t kColumns = 8;
template <typename S, typename A, bool DROPPED, int BLOCK> __device__ __forceinline__ void sum_columns(const NormBackward &a, uint32_t block) {
  constexpr uint32_t ROWS = BLOCK / kColumns, LOADS = 8;
  __shared__ float2 sums[ROWS][kColumns];
  const uint32_t x = threadIdx.x % kColumns, y = threadIdx.x / kColumns, c = block * kColumns + x;
  const uint64_t step = DROPPED ? step_of(a.drop) : 0;
  float w = 0.f, b = 0.f;
  for (uint64_t r = y; r < a.rows; r += ROWS * LOADS) {
    float g[LOADS], s[LOADS], mean[LOADS], rstd[LOADS];
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) {
      const uint64_t at = r + k * ROWS;
      const bool there = at < a.rows && c < a.width;
      g[k] = there ? (float)((const A *)a.dy)[(int64_t)at * a.dy_stride + c] : 0.f;
      s[k] = there ? (float)((const S *)a.s)[(int64_t)at * a.s_stride + c] : 0.f;
      mean[k] = there ? a.mean[at] : 0.f;
      rstd[k] = there ? a.rstd[at] : 0.f;
    }
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) {
      if constexpr (DROPPED) {
        const Quad q = philox((r + k * ROWS) * a.drop.quads + c / 4, step, a.drop.seed);
        const uint32_t word = c % 4 < 2 ? (c % 4 == 0 ? q.w[0] : q.w[1]) : (c % 4 == 2 ? q.w[2] : q.w[3]);
        g[k] = word > a.drop.last ? g[k] * a.drop.scale : 0.f;
      }
      w = fmaf(g[k], (s[k] - mean[k]) * rstd[k], w);
      b += g[k];
    }
  }
  sums[y][x] = make_float2(w, b);
  __syncthreads();
  if (threadIdx.x >= 2 * kColumns || c >= a.width) return; // the first kColumns threads add up dweight, the next dbias
  float sum = 0.f;
  for (uint32_t i = 0; i < ROWS; i++) sum += y ? sums[i][x].y : sums[i][x].x;
  void *out = y ? a.dbias : a.dweight;
  if (!out) return;
  if (a.narrow) ((A *)out)[c] = (A)sum;
  else ((float *)out)[c] = sum;
}

// The rows that a block works on, held in registers as by the forward pass (rows_in_registers): each is read once.  A lane has the
// same columns of every row, so it keeps their sums for weight and bias in registers too, and the block's groups join theirs at
// the end.  Bound by memory: 1.7 M rows of 128, float and bfloat16, dropped, 366 us (2.2 GB, 6.0 TB/s; a plain copy reaches 6.5);
// 16384 rows of 4096, a branch added, 174 us (6.1 TB/s).  The next row is on its way while this one is worked on; where the waves of a block share a row, their two
// sums go through LDS, in two places by turns, so that one barrier per row will do.
template <typename S, typename A, bool ADD, bool DROP, Rows R, int LANES, int ITEMS>
__global__ __launch_bounds__(block_of<LANES>) void grad_rows(NormBackward a) {
  constexpr int V = kVec<S>, BLOCK = block_of<LANES>, GROUP = LANES < kWave ? LANES : kWave, WAVES = LANES / GROUP, GROUPS = BLOCK / LANES;
  if (blockIdx.x >= a.row_blocks) return sum_columns<S, A, DROP && !ADD, BLOCK>(a, blockIdx.x - a.row_blocks);
  // The widest rows leave 128 registers: the row's own values and sums, the next row if it is two matrices of 16-bit values, and no weight,
  // of which every lane puts its columns in LDS.  (1.2e8 bfloat16 values in rows of 11381: 219 us with neither, 181 this way.)
  constexpr bool TIGHT = LANES == 1024 && ITEMS * V == 16, AHEAD = !TIGHT || (sizeof(S) == 2 && !ADD);
  __shared__ float4 shelf[TIGHT ? ITEMS * V / 4 * BLOCK : 1];
  __shared__ float2 found[2][WAVES];
  __shared__ float joined[GROUPS > 1 ? GROUPS * LANES * ITEMS * V : 1];
  const uint32_t lane = threadIdx.x % GROUP, wave = WAVES > 1 ? threadIdx.x / kWave : 0;
  uint32_t first = wave * GROUP * V * ITEMS + lane * V;
  const uint64_t step = DROP ? step_of(a.drop) : 0, stride = (uint64_t)a.row_blocks * GROUPS;
  // whether the wave has columns in its piece i: if not, nothing is drawn or worked out for it
  const uint32_t begin = WAVES > 1 ? __builtin_amdgcn_readfirstlane(wave * GROUP * V * ITEMS) : 0;
  const auto used = [&](int i) { return (WAVES == 1 && i == 0) || begin + i * GROUP * V < a.width; };
  Floats<V> w[ITEMS], dweight[ITEMS], dbias[ITEMS];
  const auto fetch_weight = [&] {
    load_affine<V, A, R>(w, a.weight, a.narrow, first, GROUP * V, a.width, 1.f);
    if constexpr (DROP && !ADD) scale_all(w, a.drop.scale); // what is kept is scaled with it
    if constexpr (TIGHT) {
#pragma unroll
      for (int i = 0; i < ITEMS; i++)
#pragma unroll
        for (int q = 0; q < V / 4; q++)
          shelf[(i * (V / 4) + q) * BLOCK + threadIdx.x] = make_float4(w[i].v[4 * q], w[i].v[4 * q + 1], w[i].v[4 * q + 2], w[i].v[4 * q + 3]);
    }
  };
  fetch_weight();
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
#pragma unroll
    for (int j = 0; j < V; j++) dweight[i].v[j] = dbias[i].v[j] = 0.f;
  }
  typename Packed<A, V>::type dy[ITEMS];
  typename Packed<S, V>::type s[ITEMS];
  typename Packed<S, V>::type ds[ITEMS];
  float mean = 0.f, rstd = 0.f;
  const auto fetch = [&](uint64_t r) {
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const uint32_t c = first + i * GROUP * V;
      dy[i] = load_raw<V, R>((const A *)a.dy + (int64_t)r * a.dy_stride, c, a.width);
      s[i] = load_raw<V, R>((const S *)a.s + (int64_t)r * a.s_stride, c, a.width);
      if constexpr (ADD && AHEAD)
        if (a.ds) ds[i] = load_raw<V, R>((const S *)a.ds + (int64_t)r * a.ds_stride, c, a.width);
    }
    mean = a.mean[r];
    rstd = a.rstd[r];
  };
  uint64_t r = (uint64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
  if (AHEAD && r < a.rows) fetch(r);
  int turn = 0;
  for (; r < a.rows; r += stride) {
    if constexpr (TIGHT) asm volatile("" : "+v"(first)); // no address is worked out, and kept, before the loop
    if constexpr (!AHEAD) fetch(r);
    Floats<V> g[ITEMS], h[ITEMS];
    typename Packed<S, V>::type more[ITEMS];
    float sums[2] = {0.f, 0.f}; // of g and of g * h
    const float scale = rstd;
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const uint32_t c = first + i * GROUP * V;
      g[i] = floats<V>(settled<V, R>(dy[i], c, a.width));
      // Columns behind the end have no gradient; for the product of the two to be nothing h has to be finite there, as -mean * scale is not
      // where rows lie far enough from zero.  Ragged rows hold columns of their own there where a vector was moved; else h is 0.
      h[i] = floats<V>(settled<V, R, R == Rows::kRagged>(s[i], c, a.width));
      if constexpr (ADD && AHEAD) more[i] = ds[i];
#pragma unroll
      for (int j = 0; j < V; j++) h[i].v[j] = (h[i].v[j] - ((R == Rows::kTiny ? c + j : c) < a.width ? mean : 0.f)) * scale;
    }
    if (AHEAD && r + stride < a.rows) fetch(r + stride);
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      if (!used(i)) continue;
      if constexpr (DROP && !ADD) drop_columns<false>(g[i], a.drop, step, r * a.drop.quads + (first + i * GROUP * V) / 4);
      if constexpr (TIGHT) {
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
          const float4 x4 = shelf[(i * (V / 4) + q) * BLOCK + threadIdx.x];
          w[i].v[4 * q] = x4.x, w[i].v[4 * q + 1] = x4.y, w[i].v[4 * q + 2] = x4.z, w[i].v[4 * q + 3] = x4.w;
        }
      }
#pragma unroll
      for (int j = 0; j < V; j++) { // columns behind the end have no gradient, and add nothing
        dweight[i].v[j] = fmaf(g[i].v[j], h[i].v[j], dweight[i].v[j]);
        dbias[i].v[j] += g[i].v[j];
        g[i].v[j] *= w[i].v[j];
        sums[0] += g[i].v[j];
        sums[1] = fmaf(g[i].v[j], h[i].v[j], sums[1]);
      }
    }
    group_sums<GROUP>(sums);
    if constexpr (WAVES > 1) {
      if (lane == 0) found[turn][wave] = make_float2(sums[0], sums[1]);
      __syncthreads();
      const float2 other = found[turn][lane % WAVES]; // every lane takes one wave's
      sums[0] = other.x, sums[1] = other.y;
      group_sums<WAVES>(sums);
      turn ^= 1;
    }
    const float mean_g = sums[0] * a.inv_width, mean_gh = sums[1] * a.inv_width;
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
      if (!used(i)) continue;
      const uint32_t c = first + i * GROUP * V;
      Floats<V> d;
#pragma unroll
      for (int j = 0; j < V; j++) d.v[j] = scale * (fmaf(-h[i].v[j], mean_gh, g[i].v[j]) - mean_g);
      if constexpr (ADD) {
        if (a.ds) {
          if constexpr (!AHEAD) more[i] = load_raw<V, R>((const S *)a.ds + (int64_t)r * a.ds_stride, c, a.width);
          const Floats<V> e = floats<V>(settled<V, R>(more[i], c, a.width));
#pragma unroll
          for (int j = 0; j < V; j++) d.v[j] += e.v[j];
        }
        if (a.dresidual) store_columns<V, R>((S *)a.dresidual + (int64_t)r * a.dresidual_stride, c, a.width, d);
        if (a.dx) {
          if constexpr (DROP) drop_columns(d, a.drop, step, r * a.drop.quads + c / 4);
          store_columns<V, R>((A *)a.dx + (int64_t)r * a.dx_stride, c, a.width, d);
        }
      } else {
        store_columns<V, R>((S *)a.dx + (int64_t)r * a.dx_stride, c, a.width, d);
      }
    }
  }
  if (!a.partial) return;
  if constexpr (DROP && !ADD) {
    scale_all(dweight, a.drop.scale);
    scale_all(dbias, a.drop.scale);
  }
  float *out = a.partial + (uint64_t)blockIdx.x * 2 * a.width;
  const auto join = [&](Floats<V> (&own)[ITEMS], float *row) { // in the order of the groups, and one row of results
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ITEMS; i++)
#pragma unroll
        for (int j = 0; j < V; j++) joined[threadIdx.x / LANES * (LANES * ITEMS * V) + (i * GROUP + lane) * V + j] = own[i].v[j];
      __syncthreads();
      for (uint32_t c = threadIdx.x; c < a.width; c += BLOCK) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < GROUPS; k++) sum += joined[k * (LANES * ITEMS * V) + c];
        row[c] = sum;
      }
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; i++) store_columns<V, R>(row, first + i * GROUP * V, a.width, own[i]);
    }
  };
  join(dweight, out);
  join(dbias, out + a.width);
}

template <typename S, typename A, bool ADD, bool DROP> unsigned launch_grad(const NormBackward &p, hipStream_t s) {
  const unsigned blocks = norm_grad_blocks(p.rows, p.width, kVec<S>, (int)(sizeof(A) + sizeof(S) * (p.ds ? 2 : 1)));
  NormBackward q = p;
  q.row_blocks = blocks;
  const bool held = rows_in_registers<S>(p.width, [&](auto how, auto lanes, auto items) {
    constexpr int LANES = decltype(lanes)::value, ITEMS = decltype(items)::value, BLOCK = block_of<LANES>;
    const unsigned columns = p.dweight || p.dbias ? div_up(p.width, kColumns) : 0;
    hipLaunchKernelGGL((grad_rows<S, A, ADD, DROP, decltype(how)::value, LANES, ITEMS>), dim3(blocks + columns), dim3(BLOCK), 0, s, q);
  });
  if (!held) hipLaunchKernelGGL((grad_wide<S, A, ADD, DROP>), dim3(blocks), dim3(kWideGradBlock), 0, s, p);
  HCTR_HIP(hipGetLastError());
  return blocks;
}

} // namespace

template <typename S, typename A> unsigned launch_norm_grad(const NormBackward &p, bool add, bool dropped, hipStream_t s) {
  if (add) return dropped ? launch_grad<S, A, true, true>(p, s) : launch_grad<S, A, true, false>(p, s);
  return dropped ? launch_grad<S, A, false, true>(p, s) : launch_grad<S, A, false, false>(p, s);
}

} // namespace hctr
