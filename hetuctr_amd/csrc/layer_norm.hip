// Layer normalisation of rows, with dropout behind it or a dropped-out branch added before it.
#include <algorithm>

#include "layer_norm.h"

namespace hctr {
namespace {

constexpr int kBlock = 256;

// One block per row at a time, which it reads again for each of mean, variance and result: rows of any width.
template <typename S, typename A, bool ADD, bool DROP>
__global__ __launch_bounds__(kBlock) void norm_wide(NormForward a) {
  constexpr int V = kVec<S>;
  __shared__ float smem[kBlock / kWave];
  const uint64_t step = DROP ? step_of(a.drop) : 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const auto value = [&](uint32_t c) { // what is normalised, in 32 bits
      if constexpr (ADD) {
        Floats<V> f = load_columns<V>((const A *)a.x + (int64_t)r * a.x_stride, c, a.width);
        if constexpr (DROP) drop_columns(f, a.drop, step, r * a.drop.quads + c / 4);
        const Floats<V> g = load_columns<V>((const S *)a.residual + (int64_t)r * a.residual_stride, c, a.width);
#pragma unroll
        for (int j = 0; j < V; j++) f.v[j] += g.v[j];
        return f;
      } else {
        return load_columns<V>((const S *)a.x + (int64_t)r * a.x_stride, c, a.width);
      }
    };
    float sum = 0.f;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kBlock * V) {
      const Floats<V> f = value(c);
      if constexpr (ADD) store_columns((S *)a.sum + (int64_t)r * a.sum_stride, c, a.width, f);
#pragma unroll
      for (int j = 0; j < V; j++) sum += f.v[j];
    }
    const float mean = block_sum<kBlock>(sum, smem) * a.inv_width;
    float square = 0.f;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kBlock * V) {
      const Floats<V> f = value(c);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float d = c + j < a.width ? f.v[j] - mean : 0.f;
        square = fmaf(d, d, square);
      }
    }
    const float rstd = rsqrtf(block_sum<kBlock>(square, smem) * a.inv_width + a.eps);
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kBlock * V) {
      Floats<V> f = value(c);
      const Floats<V> w = load_affine<V, A>(a.weight, a.narrow, c, a.width, 1.f), b = load_affine<V, A>(a.bias, a.narrow, c, a.width, 0.f);
#pragma unroll
      for (int j = 0; j < V; j++) f.v[j] = fmaf((f.v[j] - mean) * rstd, w.v[j], b.v[j]);
      if constexpr (DROP && !ADD) drop_columns(f, a.drop, step, r * a.drop.quads + c / 4);
      store_columns((A *)a.y + (int64_t)r * a.y_stride, c, a.width, f);
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
  }
}

// ITEMS pieces of V columns per lane of a row that LANES lanes hold in registers: the row is read once.  Up to a wave's
// lanes, a group of lanes has a row to itself and a block as many rows as it has groups; beyond that the waves of a block share
// a row, each a stretch of neighbouring columns, and join what they found: a wave's sum and its squares around its own
// mean.  (Squares around a mean that is not the row's would cancel; put together as n * (wave's mean - mean)^2 they do not,
// and the block waits once instead of twice.)
template <typename S, typename A, bool ADD, bool DROP, int LANES, int ITEMS>
__global__ __launch_bounds__(block_of<LANES>) void norm_rows(NormForward a) {
  constexpr int V = kVec<S>, BLOCK = block_of<LANES>, GROUP = LANES < kWave ? LANES : kWave, WAVES = LANES / GROUP;
  constexpr uint32_t STRETCH = GROUP * V * ITEMS; // columns of a group, or wave
  __shared__ float2 found[WAVES];
  const uint32_t lane = threadIdx.x % GROUP, wave = WAVES > 1 ? threadIdx.x / kWave : 0, first = wave * STRETCH + lane * V;
  const bool even = a.width % V == 0;
  const uint64_t step = DROP ? step_of(a.drop) : 0;
  for (uint64_t r = (uint64_t)blockIdx.x * (BLOCK / LANES) + threadIdx.x / LANES; r < a.rows; r += (uint64_t)gridDim.x * (BLOCK / LANES)) {
    Floats<V> f[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const uint32_t c = first + i * GROUP * V;
      if constexpr (ADD) f[i] = load_columns<V>((const A *)a.x + (int64_t)r * a.x_stride, c, a.width);
      else f[i] = load_columns<V>((const S *)a.x + (int64_t)r * a.x_stride, c, a.width);
    }
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < ITEMS; i++) {
        const uint32_t c = first + i * GROUP * V;
        const Floats<V> g = load_columns<V>((const S *)a.residual + (int64_t)r * a.residual_stride, c, a.width);
        if constexpr (DROP) drop_columns(f[i], a.drop, step, r * a.drop.quads + c / 4);
#pragma unroll
        for (int j = 0; j < V; j++) f[i].v[j] += g.v[j];
        store_columns((S *)a.sum + (int64_t)r * a.sum_stride, c, a.width, f[i]);
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; i++)
#pragma unroll
      for (int j = 0; j < V; j++) sum += f[i].v[j];
    sum = group_sum<GROUP>(sum);
    // columns behind the end hold zeros and have to add nothing to the squares
    const float n = WAVES > 1 ? (float)min(a.width - min(a.width, wave * STRETCH), STRETCH) : 0.f;
    const float middle = WAVES > 1 ? sum / fmaxf(n, 1.f) : sum * a.inv_width;
    float square = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const uint32_t c = first + i * GROUP * V;
      if (even) {
        const float m = c < a.width ? middle : 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) square = fmaf(f[i].v[j] - m, f[i].v[j] - m, square);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float d = f[i].v[j] - (c + j < a.width ? middle : 0.f);
          square = fmaf(d, d, square);
        }
      }
    }
    square = group_sum<GROUP>(square);
    float mean = middle;
    if constexpr (WAVES > 1) {
      __syncthreads(); // the row before has been read
      if (lane == 0) found[wave] = make_float2(sum, square);
      __syncthreads();
      sum = square = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) sum += found[w].x;
      mean = sum * a.inv_width;
#pragma unroll
      for (int w = 0; w < WAVES; w++) {
        const float k = (float)min(a.width - min(a.width, w * STRETCH), STRETCH), off = found[w].x / fmaxf(k, 1.f) - mean;
        square += fmaf(k * off, off, found[w].y);
      }
    }
    const float rstd = rsqrtf(fmaf(square, a.inv_width, a.eps));
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const uint32_t c = first + i * GROUP * V;
      const Floats<V> w = load_affine<V, A>(a.weight, a.narrow, c, a.width, 1.f), b = load_affine<V, A>(a.bias, a.narrow, c, a.width, 0.f);
#pragma unroll
      for (int j = 0; j < V; j++) f[i].v[j] = fmaf((f[i].v[j] - mean) * rstd, w.v[j], b.v[j]);
      if constexpr (DROP && !ADD) drop_columns(f[i], a.drop, step, r * a.drop.quads + c / 4);
      store_columns((A *)a.y + (int64_t)r * a.y_stride, c, a.width, f[i]);
    }
    if (threadIdx.x % LANES == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
  }
}

template <typename S, typename A, bool ADD, bool DROP> void launch(const NormForward &p, hipStream_t s) {
  const bool held = rows_in_registers<S>(p.width, [&](auto lanes, auto items) {
    constexpr int LANES = decltype(lanes)::value, ITEMS = decltype(items)::value, BLOCK = block_of<LANES>;
    const uint64_t blocks = (p.rows + BLOCK / LANES - 1) / (BLOCK / LANES);
    hipLaunchKernelGGL((norm_rows<S, A, ADD, DROP, LANES, ITEMS>), dim3((unsigned)std::min<uint64_t>(blocks, (1u << 31) / BLOCK)),
                       dim3(BLOCK), 0, s, p);
  });
  if (!held)
    hipLaunchKernelGGL((norm_wide<S, A, ADD, DROP>), dim3((unsigned)std::min<uint64_t>(p.rows, 1u << 20)), dim3(kBlock), 0, s, p);
  HCTR_HIP(hipGetLastError());
}

template <typename S, typename A> void launch_types(const NormForward &p, bool add, bool on, hipStream_t s) {
  if (add) on ? launch<S, A, true, true>(p, s) : launch<S, A, true, false>(p, s);
  else on ? launch<S, A, false, true>(p, s) : launch<S, A, false, false>(p, s);
}

} // namespace

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
  if (a.stream_dtype == HCTR_BF16) launch_types<bf16_t, bf16_t>(p, add, on, s);
  else if (a.stream_dtype == HCTR_F16) launch_types<f16_t, f16_t>(p, add, on, s);
  else if (a.act_dtype == HCTR_BF16) launch_types<float, bf16_t>(p, add, on, s);
  else if (a.act_dtype == HCTR_F16) launch_types<float, f16_t>(p, add, on, s);
  else launch_types<float, float>(p, add, on, s);
}

} // namespace hctr
