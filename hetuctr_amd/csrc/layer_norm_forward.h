// The kernels of layer normalisation, with dropout behind it or a dropped-out branch added before it.
#pragma once
#include "layer_norm.h"

namespace hctr {
namespace {

// One block per row at a time, which it reads again for each of mean, variance and result: rows of any width.  1.2e8 floats in rows
// of 20000 313 us (3.1 TB/s of what the operator has to move), of 65536 407 (2.4); bfloat16 162 (3.0) and 217 (2.2).
template <typename S, typename A, bool ADD, bool DROP>
__global__ __launch_bounds__(kWideBlock) void norm_wide(NormForward a) {
  constexpr int V = kVec<S>;
  __shared__ float smem[kWideBlock / kWave];
  const uint64_t step = DROP ? step_of(a.drop) : 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const auto value = [&](uint32_t c) { // what is normalised, in 32 bits
      if constexpr (ADD) {
        Floats<V> f = load_columns<V, Rows::kLong>((const A *)a.x + (int64_t)r * a.x_stride, c, a.width);
        if constexpr (DROP) drop_columns(f, a.drop, step, r * a.drop.quads + c / 4);
        const Floats<V> g = load_columns<V, Rows::kLong>((const S *)a.residual + (int64_t)r * a.residual_stride, c, a.width);
#pragma unroll
        for (int j = 0; j < V; j++) f.v[j] += g.v[j];
        return f;
      } else {
        return load_columns<V, Rows::kLong>((const S *)a.x + (int64_t)r * a.x_stride, c, a.width);
      }
    };
    float sum = 0.f;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kWideBlock * V) {
      const Floats<V> f = value(c);
      if constexpr (ADD) store_columns<V, Rows::kLong>((S *)a.sum + (int64_t)r * a.sum_stride, c, a.width, f);
#pragma unroll
      for (int j = 0; j < V; j++) sum += f.v[j];
    }
    const float mean = block_sum<kWideBlock>(sum, smem) * a.inv_width;
    float square = 0.f;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kWideBlock * V) {
      const Floats<V> f = value(c);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float d = c + j < a.width ? f.v[j] - mean : 0.f;
        square = fmaf(d, d, square);
      }
    }
    const float rstd = rsqrtf(block_sum<kWideBlock>(square, smem) * a.inv_width + a.eps);
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kWideBlock * V) {
      Floats<V> f = value(c);
      Floats<V> w[1], b[1];
      load_affine<V, A, Rows::kLong>(w, a.weight, a.narrow, c, 0, a.width, 1.f);
      load_affine<V, A, Rows::kLong>(b, a.bias, a.narrow, c, 0, a.width, 0.f);
#pragma unroll
      for (int j = 0; j < V; j++) f.v[j] = fmaf((f.v[j] - mean) * rstd, w[0].v[j], b[0].v[j]);
      if constexpr (DROP && !ADD) drop_columns(f, a.drop, step, r * a.drop.quads + c / 4);
      store_columns<V, Rows::kLong>((A *)a.y + (int64_t)r * a.y_stride, c, a.width, f);
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
  }
}

// Rows of more than 512 columns: a block stays for several.
template <typename S, int LANES, int ITEMS> constexpr bool stays = LANES * ITEMS * kVec<S> > 512;
// The widest leave no registers for weight and bias beside the next row: every lane puts what it needs of them in LDS, 128 KiB
// in all.  (Read again for every row they are more bytes than the row: 1.2e8 bfloat16 values in rows of 16384 124 us, 83 this way.)
template <typename S, int LANES, int ITEMS> constexpr bool shelved = LANES == 1024 && ITEMS * kVec<S> == 16;

// ITEMS pieces of V columns per lane of a row that LANES lanes hold in registers: the row is read once.  Up to a wave's
// lanes, a group of lanes has a row to itself, ROWS of them at a time, and a block as many as it has groups; beyond that the waves of a
// block share a row, each a stretch of neighbouring columns, and join what they found: a wave's sum and its squares around
// its own mean.  (Squares around a mean that is not the row's would cancel; put together as n * (wave's mean - mean)^2 they do
// not, and the block waits once instead of twice.)  Bound by memory, and by arithmetic as much where values are drawn: 1.7 M rows
// of 128, float to bfloat16, dropped, 214 us (1.3 GB, 6.2 TB/s; a plain copy reaches 6.5); 16384 rows of 4096, a branch dropped
// and added, 131 us (6.1 TB/s).
template <typename S, typename A, bool ADD, bool DROP, Rows R, int LANES, int ITEMS, int ROWS>
__global__ __launch_bounds__(block_of<LANES>) void norm_rows(NormForward a) {
  constexpr int V = kVec<S>, BLOCK = block_of<LANES>, GROUP = LANES < kWave ? LANES : kWave, WAVES = LANES / GROUP, GROUPS = BLOCK / LANES;
  constexpr uint32_t STRETCH = GROUP * V * ITEMS; // columns of a group, or wave
  static_assert(WAVES == 1 || ROWS == 1, "a block that shares a row has one at a time");
  // Wide rows: a block stays for several, weight and bias in its registers, the next row on its way while one is worked on.
  constexpr bool STAYS = stays<S, LANES, ITEMS>;
  constexpr bool SHELVED = shelved<S, LANES, ITEMS>;
  __shared__ float4 shelf[SHELVED ? 2 * ITEMS * V / 4 * BLOCK : 1];
  __shared__ float2 found[2][WAVES]; // by turns, so that one barrier per row will do
  const uint32_t lane = threadIdx.x % GROUP, wave = WAVES > 1 ? threadIdx.x / kWave : 0;
  uint32_t first = wave * STRETCH + lane * V;
  const uint64_t step = DROP ? step_of(a.drop) : 0;
  typedef std::conditional_t<ADD, A, S> X;
  typename Packed<X, V>::type x[ROWS][ITEMS];
  typename Packed<S, V>::type residual[ROWS][ITEMS];
  Floats<V> w[ITEMS], b[ITEMS];
  // The group's rows are r0, r0 + GROUPS, .., and r0 moves on by `stride`; their addresses move with it.
  const uint64_t block0 = (uint64_t)blockIdx.x * (GROUPS * ROWS), stride = (uint64_t)gridDim.x * (GROUPS * ROWS);
  constexpr bool UNIFORM = LANES >= kWave;
  const uint32_t group = GROUPS == 1 ? 0 : UNIFORM ? __builtin_amdgcn_readfirstlane(threadIdx.x / LANES) : threadIdx.x / LANES;
  uint64_t r0 = block0 + group, quad = DROP ? rows_away<UNIFORM>(block0, group, a.drop.quads) : 0;
  S *ps = ADD ? (S *)a.sum + rows_away<UNIFORM>(block0, group, a.sum_stride) : nullptr;
  A *py = (A *)a.y + rows_away<UNIFORM>(block0, group, a.y_stride);
  // a row that is not there is one of no columns
  const auto width = [&](int k, uint64_t r) { return k == 0 || r + k * GROUPS < a.rows ? a.width : 0; };
  const X *px = (const X *)a.x + rows_away<UNIFORM>(block0, group, a.x_stride);
  const S *pr = ADD ? (const S *)a.residual + rows_away<UNIFORM>(block0, group, a.residual_stride) : nullptr;
  const auto fetch = [&](uint64_t r) {
    if constexpr (STAYS) { // ahead of the loop
      px = (const X *)a.x + (int64_t)r * a.x_stride;
      pr = ADD ? (const S *)a.residual + (int64_t)r * a.residual_stride : nullptr;
    }
#pragma unroll
    for (int k = 0; k < ROWS; k++)
#pragma unroll
      for (int i = 0; i < ITEMS; i++) {
        const uint32_t c = first + i * GROUP * V;
        x[k][i] = load_raw<V, R>(px + k * GROUPS * a.x_stride, c, width(k, r));
        if constexpr (ADD) residual[k][i] = load_raw<V, R>(pr + k * GROUPS * a.residual_stride, c, width(k, r));
      }
    px += (int64_t)stride * a.x_stride;
    if constexpr (ADD) pr += (int64_t)stride * a.residual_stride;
  };
  // whether the wave has columns in its piece i: if not, nothing is drawn or worked out for it
  const uint32_t begin = WAVES > 1 ? __builtin_amdgcn_readfirstlane(wave * STRETCH) : 0;
  const auto used = [&](int i) { return (WAVES == 1 && i == 0) || begin + i * GROUP * V < a.width; };
  const auto fetch_affine = [&] {
    load_affine<V, A, R>(w, a.weight, a.narrow, first, GROUP * V, a.width, 1.f);
    load_affine<V, A, R>(b, a.bias, a.narrow, first, GROUP * V, a.width, 0.f);
    if constexpr (DROP && !ADD) { // what is kept is scaled with them
      scale_all(w, a.drop.scale);
      scale_all(b, a.drop.scale);
    }
    if constexpr (SHELVED) {
#pragma unroll
      for (int i = 0; i < ITEMS; i++)
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
          float4 *place = shelf + ((i * (V / 4) + q) * 2) * BLOCK + threadIdx.x; // no other lane's
          place[0] = make_float4(w[i].v[4 * q], w[i].v[4 * q + 1], w[i].v[4 * q + 2], w[i].v[4 * q + 3]);
          place[BLOCK] = make_float4(b[i].v[4 * q], b[i].v[4 * q + 1], b[i].v[4 * q + 2], b[i].v[4 * q + 3]);
        }
    }
  };
  if (STAYS && r0 < a.rows) {
    fetch(r0);
    fetch_affine();
  }
  for (int turn = 0; r0 < a.rows; r0 += stride, turn ^= 1) {
    if constexpr (!STAYS) {
      asm volatile("" : "+v"(first)); // no address is worked out, and kept, before the loop
      fetch(r0);
      fetch_affine();
    }
    Floats<V> f[ROWS][ITEMS];
#pragma unroll
    for (int k = 0; k < ROWS; k++)
#pragma unroll
      for (int i = 0; i < ITEMS; i++) {
        const uint32_t c = first + i * GROUP * V;
        f[k][i] = floats<V>(settled<V, R>(x[k][i], c, a.width));
        if constexpr (ADD) {
          const Floats<V> g = floats<V>(settled<V, R>(residual[k][i], c, a.width));
          if constexpr (DROP)
            if (used(i)) drop_columns(f[k][i], a.drop, step, quad + k * GROUPS * a.drop.quads + c / 4);
#pragma unroll
          for (int j = 0; j < V; j++) f[k][i].v[j] += g.v[j];
          store_columns<V, R>(ps + k * GROUPS * a.sum_stride, c, width(k, r0), f[k][i]);
        }
      }
    if (STAYS && r0 + stride < a.rows) fetch(r0 + stride);
    float sum[ROWS], square[ROWS], mean[ROWS], rstd[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      sum[k] = 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; i++)
#pragma unroll
        for (int j = 0; j < V; j++) sum[k] += f[k][i].v[j];
    }
    group_sums<GROUP>(sum);
    const float n = WAVES > 1 ? (float)min(a.width - min(a.width, wave * STRETCH), STRETCH) : 0.f;
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      mean[k] = WAVES > 1 ? sum[k] / fmaxf(n, 1.f) : sum[k] * a.inv_width;
      square[k] = 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; i++) {
        const uint32_t c = first + i * GROUP * V;
#pragma unroll
        for (int j = 0; j < V; j++) {
          // columns behind the end hold zeros and have to add nothing to the squares
          const float d = f[k][i].v[j] - ((R == Rows::kEven ? c : c + j) < a.width ? mean[k] : 0.f);
          square[k] = fmaf(d, d, square[k]);
          if constexpr (WAVES == 1) f[k][i].v[j] = d;
        }
      }
    }
    group_sums<GROUP>(square);
    if constexpr (WAVES > 1) {
      if (lane == 0) found[turn][wave] = make_float2(sum[0], square[0]);
      __syncthreads();
      // every lane takes one wave's
      const float2 other = found[turn][lane % WAVES];
      const float m = (float)min(a.width - min(a.width, lane % WAVES * STRETCH), STRETCH);
      mean[0] = group_sum<WAVES>(other.x) * a.inv_width;
      const float off = other.x / fmaxf(m, 1.f) - mean[0];
      square[0] = group_sum<WAVES>(fmaf(m * off, off, other.y));
#pragma unroll
      for (int i = 0; i < ITEMS; i++)
#pragma unroll
        for (int j = 0; j < V; j++) f[0][i].v[j] -= mean[0];
    }
#pragma unroll
    for (int k = 0; k < ROWS; k++) rstd[k] = rsqrtf(fmaf(square[k], a.inv_width, a.eps));
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
      const uint32_t c = first + i * GROUP * V;
      if constexpr (SHELVED) {
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
          const float4 *place = shelf + ((i * (V / 4) + q) * 2) * BLOCK + threadIdx.x, x4 = place[0], y4 = place[BLOCK];
          w[i].v[4 * q] = x4.x, w[i].v[4 * q + 1] = x4.y, w[i].v[4 * q + 2] = x4.z, w[i].v[4 * q + 3] = x4.w;
          b[i].v[4 * q] = y4.x, b[i].v[4 * q + 1] = y4.y, b[i].v[4 * q + 2] = y4.z, b[i].v[4 * q + 3] = y4.w;
        }
      }
      if (!used(i)) continue;
#pragma unroll
      for (int k = 0; k < ROWS; k++) {
#pragma unroll
        for (int j = 0; j < V; j++) f[k][i].v[j] = fmaf(f[k][i].v[j] * rstd[k], w[i].v[j], b[i].v[j]);
        if constexpr (DROP && !ADD) drop_columns<false>(f[k][i], a.drop, step, quad + k * GROUPS * a.drop.quads + c / 4);
        store_columns<V, R>(py + k * GROUPS * a.y_stride, c, width(k, r0), f[k][i]);
      }
    }
    if (threadIdx.x % LANES == 0) {
#pragma unroll
      for (int k = 0; k < ROWS; k++)
        if (width(k, r0)) {
          if (a.mean) a.mean[r0 + k * GROUPS] = mean[k];
          if (a.rstd) a.rstd[r0 + k * GROUPS] = rstd[k];
        }
    }
    quad += stride * a.drop.quads;
    py += (int64_t)stride * a.y_stride;
    if constexpr (ADD) ps += (int64_t)stride * a.sum_stride;
  }
}

template <typename S, typename A, bool ADD, bool DROP> void launch(const NormForward &p, hipStream_t s) {
  const bool held = rows_in_registers<S>(p.width, [&](auto rows, auto lanes, auto items) {
    constexpr Rows R = decltype(rows)::value;
    constexpr int LANES = decltype(lanes)::value, ITEMS = decltype(items)::value, BLOCK = block_of<LANES>;
    // Four rows at a time (two, if each is two pieces a lane) where the memory would wait for the lanes: they draw, convert two values
    // a register, or leave some of their loads empty.  us with one row and with four, 1.2e8 values: float to bfloat16, dropped, 16
    // columns 147, 126, 256 columns 152, 121, 37 columns 326, 209, 333 columns 224, 188; float, 37 columns 271, 191; bfloat16, 64
    // columns 87, 81, 333 columns 166, 107; a branch added, bfloat16, dropped, 37 columns 319, 280.  Elsewhere four are no better or
    // worse: float, 64 columns 157, 157, 256 columns 157, 165; a branch added, float and bfloat16, 256 columns 236, 245, bfloat16,
    // dropped, 16 columns 154, 161.
    constexpr bool FOUR = LANES <= kWave && ITEMS == 1 && (R != Rows::kEven || (!ADD && (DROP || sizeof(S) == 2)));
    constexpr int ROWS = FOUR ? 4 : LANES <= kWave && ITEMS == 2 && R == Rows::kRagged && !stays<S, LANES, ITEMS> ? 2 : 1, PER = BLOCK / LANES * ROWS;
    // Blocks that stay: as many per CU as fetch 16 KiB at a time, or sixteen where the draws' arithmetic wants them.  us for 1.2e8
    // values with 256, 512, 1024, 4096 blocks and with one for each row (chosen: *): float, 4096 columns 161*, 162, 165, 163, 176;
    // bfloat16, 2048 columns 166, 106, 82*, 87, 102, 8192 columns 81*, 82, 90, 85, 108; a branch added, float and bfloat16, 1024
    // columns 244*, 262, 256, 250, 241, 4096 columns 241*, 257, 255, 250, 250; float to bfloat16, dropped, 4096 columns 150, 121,
    // 127, 123*, 142.
    uint64_t most = (1u << 31) / BLOCK;
    if constexpr (stays<S, LANES, ITEMS>) {
      const uint64_t fetch = (uint64_t)PER * p.width * (ADD ? sizeof(A) + sizeof(S) : sizeof(S));
      most = 256 * (DROP && !ADD && !shelved<S, LANES, ITEMS> ? 16 : (16 * 1024 - 1) / fetch + 1);
    }
    const uint64_t blocks = std::min<uint64_t>((p.rows + PER - 1) / PER, most);
    hipLaunchKernelGGL((norm_rows<S, A, ADD, DROP, R, LANES, ITEMS, ROWS>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, p);
  });
  if (!held)
    hipLaunchKernelGGL((norm_wide<S, A, ADD, DROP>), dim3((unsigned)std::min<uint64_t>(p.rows, 1u << 20)), dim3(kWideBlock), 0, s, p);
  HCTR_HIP(hipGetLastError());
}

} // namespace

template <typename S, typename A> void launch_norm(const NormForward &p, bool add, bool dropped, hipStream_t s) {
  if (add) dropped ? launch<S, A, true, true>(p, s) : launch<S, A, true, false>(p, s);
  else dropped ? launch<S, A, false, true>(p, s) : launch<S, A, false, false>(p, s);
}

} // namespace hctr
