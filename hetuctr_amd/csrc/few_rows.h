// Products of a few rows (up to 64) with a matrix of weights, which is all that takes time: it is read once, straight into registers.
#pragma once
#include "matmul.h"

namespace hctr {

constexpr uint32_t kFewRows = 64;

// ROWS (16, 32 or 64) rows of x times 32 rows of weights: 16 of each of two matrices, or 32 of one.  A block's waves share out k; every
// wave has the fragments of kAhead steps under way, which lanes fetch from any address an element can have.  The waves' sums
// are joined in LDS, in order.
template <typename T, int ROWS> struct FewRows {
  static constexpr int kWaves = 8, kThreads = kWaves * kWave, kTiles = ROWS / 16, kAhead = ROWS == 64 ? 2 : 4, kPitch = 36;
  typedef float Sums[ROWS][kPitch];
  typedef typename Packed<T, kVec<T>>::memory Loose;
  static constexpr uint32_t kStepK = 64 / sizeof(T);

  // sums[r][c] = sum over k of x's row r times row c of `first`, or, from c = 16 on, row c - 16 of `second`; of the two first_left and
  // second_left rows are there (what is summed for others, and for rows of x behind its last, is anything).  Ends with a barrier.
  static __device__ __forceinline__ void run(const T *x, int64_t x_stride, uint32_t rows, const T *first, const T *second, uint32_t first_left,
                                             uint32_t second_left, int64_t first_stride, int64_t second_stride, uint32_t k, Sums *waves_sums) {
    const uint32_t l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    f32x4 sum[kTiles][2];
#pragma unroll
    for (int i = 0; i < kTiles; i++) sum[i][0] = sum[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    const T *w[2] = {first + (int64_t)min(l % 16, first_left - 1) * first_stride, second + (int64_t)min(l % 16, second_left - 1) * second_stride};
    const T *at[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; i++) at[i] = x + (int64_t)min(i * 16 + l % 16, rows - 1) * x_stride;
    const uint32_t lane_k = l / 16 * kVec<T>, steps = k / kStepK, each = (steps + kWaves - 1) / kWaves;
    const uint32_t from = min(steps, wave * each), to = min(steps, from + each);
    const auto turn = [&](auto ahead, uint32_t step) {
      constexpr int N = decltype(ahead)::value;
      Fragment<T> fw[N][2], fx[N][kTiles];
#pragma unroll
      for (int a = 0; a < N; a++) {
        const uint32_t c = (step + a) * kStepK + lane_k;
#pragma unroll
        for (int j = 0; j < 2; j++) fw[a][j].v = *(const Loose *)(w[j] + c);
#pragma unroll
        for (int i = 0; i < kTiles; i++) fx[a][i].v = *(const Loose *)(at[i] + c);
      }
#pragma unroll
      for (int a = 0; a < N; a++)
#pragma unroll
        for (int i = 0; i < kTiles; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) sum[i][j] = multiply<T>(fw[a][j], fx[a][i], sum[i][j]);
    };
    uint32_t step = from;
    for (; step + kAhead <= to; step += kAhead) turn(std::integral_constant<int, kAhead>(), step);
    for (; step < to; step++) turn(std::integral_constant<int, 1>(), step);
    if (wave == kWaves - 1 && steps * kStepK < k) { // what is left of k, zeros behind it
      const uint32_t c = steps * kStepK + lane_k;
      const auto rest = [&](const T *row) { return settled<kVec<T>, Rows::kLong>(load_raw<kVec<T>, Rows::kLong>(row, c, k), c, k); };
      Fragment<T> fw[2], fx;
#pragma unroll
      for (int j = 0; j < 2; j++) fw[j].v = rest(w[j]);
#pragma unroll
      for (int i = 0; i < kTiles; i++) {
        fx.v = rest(at[i]);
#pragma unroll
        for (int j = 0; j < 2; j++) sum[i][j] = multiply<T>(fw[j], fx, sum[i][j]);
      }
    }
#pragma unroll
    for (int i = 0; i < kTiles; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) *(f32x4 *)&waves_sums[wave][i * 16 + l % 16][j * 16 + l / 16 * 4] = sum[i][j];
    __syncthreads();
  }
  // columns c .. c + 3 of row r, all of k
  static __device__ __forceinline__ f32x4 joined(const Sums *waves_sums, uint32_t r, uint32_t c) {
    f32x4 s = *(const f32x4 *)&waves_sums[0][r][c];
#pragma unroll
    for (int w = 1; w < kWaves; w++) s += *(const f32x4 *)&waves_sums[w][r][c];
    return s;
  }
};

} // namespace hctr
