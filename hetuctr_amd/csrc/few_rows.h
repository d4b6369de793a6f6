// Products of a few rows (up to 32) with a matrix of weights, which is all that takes time: it is read once, straight into registers.
#pragma once
#include "matmul.h"

namespace hctr {

constexpr uint32_t kFewRows = 32;

// How many groups of 16 rows of weights a wave takes at a time: four, so that x, which every block reads, is not most of what goes through the
// caches, but two where that leaves CUs idle, and for the fewest rows, whose x is next to nothing, where it leaves few blocks for the last
// ones.  (us, bfloat16, with two and four: 16384 x 4096 twice, 1 row 46.9, 49.2, 16 rows 60.6, 51.1; 131072 x 4096, 1 row 223, 206,
// 16 rows 253, 201.)
inline int few_groups(size_t rows, size_t weights) {
  const size_t blocks = weights / 64;
  return blocks < 256 || (rows <= 4 && blocks < 1024) ? 2 : 4;
}

// ROWS (16 or 32) rows of x times GROUPS * 16 rows of weights, in groups of 16 that the caller says the places of.  A block's waves share out
// k; every wave has the fragments of kAhead steps under way, which lanes fetch from any address an element can have: as many as leave
// room for several blocks on a CU, which hide more than further steps of one would (32 rows and 131072 x 4096: 226 us with four steps, 206
// with two).  The waves' sums are joined through LDS, in pairs.
template <typename T, int ROWS, int GROUPS> struct FewRows {
  static constexpr int kWaves = 8, kThreads = kWaves * kWave, kTiles = ROWS / 16, kGroups = GROUPS, kWeights = kGroups * 16, kAhead = kTiles == 1 && GROUPS == 2 ? 8 : kTiles == 1 ? 4 : 2,
                       kPitch = kWeights + 4;
  typedef float Sums[ROWS][kPitch];
  typedef typename Packed<T, kVec<T>>::memory Loose;
  static constexpr uint32_t kStepK = 64 / sizeof(T);

  // sums[0][r][c] = sum over k of x's row r times row c % 16 of group c / 16, which lies at w[c / 16], and of which left[c / 16] rows (one at
  // least) are there: what is summed for others, and for rows of x behind its last, is anything.  Ends with a barrier.
  static __device__ __forceinline__ void run(const T *x, int64_t x_stride, uint32_t rows, const T *const (&groups)[kGroups], const uint32_t (&left)[kGroups],
                                             const int64_t (&stride)[kGroups], uint32_t k, Sums *sums) {
    const uint32_t l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    f32x4 sum[kTiles][kGroups];
#pragma unroll
    for (int i = 0; i < kTiles; i++)
#pragma unroll
      for (int j = 0; j < kGroups; j++) sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const T *w[kGroups], *at[kTiles];
#pragma unroll
    for (int j = 0; j < kGroups; j++) w[j] = groups[j] + (int64_t)min(l % 16, left[j] - 1) * stride[j];
#pragma unroll
    for (int i = 0; i < kTiles; i++) at[i] = x + (int64_t)min(i * 16 + l % 16, rows - 1) * x_stride;
    const uint32_t lane_k = l / 16 * kVec<T>, steps = k / kStepK, each = (steps + kWaves - 1) / kWaves;
    const uint32_t from = min(steps, wave * each), to = min(steps, from + each);
    const auto turn = [&](auto ahead, uint32_t step) {
      constexpr int N = decltype(ahead)::value;
      Fragment<T> fw[N][kGroups], fx[N][kTiles];
#pragma unroll
      for (int a = 0; a < N; a++) {
        const uint32_t c = (step + a) * kStepK + lane_k;
#pragma unroll
        for (int j = 0; j < kGroups; j++) fw[a][j].v = *(const Loose *)(w[j] + c);
#pragma unroll
        for (int i = 0; i < kTiles; i++) fx[a][i].v = *(const Loose *)(at[i] + c);
      }
      __builtin_amdgcn_sched_barrier(0); // all loads first, whatever registers that takes
#pragma unroll
      for (int a = 0; a < N; a++)
#pragma unroll
        for (int i = 0; i < kTiles; i++)
#pragma unroll
          for (int j = 0; j < kGroups; j++) sum[i][j] = multiply<T>(fw[a][j], fx[a][i], sum[i][j]);
    };
    uint32_t step = from;
    for (; step + kAhead <= to; step += kAhead) turn(std::integral_constant<int, kAhead>(), step);
    for (; step < to; step++) turn(std::integral_constant<int, 1>(), step);
    if (wave == kWaves - 1 && steps * kStepK < k) { // what is left of k, zeros behind it
      const uint32_t c = steps * kStepK + lane_k;
      const auto rest = [&](const T *row) { return settled<kVec<T>, Rows::kLong>(load_raw<kVec<T>, Rows::kLong>(row, c, k), c, k); };
      Fragment<T> fw[kGroups], fx;
#pragma unroll
      for (int j = 0; j < kGroups; j++) fw[j].v = rest(w[j]);
#pragma unroll
      for (int i = 0; i < kTiles; i++) {
        fx.v = rest(at[i]);
#pragma unroll
        for (int j = 0; j < kGroups; j++) sum[i][j] = multiply<T>(fw[j], fx, sum[i][j]);
      }
    }
#pragma unroll
    for (uint32_t n = kWaves / 2; n; n /= 2) {
      const auto place = [&](uint32_t of, int i, int j) { return (f32x4 *)&sums[of][i * 16 + l % 16][j * 16 + l / 16 * 4]; };
      if (n < kWaves / 2) __syncthreads(); // what was written before is read
      if (wave >= n && wave < 2 * n)
#pragma unroll
        for (int i = 0; i < kTiles; i++)
#pragma unroll
          for (int j = 0; j < kGroups; j++) *place(wave - n, i, j) = sum[i][j];
      __syncthreads();
      if (wave < n)
#pragma unroll
        for (int i = 0; i < kTiles; i++)
#pragma unroll
          for (int j = 0; j < kGroups; j++) {
            sum[i][j] += *place(wave, i, j);
            if (n == 1) *place(0, i, j) = sum[i][j];
          }
    }
    __syncthreads();
  }
  static constexpr int kSums = kWaves / 2; // that `sums` has room for
};

} // namespace hctr
