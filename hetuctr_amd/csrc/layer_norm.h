// Device code that layer normalisation and its gradient share.
#pragma once
#include <algorithm>
#include <type_traits>

#include "dense.h"

namespace hctr {

// The sums of v[0], v[1], .. over each group of LANES neighbouring lanes, the same bits in all of them: every step adds what two
// halves hold, in either order.  Quads and rows of 16 lanes take it in data-parallel moves, wider groups by swapping rows or
// halves of the wave between two registers; none of it goes through LDS, and the sums fill each other's waits.
template <int LANES, int N> __device__ __forceinline__ void group_sums(float (&v)[N]) {
  static_assert(LANES >= 2 && LANES <= kWave && (LANES & (LANES - 1)) == 0, "lanes of a group");
  const auto move = [&](auto ctrl) {
#pragma unroll
    for (int i = 0; i < N; i++)
      v[i] += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v[i]), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  // (r[0] and r[1] go through integers of their own: the cast of an element itself takes the first one)
  const auto swap = [&](auto f) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const auto r = f(__builtin_bit_cast(unsigned, v[i]));
      const unsigned low = r[0], high = r[1];
      v[i] = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
    }
  };
  move(std::integral_constant<int, 0xB1>());                            // lane ^ 1
  if constexpr (LANES >= 4) move(std::integral_constant<int, 0x4E>());  // lane ^ 2
  if constexpr (LANES >= 8) move(std::integral_constant<int, 0x141>()); // 7 - lane, of 8
  if constexpr (LANES >= 16) move(std::integral_constant<int, 0x140>()); // 15 - lane, of 16
  if constexpr (LANES >= 32) swap([](unsigned x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  if constexpr (LANES >= 64) swap([](unsigned x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
}
template <int LANES> __device__ __forceinline__ float group_sum(float v) {
  float one[1] = {v};
  group_sums<LANES>(one);
  return one[0];
}

// The sum of v over the NT threads of a block, the same in all of them.  `smem` needs NT / 64 floats; the barriers inside keep
// one sum's words apart from the next one's.
template <int NT> __device__ __forceinline__ float block_sum(float v, float *smem) {
  v = group_sum<kWave>(v);
  __syncthreads();
  if (lane_id() == 0) smem[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < NT / kWave; i++) v += smem[i];
  return v;
}

// (first + group) * stride, where first and stride are the same in all lanes, and the group is too if UNIFORM.  The lanes are spared
// the product of two 64-bit numbers that scalar arithmetic can do (it takes them nine multiplications' time, as much as a
// round of the draws), and kept apart, so that the compiler does not put the two products together again.
template <bool UNIFORM> __device__ __forceinline__ int64_t rows_away(uint64_t first, uint32_t group, int64_t stride) {
  int64_t own = (int64_t)group * stride;
  if constexpr (UNIFORM) asm("" : "+s"(own));
  else asm("" : "+v"(own));
  return (int64_t)first * stride + own;
}

// Columns of weight or bias, ITEMS pieces that lie `apart` columns from each other: `narrow`, they are of type A, else float;
// without any, `none`.
template <int V, typename A, Rows R, int ITEMS>
__device__ __forceinline__ void load_affine(Floats<V> (&f)[ITEMS], const void *p, bool narrow, uint32_t c, uint32_t apart, uint32_t width,
                                            float none) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < ITEMS; i++)
#pragma unroll
      for (int j = 0; j < V; j++) f[i].v[j] = none;
  } else if (narrow) {
#pragma unroll
    for (int i = 0; i < ITEMS; i++) f[i] = load_columns<V, R, false>((const A *)p, c + i * apart, width);
  } else {
#pragma unroll
    for (int i = 0; i < ITEMS; i++) f[i] = load_columns<V, R, false>((const float *)p, c + i * apart, width);
  }
}

template <int V, int ITEMS> __device__ __forceinline__ void scale_all(Floats<V> (&f)[ITEMS], float scale) {
#pragma unroll
  for (int i = 0; i < ITEMS; i++)
#pragma unroll
    for (int j = 0; j < V; j++) f[i].v[j] *= scale;
}

// threads of a block that reads its row again and again; the gradient has few blocks, for the sake of their sums
constexpr int kWideBlock = 256, kWideGradBlock = 1024;

// threads of a block whose rows are held by LANES lanes each: 256, or those of one row if they are more than a wave
template <int LANES> constexpr int block_of = LANES <= kWave ? 256 : LANES;

// The lanes that hold a row of `width` columns in registers, and the pieces of V columns that each of them holds: as few lanes as
// can read the row at once, up to a wave of them; then up to 16 columns a lane (32 do not fit beside weight and bias into the
// 128 registers of a block of 1024).  A block that shares a row has four waves at least: with two, half of a CU's four SIMDs
// had no work (the gradient of 2^27 values, a branch added and dropped, 2048 columns: 405 us with 128 lanes, 354 with 256).
// No lanes: the row is wider than 16384 columns.
struct Held {
  int lanes, items;
};
constexpr Held held_by(uint32_t width, int V) {
  const uint32_t pieces = (width - 1) / V + 1;
  const int most = 16 / V;
  for (int lanes = 2; lanes <= kWave; lanes *= 2)
    if (pieces <= (uint32_t)lanes) return {lanes, 1};
  for (int items = 2; items <= most; items *= 2)
    if (pieces <= (uint32_t)(kWave * items)) return {kWave, items};
  if (pieces <= (uint32_t)(256 * most / 2)) return {256, most / 2};
  for (int lanes = 256; lanes <= 1024; lanes *= 2)
    if (pieces <= (uint32_t)(lanes * most)) return {lanes, most};
  return {0, 0};
}
// f(rows, lanes, items), constants, for how rows of `width` columns are read and held; false: they are not held
template <typename S, typename F> bool rows_in_registers(uint32_t width, F &&f) {
  constexpr int V = kVec<S>, MOST = 16 / V;
  const Held h = held_by(width, V);
  const auto with = [&](auto lanes, auto items) {
    if (h.lanes != lanes || h.items != items) return false;
    // (what more than two lanes hold has more than two pieces)
    if (width % V) f(std::integral_constant<Rows, decltype(lanes)::value == 2 ? Rows::kTiny : Rows::kRagged>(), lanes, items);
    else f(std::integral_constant<Rows, Rows::kEven>(), lanes, items);
    return true;
  };
  using std::integral_constant;
  constexpr integral_constant<int, 1> one;
  constexpr integral_constant<int, MOST / 2> half;
  constexpr integral_constant<int, MOST> most;
  constexpr integral_constant<int, 64> wave;
  constexpr integral_constant<int, 256> four;
  bool done = with(integral_constant<int, 2>(), one) || with(integral_constant<int, 4>(), one) || with(integral_constant<int, 8>(), one) ||
              with(integral_constant<int, 16>(), one) || with(integral_constant<int, 32>(), one) || with(wave, one) || with(wave, most) ||
              with(four, half) || with(four, most) || with(integral_constant<int, 512>(), most) || with(integral_constant<int, 1024>(), most);
  if constexpr (MOST > 2) done = done || with(wave, half);
  return done;
}

// Blocks of the gradient's kernels, each of which writes a row of sums for weight and bias: as many per CU as fetch 17 KiB at a
// time (bytes: of a column's values, read), so few that the memory sees long stretches and the rows of sums are little beside the data, at
// least one and at most eight.  us on an MI355X for 1.2e8 values with 256, 512, 768, 1024 blocks (chosen: *): float, 64 columns
// 360, 249, 243*, 255; 1024 columns 235*, 255, 248, 254; bfloat16, 4096 columns 131, 125*, 136, 140; float and bfloat16, dropped, 128
// columns 357, 228, 200*, 209; a branch added, 37 columns 735, 465, 406*, 462, 64 columns 420, 315*, 338, 368, 512 columns 311*, 339,
// 354, 374, 2048 columns 312*, 324, 360, 370; 4096 rows of 8192 halves 44*, 50, 62, 68.
// The rule does not know how many blocks fit beside each other: where values are drawn behind the norm the kernel has 105 or 107
// registers, so four do, and a fifth and sixth start when others are done.  That costs ragged rows a fifth: float and bfloat16,
// dropped, with 3 to 6 per CU, 33 columns 327, 282, 362, 345*, 37 columns 301, 270, 340*, 324, 65 columns 332, 286, 374, 356*; bfloat16,
// dropped, 33 columns 235, 195, 233*, 213.
inline unsigned norm_grad_blocks(uint64_t rows, uint32_t width, int V, int bytes) {
  const Held h = held_by(width, V);
  const uint64_t groups = h.lanes && h.lanes < 256 ? 256 / h.lanes : 1, fetch = groups * width * bytes;
  const uint64_t per_cu = std::min<uint64_t>((17 * 1024 - 1) / fetch + 1, 8);
  return (unsigned)std::min(256 * per_cu, (rows + groups - 1) / groups);
}

// The kernels' launches, one instance per pair of types in a file of its own (layer_norm_*.hip); add, dropped: which of the four
// forms.  The gradient's returns how many rows of sums it leaves in p.partial.
template <typename S, typename A> void launch_norm(const NormForward &p, bool add, bool dropped, hipStream_t s);
template <typename S, typename A> unsigned launch_norm_grad(const NormBackward &p, bool add, bool dropped, hipStream_t s);

} // namespace hctr
