// Device code that layer normalisation and its gradient share.
#pragma once
#include <type_traits>

#include "dense.h"

namespace hctr {

// The sum of v over each group of LANES neighbouring lanes, the same bits in all of them: every step adds what two halves
// hold, in either order.  Quads and rows of 16 lanes take it in data-parallel moves, wider groups by swapping rows or halves
// of the wave between two registers; none of it goes through LDS.
template <int LANES> __device__ __forceinline__ float group_sum(float v) {
  static_assert(LANES >= 2 && LANES <= kWave && (LANES & (LANES - 1)) == 0, "lanes of a group");
  const auto moved = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += moved(v, std::integral_constant<int, 0xB1>()); // lane ^ 1
  if constexpr (LANES >= 4) v += moved(v, std::integral_constant<int, 0x4E>()); // lane ^ 2
  if constexpr (LANES >= 8) v += moved(v, std::integral_constant<int, 0x141>()); // 7 - lane, of 8
  if constexpr (LANES >= 16) v += moved(v, std::integral_constant<int, 0x140>()); // 15 - lane, of 16
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned low = r[0], high = r[1]; // (the cast of an element itself takes the first one)
    v = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
  }
  if constexpr (LANES >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned low = r[0], high = r[1]; // (the cast of an element itself takes the first one)
    v = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
  }
  return v;
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

// columns of weight or bias: `narrow`, they are of type A, else float; without any, `none`
template <int V, typename A>
__device__ __forceinline__ Floats<V> load_affine(const void *p, bool narrow, uint32_t c, uint32_t width, float none) {
  if (!p) {
    Floats<V> f;
#pragma unroll
    for (int j = 0; j < V; j++) f.v[j] = none;
    return f;
  }
  return narrow ? load_columns<V, false>((const A *)p, c, width) : load_columns<V, false>((const float *)p, c, width);
}

// threads of a block whose rows are held by LANES lanes each: 256, or those of one row if they are more than a wave
template <int LANES> constexpr int block_of = LANES <= kWave ? 256 : LANES;

// f(lanes, items), constants, for the lanes that hold a row of `width` columns in registers, and the pieces of kVec<S> columns that
// each of them holds: as few lanes as can read the row at once, up to a wave of them, then up to 16 columns a lane (32 do
// not fit beside weight and bias into the 128 registers of a block of 1024).  False: the row is wider than 16384 columns.
template <typename S, typename F> bool rows_in_registers(uint32_t width, F &&f) {
  constexpr int MOST = 16 / kVec<S>;
  using std::integral_constant;
  const uint32_t pieces = div_up(width, kVec<S>);
  if (pieces <= 2) f(integral_constant<int, 2>(), integral_constant<int, 1>());
  else if (pieces <= 4) f(integral_constant<int, 4>(), integral_constant<int, 1>());
  else if (pieces <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (pieces <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (pieces <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (pieces <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (pieces <= 128) f(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (pieces <= 64 * MOST) f(integral_constant<int, 64>(), integral_constant<int, MOST>());
  else if (pieces <= 128 * MOST) f(integral_constant<int, 128>(), integral_constant<int, MOST>());
  else if (pieces <= 256 * MOST) f(integral_constant<int, 256>(), integral_constant<int, MOST>());
  else if (pieces <= 512 * MOST) f(integral_constant<int, 512>(), integral_constant<int, MOST>());
  else if (pieces <= 1024 * MOST) f(integral_constant<int, 1024>(), integral_constant<int, MOST>());
  else return false;
  return true;
}

} // namespace hctr
