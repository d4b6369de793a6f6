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

constexpr int kWideBlock = 256; // threads of a block that reads its row again and again

// threads of a block whose rows are held by LANES lanes each: 256, or those of one row if they are more than a wave
template <int LANES> constexpr int block_of = LANES <= kWave ? 256 : LANES;

// f(rows, lanes, items), constants: how rows of `width` columns are read, the lanes that hold one in registers, and the pieces of
// kVec<S> columns that each of them holds: as few lanes as can read the row at once, up to a wave of them, then up to 16
// columns a lane (32 do not fit beside weight and bias into the 128 registers of a block of 1024).  False: the row is wider
// than 16384 columns.
template <Rows R, typename S, typename F> bool lanes_of_rows(uint32_t pieces, F &&f) {
  constexpr int MOST = 16 / kVec<S>;
  constexpr std::integral_constant<Rows, R> rows;
  using std::integral_constant;
  if (pieces <= 2) f(rows, integral_constant<int, 2>(), integral_constant<int, 1>());
  else if (pieces <= 4) f(rows, integral_constant<int, 4>(), integral_constant<int, 1>());
  else if (pieces <= 8) f(rows, integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (pieces <= 16) f(rows, integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (pieces <= 32) f(rows, integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (pieces <= 64) f(rows, integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (pieces <= 128) f(rows, integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (pieces <= 64 * MOST) f(rows, integral_constant<int, 64>(), integral_constant<int, MOST>());
  else if (pieces <= 128 * MOST) f(rows, integral_constant<int, 128>(), integral_constant<int, MOST>());
  else if (pieces <= 256 * MOST) f(rows, integral_constant<int, 256>(), integral_constant<int, MOST>());
  else if (pieces <= 512 * MOST) f(rows, integral_constant<int, 512>(), integral_constant<int, MOST>());
  else if (pieces <= 1024 * MOST) f(rows, integral_constant<int, 1024>(), integral_constant<int, MOST>());
  else return false;
  return true;
}
template <typename S, typename F> bool rows_in_registers(uint32_t width, F &&f) {
  const uint32_t pieces = div_up(width, kVec<S>);
  return width % kVec<S> ? lanes_of_rows<Rows::kRagged, S>(pieces, f) : lanes_of_rows<Rows::kEven, S>(pieces, f);
}

// Blocks of the gradient's kernels, each of which writes a row of sums for weight and bias: few of them, since the sums are written
// and read beside the data, but enough loads under way to fill the memory, and a multiple of the 256 CUs.  us on an MI355X
// with 256, 512, 768, 1280 blocks, 2^27 values: float, 64 columns 411, 283, 277, 302; float and bfloat16, dropped, 128
// columns -, 262, 230, 256; a branch added (its sum's gradient is loaded ahead too) 64 columns -, 356, 385, 425; float, 2048
// columns 308, 274, 283, 298; 4096 columns 276, 281, 284, 284; 4096 rows of 8192 halves 52, 66, 78, 103.  Narrow rows that
// leave lanes idle want more: 37 columns, dropped, -, 647, 493, 351, a branch added -, 740, 560, 470.
constexpr unsigned norm_grad_blocks(uint64_t rows, uint32_t width, bool add, bool ragged) {
  const unsigned most = width > 4096 ? 256 : width > 1024 ? 512 : ragged ? 1280 : add ? 512 : 768;
  return rows < most ? (unsigned)rows : most;
}

// The kernels' launches, one instance per pair of types in a file of its own (layer_norm_*.hip); add, dropped: which of the four
// forms.  The gradient's returns how many rows of sums it leaves in p.partial.
template <typename S, typename A> void launch_norm(const NormForward &p, bool add, bool dropped, hipStream_t s);
template <typename S, typename A> unsigned launch_norm_grad(const NormBackward &p, bool add, bool dropped, hipStream_t s);

} // namespace hctr
