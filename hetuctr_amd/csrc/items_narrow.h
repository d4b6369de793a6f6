// Cross entropy over many items where rows are narrow: kernels of items.h for one 16-bit type.
//
// Of rows of 128 columns a matrix of logits, or of their slopes, is larger than all that is made of it (4096 rows, a million items: 8.2 GB to
// write once and read twice), and the arithmetic on a logit costs as much as the product that makes it.  So the gradients make the logits
// again and keep nothing of them: a wave owns rows of one matrix as fragments in registers, the rows of the other go through LDS, and
// the slopes of 32 of them are, as they lie in the registers behind the first product, the fragments of the second: a lane holds one
// owned row and 4 + 4 of the others, which the second product takes as its k, in whatever order, if the other operand comes in the same
// one.  That is the same tile in LDS, read across.
//
// Bound by the vector units: forward an exponential (a quarter of the others' rate) and four instructions a logit, 81 % of the cycles beside 40 %
// in the matrix cores.  4096 rows, a million items of 128 bfloat16: 1.17 ms (0.89 PFLOP/s), by tiles, each of which joins lanes and waves
// for itself, 2.75; dx 2.0 and the weights' gradient 2.1, with d in memory 8.9 together.  Of 32 columns 0.77, 0.90 and 0.99.
#pragma once
#include "items.h"
#include "items_tail.h"

namespace hctr {

enum class Narrow { kForward, kDx, kDweight };

// rows of `width` columns, up to KS * 32
template <typename T, int KS> struct NarrowTiles {
  static constexpr int kThrough = 64, kLine = KS * 64, kPieces = KS * 4, kPasses = kThrough * kPieces / 256;
  static_assert(kPasses >= 1);
  static constexpr uint32_t kBytes = kThrough * kLine;
  // 16 rows' pieces lie in different banks.  32 bytes of 16 rows, read across, do two by two in the same ones: neighbours have the same two pieces, which
  // costs a third of the cycles with reads in the gradients.  (With the row's bits rotated by one none would, and took as long: 4096 rows, a
  // million items, 128 columns 4066 to 4087 us either way, 64 columns 2651 and 2674.)
  static __device__ __forceinline__ uint32_t placed(uint32_t row, uint32_t piece) { return piece ^ (row / (4 / KS) & (kPieces - 1)); }
  uint32_t offset; // the order of a row's pieces is that of the rows kRows further down
  static constexpr uint32_t kRows = 256 / kPieces;
  __device__ __forceinline__ void init(uint32_t stride, uint32_t width) {
    const uint32_t line = threadIdx.x / kPieces, piece = placed(line, threadIdx.x % kPieces);
    offset = piece * 8 < width ? line * stride + piece * 16 : kNowhere;
  }
  // `there`: rows from the tile's first one on
  __device__ __forceinline__ void load(const char *from, int64_t stride, uint32_t there, uint32_t lds) const {
    const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * (kWave * 16);
#pragma unroll
    for (uint32_t i = 0; i < kPasses; i++) {
      uint32_t o = offset;
      if (there < kThrough) o = i * kRows + threadIdx.x / kPieces < there ? o : kNowhere;
      load_to_lds(buffer_at(from + (int64_t)(i * kRows) * stride), o, to + i * (256 * 16));
    }
  }
  // Where a lane's part of the tile's first fragment along the rows, and across them, lies.  Those of other pieces lie at the same place with
  // some bits turned over, those of other rows (16 further down, where the order is the same) a fixed number of bytes behind: kept
  // as such, they are an instruction each, and not a register each throughout the loop.
  static __device__ __forceinline__ uint32_t along_at() {
    const uint32_t l = lane_id();
    return l % 16 * kLine + placed(l % 16, l / 16) * 16;
  }
  static __device__ __forceinline__ uint32_t across_at() {
    const uint32_t l = lane_id(), row = l / 16 * 4 + l % 16 / 4;
    return row * kLine + placed(row, l % 4 / 2) * 16 + l % 2 * 8;
  }
  // rows r0 .. r0 + 15 of the tile, as Fragment lies: lane l has row l % 16 and of its columns the eight from (kk * 4 + l / 16) * 8 on
  static __device__ __forceinline__ Fragment<T> along(uint32_t at, uint32_t r0, uint32_t kk) {
    Fragment<T> f;
    f.v = *(const __attribute__((address_space(3))) typename Fragment<T>::type *)(uintptr_t)((at ^ kk * 64) + r0 * kLine);
    return f;
  }
  // columns c * 16 .. c * 16 + 15 across rows r0 .. r0 + 31: lane l has column l % 16, rows r0 + l / 16 * 4 + 0 .. 3 and those 16 further down
  static __device__ __forceinline__ Fragment<T> across(uint32_t at, uint32_t r0, uint32_t c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    s4 h[2];
#pragma unroll
    for (int j = 0; j < 2; j++) h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(uintptr_t)((at ^ c * 32) + (r0 + j * 16) * kLine));
    Fragment<T> f;
    f.v = __builtin_bit_cast(typename Fragment<T>::type, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    return f;
  }
};

// Owned rows of a wave, in 16s: of 128 columns the sums of 48 rows, the rows themselves and the logits of 32 others fit into half of a
// SIMD's registers, so that two waves can share it, and one's exponentials run beside the other's products.
template <int KS, Narrow MODE> constexpr int kOwned = MODE != Narrow::kForward && KS == 4 ? 3 : 4;

template <typename T, int KS, Narrow MODE>
__global__ __launch_bounds__(256, narrow_share(KS * 32, MODE != Narrow::kForward)) void items_narrow(ItemsNarrow p) {
  typedef NarrowTiles<T, KS> N;
  constexpr int OI = kOwned<KS, MODE>, J = MODE == Narrow::kForward ? 4 : 2;
  constexpr bool WEIGHT = MODE == Narrow::kDweight;
  __shared__ __attribute__((aligned(1024))) char tiles[2 * N::kBytes];
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)tiles, l = lane_id(), wave = threadIdx.x / kWave;
  const uint32_t count = min(p.rows, *p.taken.count);
  const uint32_t owned = WEIGHT ? p.items : count, through = WEIGHT ? count : p.items;
  const uint32_t owners = (owned + OI * 64 - 1) / (OI * 64), live = owners * p.ranges;
  if (blockIdx.x >= live) return;
  uint32_t owner, range;
  tile_of(blockIdx.x, live, owners, p.ranges, owners, owner, range);
  const uint32_t first = owner * (OI * 64) + wave * (OI * 16);
  const char *own = WEIGHT ? p.weight : p.x, *other = WEIGHT ? p.x : p.weight;
  const int64_t own_stride = WEIGHT ? p.weight_stride : p.x_stride, stride = WEIGHT ? p.x_stride : p.weight_stride;

  // Of two waves that share a SIMD one goes first, so that they do not do the same at the same time: by the number that the hardware gave it
  // (us, weights' gradient: 4096 rows and a million items 2236 -> 2136, 65536 and 20000 956 -> 865; the others the same or 1 % slower).
  if (WEIGHT && __builtin_amdgcn_s_getreg(3 << 11 | 4) & 1) __builtin_amdgcn_s_setprio(1);
  Fragment<T> mine[OI][KS];
  float own_bias[OI], lse[OI], dloss[OI];
  uint32_t target[OI];
#pragma unroll
  for (int i = 0; i < OI; i++) {
    const uint32_t r = first + i * 16 + l % 16;
#pragma unroll
    for (int kk = 0; kk < KS; kk++) {
      const uint32_t c = (kk * 4 + l / 16) * 8;
      mine[i][kk].v = (T)0;
      if (r < owned && c < p.width) mine[i][kk].v = *(const typename Fragment<T>::type *)(own + (int64_t)r * own_stride + c * 2);
    }
    if constexpr (MODE == Narrow::kDx) {
      lse[i] = r < owned ? p.taken.lse[r] : kInfinity;
      dloss[i] = r < owned ? p.taken.dloss[r] * p.taken.scale[0] : 0.f;
      target[i] = r < owned ? p.taken.target[r] : kNoItem;
    }
    if constexpr (WEIGHT) own_bias[i] = r < owned ? p.taken.bias[r] : -kInfinity;
  }
  const float scale = MODE == Narrow::kForward ? 1.f : p.taken.scale[0];

  f32x4 out[OI][2 * KS] = {};
  float most[OI], total[OI] = {};
#pragma unroll
  for (int i = 0; i < OI; i++) most[i] = kLowest;

  const uint32_t all = (through + N::kThrough - 1) / N::kThrough, each = (all + p.ranges - 1) / p.ranges;
  const uint32_t begin = min(all, range * each), end = min(all, begin + each);
  N n;
  n.init((uint32_t)stride, p.width);
  const auto load = [&](uint32_t tile, uint32_t stage) { n.load(other + (int64_t)tile * (N::kThrough * stride), stride, through - tile * N::kThrough, lds + stage * N::kBytes); };
  if (begin < end) load(begin, 0);
  for (uint32_t tile = begin; tile < end; tile++) {
    tiles_ready<0>();
    const uint32_t stage = (tile - begin) & 1;
    uint32_t along = lds + stage * N::kBytes + N::along_at(), across = lds + stage * N::kBytes + N::across_at();
    asm("" : "+v"(along), "+v"(across));
    if (tile + 1 < end) load(tile + 1, stage ^ 1);
#pragma unroll
    for (int half = 0; half < 4 / J; half++) {
      const uint32_t r0 = half * (J * 16), s0 = tile * N::kThrough + r0 + l / 16 * 4; // the lane's first of the others
      f32x4 sum[OI][J] = {};
#pragma unroll
      for (int kk = 0; kk < KS; kk++) {
        Fragment<T> f[J];
#pragma unroll
        for (int j = 0; j < J; j++) f[j] = N::along(along, r0 + j * 16, kk);
#pragma unroll
        for (int i = 0; i < OI; i++)
#pragma unroll
          for (int j = 0; j < J; j++) sum[i][j] = multiply<T>(f[j], mine[i][kk], sum[i][j]);
      }
      if constexpr (MODE == Narrow::kForward) {
        f32x4 bias[J];
#pragma unroll
        for (int j = 0; j < J; j++) bias[j] = *(const f32x4 *)(p.taken.bias + s0 + j * 16);
#pragma unroll
        for (int i = 0; i < OI; i++) {
          float top = most[i];
#pragma unroll
          for (int j = 0; j < J; j++) {
#pragma unroll
            for (int e = 0; e < 4; e++) sum[i][j][e] = __builtin_fmaf(sum[i][j][e], kLog2E, bias[j][e]);
#pragma unroll
            for (int e = 0; e < 4; e += 2) top = fmaxf(fmaxf(top, sum[i][j][e]), sum[i][j][e + 1]);
          }
          float s = total[i] * __builtin_amdgcn_exp2f(most[i] - top);
#pragma unroll
          for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s += __builtin_amdgcn_exp2f(sum[i][j][e] - top);
          most[i] = top, total[i] = s;
        }
      } else {
        if constexpr (MODE == Narrow::kDx) {
          f32x4 bias[J];
#pragma unroll
          for (int j = 0; j < J; j++) bias[j] = *(const f32x4 *)(p.taken.bias + s0 + j * 16);
#pragma unroll
          for (int i = 0; i < OI; i++) {
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
              for (int e = 0; e < 4; e++) sum[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sum[i][j][e] - lse[i], kLog2E, bias[j][e])) * dloss[i];
            // (a target is among these for one row in many)
            if (__ballot(target[i] - (s0 - l / 16 * 4) < J * 16))
#pragma unroll
              for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum[i][j][e] -= target[i] - s0 == (uint32_t)(j * 16 + e) ? dloss[i] : 0.f;
          }
        } else {
          f32x4 row_lse[J], row_dloss[J];
          bool near = false;
#pragma unroll
          for (int j = 0; j < J; j++) {
            row_lse[j] = *(const f32x4 *)(p.taken.lse + s0 + j * 16);
            row_dloss[j] = *(const f32x4 *)(p.taken.dloss + s0 + j * 16) * scale;
            const uint4 aim = *(const uint4 *)(p.taken.target + s0 + j * 16);
            near = near || aim.x - first < OI * 16 || aim.y - first < OI * 16 || aim.z - first < OI * 16 || aim.w - first < OI * 16;
          }
#pragma unroll
          for (int i = 0; i < OI; i++)
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                sum[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sum[i][j][e] - row_lse[j][e], kLog2E, own_bias[i])) * row_dloss[j][e];
          if (__ballot(near))
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t aim = p.taken.target[s0 + j * 16 + e] - first - l % 16;
#pragma unroll
                for (int i = 0; i < OI; i++) sum[i][j][e] -= aim == (uint32_t)(i * 16) ? row_dloss[j][e] : 0.f;
              }
          if (p.sums)
#pragma unroll
            for (int i = 0; i < OI; i++)
#pragma unroll
              for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) total[i] += sum[i][j][e];
        }
        // (rounded: the matrix cores take both operands in one type)
        Fragment<T> d[OI];
#pragma unroll
        for (int i = 0; i < OI; i++) {
          Floats<8> f;
#pragma unroll
          for (int e = 0; e < 8; e++) f.v[e] = sum[i][e / 4][e % 4];
          d[i].v = rounded<T>(f);
        }
#pragma unroll
        for (int c = 0; c < 2 * KS; c++) {
          const Fragment<T> f = N::across(across, r0, c);
#pragma unroll
          for (int i = 0; i < OI; i++) out[i][c] = multiply<T>(f, d[i], out[i][c]);
        }
      }
    }
  }

  if constexpr (MODE == Narrow::kForward) {
#pragma unroll
    for (int i = 0; i < OI; i++) {
      Tail t = join_lanes(join_lanes(Tail{most[i], total[i]}, 16), 32);
      const uint32_t r = first + i * 16 + l;
      if (l < 16 && r < owned) p.parts[(uint64_t)range * p.rows + r] = make_float2(t.most, t.sum);
    }
    // The logits of the rows' targets, once more: the products of the rows with the 16 items that they aim at, by the same instructions in the same
    // order, so that they are the logits above to the bit; what a row has of its own lies on the diagonal.  (Picked out in the loop they would
    // cost two instructions a logit where there are few items.)
    if (range == p.ranges - 1) // which has the fewest tiles
#pragma unroll
      for (int i = 0; i < OI; i++) {
        const uint32_t r = first + i * 16 + l % 16, item = r < owned ? p.taken.target[r] : kNoItem;
        f32x4 sum = {};
#pragma unroll
        for (int kk = 0; kk < KS; kk++) {
          const uint32_t c = (kk * 4 + l / 16) * 8;
          Fragment<T> f;
          f.v = (T)0;
          if (item != kNoItem && c < p.width) f.v = *(const typename Fragment<T>::type *)(p.weight + (int64_t)item * p.weight_stride + c * 2);
          sum = multiply<T>(f, mine[i][kk], sum);
        }
        const float own = l % 4 == 0 ? sum[0] : l % 4 == 1 ? sum[1] : l % 4 == 2 ? sum[2] : sum[3];
        if (l % 16 / 4 == l / 16 && item != kNoItem) p.taken.hits[r] = __builtin_fmaf(own, kLog2E, p.taken.bias[item]);
      }
  } else {
    const float back = p.partial ? 1.f : p.taken.scale[1];
    const uint32_t columns = (p.width + 3) / 4 * 4;
#pragma unroll
    for (int i = 0; i < OI; i++) {
      const uint32_t r = first + i * 16 + l % 16;
      if constexpr (WEIGHT) {
        if (p.sums) {
          float s = total[i];
          s += __shfl_xor(s, 16);
          s += __shfl_xor(s, 32);
          if (l < 16 && r < owned) p.sums[(uint64_t)range * p.items + r] = s;
        }
      }
      if (r >= owned) continue;
      T *to = p.partial ? nullptr : row_of<T>(p.result, r);
      float *part = p.partial + ((uint64_t)range * (WEIGHT ? p.items : p.rows) + r) * columns;
#pragma unroll
      for (int c = 0; c < 2 * KS; c++) {
        const uint32_t at = c * 16 + l / 16 * 4;
        if (at >= p.width) continue;
        if (p.partial) *(f32x4 *)(part + at) = out[i][c];
        else if (to) write4<T>(to, at, p.width, out[i][c] * back);
      }
    }
  }
}

template <typename T, Narrow MODE> void launch_narrow(ItemsNarrow &p, hipStream_t s) {
  const size_t owned = MODE == Narrow::kDweight ? p.items : p.rows;
  const auto launch = [&](auto kernel, int rows) {
    p.owners = div_up(owned, rows);
    hipLaunchKernelGGL(kernel, dim3(p.owners * p.ranges), dim3(256), 0, s, p);
  };
  if (p.width <= 32) launch(items_narrow<T, 1, MODE>, kOwned<1, MODE> * 64);
  else if (p.width <= 64) launch(items_narrow<T, 2, MODE>, kOwned<2, MODE> * 64);
  else launch(items_narrow<T, 4, MODE>, kOwned<4, MODE> * 64);
  HCTR_HIP(hipGetLastError());
}
template <typename T> void launch_narrow_forward(ItemsNarrow &p, hipStream_t s) { launch_narrow<T, Narrow::kForward>(p, s); }
template <typename T> void launch_narrow_dx(ItemsNarrow &p, hipStream_t s) { launch_narrow<T, Narrow::kDx>(p, s); }
template <typename T> void launch_narrow_dweight(ItemsNarrow &p, hipStream_t s) { launch_narrow<T, Narrow::kDweight>(p, s); }

} // namespace hctr
