// Products of matrices on the matrix cores, as the kernels of gated_kernels.h, items_kernels.h and products_kernels.h build them: tiles that go from memory to LDS past the
// registers, fragments from there, sums in 32 bits, and an epilogue that takes them.
#pragma once
#include <type_traits>

#include "common.h"
#include "values.h"

namespace hctr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// How an operand of a product lies in memory, seen as rows x k, where k is what is summed over: kAlong: neighbours lie along k;
// kAcross: neighbours lie along the rows.
enum class Lies { kAlong, kAcross };

// An operand: element (row, k) of kAlong lies at base + row * stride + k * size, of kAcross at base + k * stride + row * size; bytes.
// Every line of kLineBytes or more begins at a multiple of 16 bytes and its length is one too (what lies behind a shorter matrix
// there is zeros along k, anything across it).
struct Operand {
  const char *base[2]; // the second one: what Second says
  int64_t stride;
  uint32_t rows;
  uint32_t behind_from, behind_k; // kBehind: where along k the second matrix begins, a multiple of kStep; the k that each one has
};

// What the second base of an operand is: nothing, another matrix whose rows alternate with those of the first in groups of
// kPairRows, or one that follows the first along k.
enum class Second { kNone, kPaired, kBehind };
constexpr int kPairRows = 32;

constexpr int kStepBytes = 128;  // of k that a row of a tile of kAlong holds
constexpr uint32_t kNowhere = 0x80000000u; // an offset behind every buffer: the load writes zeros

template <typename T> constexpr int kStep = kStepBytes / (int)sizeof(T); // of k that a tile holds

// 16 bytes per lane from base + offset to LDS, where a wave's lanes lie one behind the other from `lds`, the same address in all
// lanes.  Not the builtin: the compiler would wait for every such load before any read of LDS.  The list of what is overwritten cannot name m0, which
// is not a register that the compiler gives to values (it warns, and builds the same code): nothing of it may be kept there across this, which
// tests/test_kernel_m0.py reads from the built library.
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "memory");
}
__device__ __forceinline__ i32x4 buffer_at(const char *base) {
  const uint64_t b = (uint64_t)base;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((int)b), (int)(__builtin_amdgcn_readfirstlane((int)(b >> 32)) & 0xffff), (int)kNowhere, 0x20000};
}
// All but the last LEFT loads that this wave has under way are there, and so are those of the block's other waves
template <int LEFT> __device__ __forceinline__ void tiles_ready() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory"); }

// Where 16-byte piece `piece` of line `line` of a tile lies among the line's pieces.  A fragment takes one piece of each of 16 rows
// (kAlong), or pieces of 16 rows from eight or four lines (kAcross): the order makes them lie in different banks.
template <typename T, Lies L, int ROWS> __device__ __forceinline__ uint32_t placed(uint32_t line, uint32_t piece) {
  if constexpr (L == Lies::kAlong) return piece ^ (line >> 1 & 7);
  else if constexpr (sizeof(T) == 4) return piece ^ ((line >> 2 & 3) << 2);
  else if constexpr (ROWS == 64) return piece ^ ((line >> 1 & 1) << 1 | (line >> 3 & 1) << 2); // lines of eight pieces
  else return piece ^ ((line & 3) << 1 | (line >> 3 & 1) << 3);
}

// One operand's tiles of ROWS rows, loaded by THREADS threads.
template <typename T, Lies L, Second S, int ROWS, int THREADS> struct Tiles {
  static constexpr int kPasses = ROWS * kStepBytes / (THREADS * 16);
  static constexpr int kPieces = L == Lies::kAlong ? 8 : ROWS * (int)sizeof(T) / 16; // of a line
  const char *base, *base2;
  int64_t stride;
  uint32_t offset[kPasses];
  uint32_t k_of[L == Lies::kAlong ? 1 : kPasses]; // kAlong: of the thread's piece, in bytes; kAcross: the line
  uint32_t behind_from, behind_k;

  __device__ __forceinline__ void init(const Operand &o, uint32_t row0) {
    stride = o.stride;
    behind_from = o.behind_from, behind_k = o.behind_k;
    const uint32_t t = threadIdx.x;
    if constexpr (L == Lies::kAlong) {
      const uint32_t slot = t % 8, line = t / 8;
      const uint32_t piece = placed<T, L, ROWS>(line, slot);
      k_of[0] = piece * 16;
      const uint32_t first = S == Second::kPaired ? row0 / 2 : row0;
      base = o.base[0] + (int64_t)first * stride;
      base2 = S == Second::kPaired ? o.base[1] + (int64_t)first * stride : nullptr;
#pragma unroll
      for (int i = 0; i < kPasses; i++) {
        uint32_t r = i * (THREADS / 8) + line;
        if constexpr (S == Second::kPaired) r = r / (2 * kPairRows) * kPairRows + r % kPairRows;
        offset[i] = first + r < o.rows ? r * (uint32_t)stride + piece * 16 : kNowhere;
      }
    } else {
      base = o.base[0] + (int64_t)row0 * sizeof(T);
      base2 = S == Second::kBehind ? o.base[1] + (int64_t)row0 * sizeof(T) : nullptr;
#pragma unroll
      for (int i = 0; i < kPasses; i++) {
        const uint32_t s = i * THREADS + t, line = s / kPieces, piece = placed<T, L, ROWS>(line, s % kPieces);
        k_of[i] = line;
        offset[i] = row0 + piece * (16 / sizeof(T)) < o.rows ? line * (uint32_t)stride + piece * 16 : kNowhere;
      }
    }
  }
  // the tile of k, k + 1, .. to LDS; `left`: of k before it ends
  __device__ __forceinline__ void load(uint32_t k, uint32_t left, uint32_t lds) const {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const char *from;
    if constexpr (L == Lies::kAlong) {
      from = base + (int64_t)k * sizeof(T);
    } else if constexpr (S == Second::kBehind) {
      const bool behind = k >= behind_from;
      k -= behind ? behind_from : 0;
      left = k < behind_k ? behind_k - k : 0;
      from = (behind ? base2 : base) + (int64_t)k * stride;
    } else {
      from = base + (int64_t)k * stride;
    }
    const i32x4 rsrc = buffer_at(from);
    i32x4 rsrc2;
    if constexpr (S == Second::kPaired) rsrc2 = buffer_at(base2 + (int64_t)k * sizeof(T));
    const uint32_t to = lds + wave * (kWave * 16);
    const bool whole = left >= (uint32_t)kStep<T>;
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
      uint32_t o = offset[i];
      if (!whole) {
        if constexpr (L == Lies::kAlong) o = k_of[0] < left * sizeof(T) ? o : kNowhere;
        else o = k_of[i] < left ? o : kNowhere;
      }
      if constexpr (S == Second::kPaired) {
        const bool second = (i * (THREADS / 8) + wave * 8) & kPairRows;
        load_to_lds(second ? rsrc2 : rsrc, o, to + i * (THREADS * 16));
      } else {
        load_to_lds(rsrc, o, to + i * (THREADS * 16));
      }
    }
  }
};

// A fragment: 16 rows of an operand, 64 bytes of k: what four lanes of 16 bytes hold.  (Of 32 rows and 32 bytes, for the matrix cores' other
// shape: with operands of zeros 8192^3 takes 689 to 755 us in the three layouts instead of 733 to 746, with random ones, for which
// the clock falls to 1.8 GHz, 917 to 1045 instead of 886 to 993.)
template <typename T> struct Fragment {
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
  type v;
};
typedef __attribute__((address_space(3))) char lds_char;

// rows r0 .. r0 + 15 of a tile, part kk (0 or 1) of its k.  Lane l holds row l % 16, and of k the 16 bytes l / 16.
template <typename T, Lies L, int ROWS> __device__ __forceinline__ Fragment<T> fragment(uint32_t lds, uint32_t r0, uint32_t kk) {
  const uint32_t l = threadIdx.x % kWave;
  Fragment<T> f;
  if constexpr (L == Lies::kAlong) {
    const uint32_t r = r0 + l % 16;
    f.v = *(const __attribute__((address_space(3))) typename Fragment<T>::type *)(uintptr_t)(lds + r * kStepBytes + placed<T, L, ROWS>(r, kk * 4 + l / 16) * 16);
  } else if constexpr (sizeof(T) == 2) {
    // Lanes 4 i .. 4 i + 3 of each 16 point at the 16 rows of line i, and get four lines of one row each.
    typedef short s4 __attribute__((ext_vector_type(4)));
    s4 h[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint32_t line = kk * 32 + l / 16 * 8 + j * 4 + l % 16 / 4;
      const uint32_t row = r0 + l % 4 * 4;
      const uint32_t at = lds + line * (ROWS * 2) + placed<T, L, ROWS>(line, row / 8) * 16 + row % 8 * 2;
      h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(uintptr_t)at);
    }
    f.v = __builtin_bit_cast(typename Fragment<T>::type, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t line = kk * 16 + l / 16 * 4 + j, row = r0 + l % 16;
      f.v[j] = *(const __attribute__((address_space(3))) float *)(uintptr_t)(lds + line * (ROWS * 4) + placed<T, L, ROWS>(line, row / 4) * 16 + row % 4 * 4);
    }
  }
  return f;
}

// c[i] += sum over k of a's row (4 * (lane / 16) + i) times b's row (lane % 16)
template <typename T> __device__ __forceinline__ f32x4 multiply(const Fragment<T> &a, const Fragment<T> &b, f32x4 c) {
  if constexpr (std::is_same_v<T, bf16_t>) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
  else if constexpr (std::is_same_v<T, f16_t>) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
  else
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// A float is the sum of three bfloat16: the one nearest to it, the one nearest to what is left, and what is then left, which has eight bits at
// most.  Of the nine products of two such sums the six largest are made; the others are below 2^-24 of the floats' product together (at most 0.9932 of that, over all of them).
// They take six times a sixteenth of the matrix cores' time for floats, and five or six instructions for each float.  us, 8192 x 8192 x 2048 in
// the three layouts: 2095, 2043 and 2098 with products of floats (131 to 135 TFLOP/s, of the 157 that the cores could do at most), 1573,
// 1466 and 1476 so.  An infinity becomes a NaN on the way, a float below 2^-110 loses some of its bits, one beyond 2^128 - 2^119 is as
// good as infinite.
struct Split {
  Fragment<bf16_t> part[3];
};
__device__ __forceinline__ Split split(const Fragment<float> &a, const Fragment<float> &b) {
  Split s;
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = a.v[e], v[e + 4] = b.v[e];
#pragma unroll
  for (int p = 0; p < 3; p++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const bf16_t x = (bf16_t)v[e];
      s.part[p].v[e] = x;
      v[e] -= (float)x;
    }
  return s;
}

// The product of tiles: BM rows of a times BN rows of b, by waves of WM x WN each.  sum[i][j][e]: row i * 16 + lane % 16 of the wave's WM of a,
// row j * 16 + lane / 16 * 4 + e of its WN of b: four neighbouring columns of the result in a lane.
template <typename T, Lies LA, Lies LB, Second SB, int BM, int BN> struct Product {
  static constexpr int WM = BM / 2, WN = 64, kWaves = 2 * (BN / WN), kThreads = kWaves * kWave;
  static constexpr int kRowTiles = WM / 16, kColumnTiles = WN / 16;
  // Tiles that LDS holds: the one that is read, and those under way.  Small ones, which are for products that leave a CU little else to do, have
  // to wait out the memory by themselves (us, loss of 35 rows of 8086 columns and 712 items in bfloat16: 83 with two, 67 with four; its
  // gradient for 259, 1149 and 3286 in float 177, 126).
  static constexpr uint32_t kStages = BM == 64 ? 4 : 2;
  static constexpr int kWavesEach = BM == 64 ? 1 : 2; // of a SIMD, at least
  static constexpr uint32_t kStageBytes = (BM + BN) * kStepBytes, kLdsBytes = kStages * kStageBytes;
  typedef f32x4 Sums[kRowTiles][kColumnTiles];

  static __device__ __forceinline__ uint32_t wave_row() { return threadIdx.x / kWave / (BN / WN) * WM; }
  static __device__ __forceinline__ uint32_t wave_column() { return threadIdx.x / kWave % (BN / WN) * WN; }

  // The same for floats, in parts: a step's fragments of b are split, then those of a, 16 rows at a time, while the ones before are multiplied.
  template <typename TA, typename TB>
  static __device__ __forceinline__ void run_floats(const TA &ta, const TB &tb, uint32_t k0, uint32_t k1, uint32_t lds, Sums &sum) {
    constexpr uint32_t step = kStep<T>;
    constexpr int kLoads = TA::kPasses + TB::kPasses;
    const auto load = [&](uint32_t k, uint32_t stage) {
      ta.load(k, k1 - k, lds + stage * kStageBytes);
      tb.load(k, k1 - k, lds + stage * kStageBytes + BM * kStepBytes);
    };
#pragma unroll
    for (uint32_t i = 0; i + 1 < kStages; i++)
      if (k0 + i * step < k1) load(k0 + i * step, i);
    uint32_t stage = 0;
    for (uint32_t k = k0; k < k1; k += step) {
      if (kStages > 2 && k + (kStages - 2) * step < k1) tiles_ready<(int)(kStages - 2) * kLoads>();
      else tiles_ready<0>();
      // (everyone has read the tile before this one)
      if (k + (kStages - 1) * step < k1) load(k + (kStages - 1) * step, stage ? stage - 1 : kStages - 1);
      const uint32_t here = lds + stage * kStageBytes;
      Split b[kColumnTiles];
#pragma unroll
      for (int j = 0; j < kColumnTiles; j++)
        b[j] = split(fragment<T, LB, BN>(here + BM * kStepBytes, wave_column() + j * 16, 0), fragment<T, LB, BN>(here + BM * kStepBytes, wave_column() + j * 16, 1));
#pragma unroll
      for (int i = 0; i < kRowTiles; i++) {
        const Split a = split(fragment<T, LA, BM>(here, wave_row() + i * 16, 0), fragment<T, LA, BM>(here, wave_row() + i * 16, 1));
        // the smallest first
#pragma unroll
        for (int both = 2; both >= 0; both--)
#pragma unroll
          for (int p = 0; p <= both; p++)
#pragma unroll
            for (int j = 0; j < kColumnTiles; j++) sum[i][j] = multiply<bf16_t>(b[j].part[both - p], a.part[p], sum[i][j]);
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }

  // k from k0 (a multiple of kStep) to k1
  static __device__ __forceinline__ void run(const Operand &a, const Operand &b, uint32_t row0, uint32_t column0, uint32_t k0, uint32_t k1,
                                             uint32_t lds, Sums &sum) {
    constexpr uint32_t step = kStep<T>;
    Tiles<T, LA, Second::kNone, BM, kThreads> ta;
    Tiles<T, LB, SB, BN, kThreads> tb;
    ta.init(a, row0);
    tb.init(b, column0);
#pragma unroll
    for (int i = 0; i < kRowTiles; i++)
#pragma unroll
      for (int j = 0; j < kColumnTiles; j++) sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k0 >= k1) return;
    // (a small tile would split each value too often: 8192 x 8192 x 2048 in 2774 us instead of 2315)
    if constexpr (sizeof(T) == 4 && BM > 64) return run_floats(ta, tb, k0, k1, lds, sum);
    const auto load = [&](uint32_t k, uint32_t stage) {
      ta.load(k, k1 - k, lds + stage * kStageBytes);
      tb.load(k, k1 - k, lds + stage * kStageBytes + BM * kStepBytes);
    };
    // Half a step's fragments are read from LDS while the other half's are multiplied, a few instructions between each of them.  The barrier
    // stands in the middle: there the second half of this step is in registers, and nobody needs its tiles any more; the next step's
    // tiles are there, which have been under way for a whole step; and there is work at hand for both sides of it.  (8192 x 8192 x 8192 in
    // bfloat16, operands of zeros, which the clock does not suffer from: 852 us with a step's reads in front of its products, 741 so; random ones
    // 1083 and 988.)
    Fragment<T> fa[2][kRowTiles], fb[2][kColumnTiles];
    const auto read = [&](uint32_t from, auto half) {
      constexpr uint32_t H = decltype(half)::value;
#pragma unroll
      for (int j = 0; j < kColumnTiles; j++) fb[H][j] = fragment<T, LB, BN>(from + BM * kStepBytes, wave_column() + j * 16, H);
#pragma unroll
      for (int i = 0; i < kRowTiles; i++) fa[H][i] = fragment<T, LA, BM>(from, wave_row() + i * 16, H);
    };
    const auto products = [&](auto half) {
      constexpr uint32_t H = decltype(half)::value;
#pragma unroll
      for (int i = 0; i < kRowTiles; i++)
#pragma unroll
        for (int j = 0; j < kColumnTiles; j++) sum[i][j] = multiply<T>(fb[H][j], fa[H][i], sum[i][j]);
    };
    constexpr std::integral_constant<uint32_t, 0> first;
    constexpr std::integral_constant<uint32_t, 1> second;
    // reads and products of one region, in turn
    constexpr int kPerFragment = sizeof(T) == 2 ? 2 : 4, kMultiplies = kRowTiles * kColumnTiles * (sizeof(T) == 2 ? 1 : 4);
    constexpr int kReads = kRowTiles * (LA == Lies::kAlong ? 1 : kPerFragment) + kColumnTiles * (LB == Lies::kAlong ? 1 : kPerFragment);
    const auto in_turn = [&] {
#pragma unroll
      for (int i = 0; i < kReads; i++) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, kMultiplies / kReads, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, kMultiplies - kReads * (kMultiplies / kReads), 0);
      __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int kLoads = Tiles<T, LA, Second::kNone, BM, kThreads>::kPasses + Tiles<T, LB, SB, BN, kThreads>::kPasses;
#pragma unroll
    for (uint32_t i = 0; i + 1 < kStages; i++)
      if (k0 + i * step < k1) load(k0 + i * step, i);
    if (k0 + (kStages - 2) * step < k1) tiles_ready<(int)(kStages - 2) * kLoads>();
    else tiles_ready<0>();
    if (k0 + (kStages - 1) * step < k1) load(k0 + (kStages - 1) * step, kStages - 1);
    read(lds, first);
    uint32_t stage = 0, k = k0;
    for (; k + step < k1; k += step) {
      __builtin_amdgcn_sched_barrier(0);
      read(lds + stage * kStageBytes, second);
      products(first);
      in_turn();
      // (at the end there are fewer tiles under way)
      if (kStages > 2 && k + (kStages - 1) * step < k1) tiles_ready<(int)(kStages - 2) * kLoads>();
      else tiles_ready<0>();
      if (k + kStages * step < k1) load(k + kStages * step, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      __builtin_amdgcn_sched_barrier(0);
      read(lds + stage * kStageBytes, first);
      products(second);
      in_turn();
    }
    read(lds + stage * kStageBytes, second);
    products(first);
    products(second);
  }
};

// A tile of results of 16 bits on its way out: the waves put four columns at a time into LDS, where they take 32 bytes of 16 rows each, in
// different banks, and the block writes whole rows of it.  Straight from the registers a store is 16 pieces of 32 bytes, one a row, which
// all go to one memory channel where rows lie a power of two apart (8192 x 32768 x 4096 in bfloat16: 2276 us, rows 128 bytes
// further apart 1898).
template <typename T, int ROWS, int COLUMNS> struct Staged {
  static_assert(sizeof(T) == 2, "pieces of eight columns");
  static constexpr uint32_t kBytes = ROWS * COLUMNS * 2, kPieces = COLUMNS / 8, kMask = COLUMNS / 16 < 16 ? COLUMNS / 16 - 1 : 15;
  static __device__ __forceinline__ void put(uint32_t lds, uint32_t row, uint32_t column, f32x4 v) {
    const Floats<4> f = {{v[0], v[1], v[2], v[3]}};
    const uint32_t at = lds + row * (COLUMNS * 2) + ((column / 16 ^ (row & kMask)) * 32 | column % 16 * 2);
    *(__attribute__((address_space(3))) typename Packed<T, 4>::type *)(uintptr_t)at = rounded<T>(f);
  }
  // f(row, column, its eight values) for every piece, by all threads of the block
  template <int THREADS, typename F> static __device__ __forceinline__ void each(uint32_t lds, F &&f) {
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < ROWS * kPieces; i += THREADS) {
      const uint32_t row = i / kPieces, piece = i % kPieces;
      const uint32_t at = lds + row * (COLUMNS * 2) + ((piece / 2 ^ (row & kMask)) * 32 | piece % 2 * 16);
      f(row, piece * 8, *(const __attribute__((address_space(3))) typename Packed<T, 8>::type *)(uintptr_t)at);
    }
  }
};

// The tile that a block works on.  Neighbouring blocks go to different XCDs: each XCD gets a stretch of neighbouring tiles, and takes them
// in bands of `band` tiles of rows, so that those at work share lines in its L2.
__device__ __forceinline__ void tile_of(uint32_t block, uint32_t blocks, uint32_t row_tiles, uint32_t column_tiles, uint32_t band, uint32_t &row, uint32_t &column) {
  constexpr uint32_t kXcds = 8;
  const uint32_t xcd = block % kXcds, each = blocks / kXcds, more = blocks % kXcds;
  const uint32_t t = block / kXcds + xcd * each + min(xcd, more);
  const uint32_t per_band = band * column_tiles, b = t / per_band, in = t % per_band;
  const uint32_t height = min(band, row_tiles - b * band);
  row = b * band + in % height;
  column = in / height;
}

} // namespace hctr
