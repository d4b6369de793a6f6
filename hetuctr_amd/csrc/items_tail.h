// Sums of exponentials that can be joined, and the size of a gradient: what the kernels of items_kernels.h and items.hip share.
//
// Logits are held in units of log 2: one product-and-sum makes one of them from the sum over k and the bias, which is multiplied beforehand,
// and an exponential is the machine's own, of two.
#pragma once
#include "common.h"

namespace hctr {

constexpr float kLog2E = 1.4426950408889634f, kLog2 = 0.69314718055994531f, kInfinity = __builtin_inff();
constexpr float kLowest = -3e38f; // stands for the largest of no values, so that differences from it are never those of infinities

// The largest of some values, in units of log 2, and the sum of their exponentials less it.
struct Tail {
  float most, sum;
};
__device__ __forceinline__ Tail join(Tail a, Tail b) {
  const float most = fmaxf(a.most, b.most);
  return {most, a.sum * __builtin_amdgcn_exp2f(a.most - most) + b.sum * __builtin_amdgcn_exp2f(b.most - most)};
}
__device__ __forceinline__ Tail join_lanes(Tail t, int mask) { return join(t, Tail{__shfl_xor(t.most, mask), __shfl_xor(t.sum, mask)}); }

// |v| as an integer that orders as it does, 0 if it is not finite
__device__ __forceinline__ uint32_t size_bits(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}

} // namespace hctr
