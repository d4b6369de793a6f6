// Sums of exponentials that can be joined, and the size of a gradient: what the kernels of items_kernels.h and items.hip share.
#pragma once
#include "common.h"

namespace hctr {

constexpr float kLog2E = 1.4426950408889634f, kInfinity = __builtin_inff();

// exp(v - most), where most is -infinity only if every v is
__device__ __forceinline__ float exp_less(float v, float most) { return __builtin_amdgcn_exp2f((v - most) * kLog2E); }

// The largest of some values and the sum of their exponentials less it: joined, and over the lanes `mask` apart.  Nothing but values of
// -infinity: a sum of 0.
struct Tail {
  float most, sum;
};
__device__ __forceinline__ Tail join(Tail a, Tail b) {
  const float most = a.most > b.most || a.most != a.most ? a.most : b.most;
  const float sa = a.most == -kInfinity ? 0.f : a.sum * exp_less(a.most, most), sb = b.most == -kInfinity ? 0.f : b.sum * exp_less(b.most, most);
  return {most, sa + sb};
}
__device__ __forceinline__ Tail join_lanes(Tail t, int mask) { return join(t, Tail{__shfl_xor(t.most, mask), __shfl_xor(t.sum, mask)}); }

// |v| as an integer that orders as it does, 0 if it is not finite
__device__ __forceinline__ uint32_t size_bits(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}
} // namespace hctr
