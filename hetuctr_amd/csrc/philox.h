// The random numbers of dropout: Philox4x32 with 7 rounds, a counter-based generator (Salmon, Moraes, Dror, Shaw: "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011).  Four 32-bit words are a function of a 128-bit counter and a 64-bit key, so
// the gradient's pass draws the forward pass's numbers again and no mask is ever stored.
//
// 7 rounds are the fewest with which the paper's authors found the generator to pass every test of BigCrush; with the 10 that
// they take for a margin the draws alone run at 0.58 T quads per second on an MI355X instead of 0.79, and dropping out 218 M
// bfloat16 values (436 MB in, 436 MB out) takes 146 us instead of 139 (a plain copy: 135).
#pragma once
#include <cstdint>

namespace hctr {

constexpr uint64_t kPhiloxMul0 = 0xD2511F53u, kPhiloxMul1 = 0xCD9E8D57u;
constexpr uint32_t kPhiloxKey0 = 0x9E3779B9u, kPhiloxKey1 = 0xBB67AE85u;
constexpr int kPhiloxRounds = 7;

struct Quad {
  uint32_t w[4];
};

// a ^ b ^ c (one instruction, where the compiler makes two)
__host__ __device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
#else
  return a ^ b ^ c;
#endif
}

// the words of counter (quad, step), low words first, under `key`
__host__ __device__ __forceinline__ Quad philox(uint64_t quad, uint64_t step, uint64_t key) {
  uint32_t c0 = (uint32_t)quad, c1 = (uint32_t)(quad >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < kPhiloxRounds; r++) {
    const uint64_t a = kPhiloxMul0 * c0, b = kPhiloxMul1 * c2;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += kPhiloxKey0;
    k1 += kPhiloxKey1;
  }
  return {{c0, c1, c2, c3}};
}

} // namespace hctr
