// Rows of float, bfloat16 or half values as the dense operators read and write them: a few columns at a time, in 32 bits.
#pragma once
#include "common.h"

namespace hctr {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Columns a lane moves at a time: 16 bytes of the type that is normalised or dropped.  Always a multiple of four, the columns
// that one draw of the generator serves.
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

template <typename T, int V> struct Packed {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); // any address a T can have
};
template <int V> struct Floats {
  float v[V];
};

// Columns c .. c + V - 1 of a row of `width` columns, those behind its end as zeros.  A row may start at any multiple of its
// element's size (gfx950 moves up to 16 bytes from any address in one instruction), and nothing outside it is read.
// ONCE: nothing reads them again soon.
template <int V, bool ONCE = true, typename T>
__device__ __forceinline__ Floats<V> load_columns(const T *row, uint32_t c, uint32_t width) {
  Floats<V> f;
  if (c + V <= width) {
    typedef const typename Packed<T, V>::type *Vector;
    const auto x = ONCE ? __builtin_nontemporal_load((Vector)(row + c)) : *(Vector)(row + c);
#pragma unroll
    for (int j = 0; j < V; j++) f.v[j] = (float)x[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) f.v[j] = 0.f;
    if (c < width) {
#pragma unroll
      for (int j = 0; j + 1 < V; j++)
        if (c + j < width) f.v[j] = (float)row[c + j];
    }
  }
  return f;
}

// the same columns written, rounded to the nearest value of T (ties to even) if that is narrower
template <int V, typename T> __device__ __forceinline__ void store_columns(T *row, uint32_t c, uint32_t width, const Floats<V> &f) {
  if (c + V <= width) {
    typename Packed<T, V>::type x;
#pragma unroll
    for (int j = 0; j < V; j++) x[j] = (T)f.v[j];
    __builtin_nontemporal_store(x, (typename Packed<T, V>::type *)(row + c));
  } else if (c < width) {
#pragma unroll
    for (int j = 0; j + 1 < V; j++)
      if (c + j < width) row[c + j] = (T)f.v[j];
  }
}

} // namespace hctr
