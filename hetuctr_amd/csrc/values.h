// Rows of float, bfloat16 or half values as the dense operators read and write them: a few columns at a time, in 32 bits.
#pragma once
#include <type_traits>

#include "common.h"

namespace hctr {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Columns a lane moves at a time: 16 bytes of the type that is normalised or dropped.  Always a multiple of four, the columns
// that one draw of the generator serves.
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

template <typename T, int V> struct Packed {
  typedef T type __attribute__((ext_vector_type(V)));                       // in registers
  typedef T memory __attribute__((ext_vector_type(V), aligned(sizeof(T)))); // at any address a T can have
};
template <int V> struct Floats {
  float v[V];
};

// How a kernel reads and writes rows of `width` columns, V at a time.
enum class Rows {
  kEven,   // short (their bytes can be counted in 32 bits), the width a multiple of V: past the caches, nothing reads them again
  kRagged, // short, at least V columns: rows share cache lines with their neighbours, which the caches put together
  kTiny,   // the same, any width
  kLong,   // any length and width
};

// where column c lies; a load or store adds 32 bits to a row's address by itself
template <Rows R, typename T> __device__ __forceinline__ T *at_column(T *row, uint32_t c) {
  if constexpr (R == Rows::kLong) return row + c;
  else return (T *)((char *)row + c * (uint32_t)sizeof(T));
}

// Columns c .. c + V - 1 as they lie in memory, those behind the row's end as zeros, in two steps, so that more can be loaded before
// what is loaded has to be there.  A row may start at any multiple of its element's size (gfx950 moves up to 16 bytes from
// any address in one instruction), and nothing outside it is read: the vector that would end behind a row of V columns or
// more is the row's last V columns (load_raw), moved down by as many as it would end behind (settled; the same number for
// every row, so the branches are scalar ones).  Rows of 37 floats, a gradient of 2^27 values: 732 us with the move in the
// branch of the load, where it waits for each load by itself, 348 in two steps.
// ONCE: nothing reads them again soon.  KEPT: behind the end of a vector that was moved lie other columns of the row, not zeros.
template <int V, Rows R, bool ONCE = R == Rows::kEven, typename T>
__device__ __forceinline__ typename Packed<T, V>::type load_raw(const T *row, uint32_t c, uint32_t width) {
  typename Packed<T, V>::type x = (T)0;
  const auto load = [&](uint32_t from) {
    const auto p = (const typename Packed<T, V>::memory *)at_column<R>(const_cast<T *>(row), from);
    x = ONCE ? __builtin_nontemporal_load(p) : *p;
  };
  if constexpr (R == Rows::kEven) {
    if (c < width) load(c);
  } else if (c < width) {
    if (R == Rows::kRagged || width >= V) load(min(c, width - V));
    else
#pragma unroll
      for (int j = 0; j + 1 < V; j++)
        if (j < width) x[j] = row[j];
  }
  return x;
}
template <int V, Rows R, bool KEPT = false, typename X> __device__ __forceinline__ X settled(X x, uint32_t c, uint32_t width) {
  if constexpr (R != Rows::kEven)
    if (c < width && c + V > width && (R == Rows::kRagged || width >= V)) {
      const uint32_t by = V - width % V;
#pragma unroll
      for (int k = 1; k < V; k *= 2)
        if (by & k) {
#pragma unroll
          for (int j = 0; j < V; j++) x[j] = j + k < V ? x[(j + k) % V] : KEPT ? x[j] : 0;
        }
    }
  return x;
}
template <int V, typename X> __device__ __forceinline__ Floats<V> floats(const X &x) {
  Floats<V> f;
#pragma unroll
  for (int j = 0; j < V; j++) f.v[j] = (float)x[j];
  return f;
}
template <int V, Rows R, bool ONCE = R == Rows::kEven, typename T>
__device__ __forceinline__ Floats<V> load_columns(const T *row, uint32_t c, uint32_t width) {
  return floats<V>(settled<V, R>(load_raw<V, R, ONCE>(row, c, width), c, width));
}

// Values rounded to T, to nearest, ties to even.  The compiler may put the product or sum that made a value and its rounding to half
// into one instruction, which does not round to 32 bits in between, in one kernel and not in another: it is kept from that,
// so that a value does not depend on where its row lies.
template <typename T, int V> __device__ __forceinline__ typename Packed<T, V>::type rounded(const Floats<V> &f) {
  typename Packed<T, V>::type x;
#pragma unroll
  for (int j = 0; j < V; j++) {
    float v = f.v[j];
    if constexpr (std::is_same_v<T, f16_t>) asm("" : "+v"(v));
    x[j] = (T)v;
  }
  return x;
}

// Columns c .. c + V - 1 written, rounded to the nearest value of T.  The last columns of a
// ragged row go out in pieces of a power of two.
template <int V, Rows R, typename T>
__device__ __forceinline__ void store_columns(T *row, uint32_t c, uint32_t width, const Floats<V> &f) {
  typename Packed<T, V>::type x = rounded<T>(f);
  T *p = at_column<R>(row, c);
  if constexpr (R == Rows::kEven) {
    if (c < width) __builtin_nontemporal_store(x, (typename Packed<T, V>::memory *)p);
  } else if (c + V <= width) {
    *(typename Packed<T, V>::memory *)p = x;
  } else if (c < width) {
    const uint32_t left = width % V;
    if (V > 4 && left & 4) {
      *(typename Packed<T, 4>::memory *)p = __builtin_shufflevector(x, x, 0, 1, 2, 3);
#pragma unroll
      for (int j = 0; j < 3; j++) x[j] = x[(j + 4) % V];
      p += 4;
    }
    if (left & 2) {
      *(typename Packed<T, 2>::memory *)p = __builtin_shufflevector(x, x, 0, 1);
      x[0] = x[2];
      p += 2;
    }
    if (left & 1) *p = x[0];
  }
}

} // namespace hctr
