// Dropout whose mask is a function of position, seed and step (philox.h), and the argument checks of the dense operators.
#include <algorithm>
#include <cmath>

#include "dense.h"

namespace hctr {
namespace {

constexpr int kBlock = 256;

// Pieces of kVec<T> values that a thread has under way at a time.  16-bit values are bound by the draws as much as by the memory, and
// more pieces let the two overlap: us on an MI355X with 1, 2, 3, 4 pieces, 2.2e8 bfloat16 values 139.7, 139.4, 138.6, 137.9 (6.3
// TB/s, a plain copy 134.7), 1.2e8 in rows of 1443 95.8, 91.1, 91.1, 98.7; float, 1.2e8 in rows of 128 151.9, 150.9, 150.6, 152.1
// (6.4 TB/s), of 1443 162.5, 178.8, 178.9, 180.0.
template <typename T> constexpr int kFlat = sizeof(T) == 2 ? 4 : 1;
template <typename T> constexpr int kRagged = sizeof(T) == 2 ? 2 : 1;

// One row of n values, or rows of whole quads one behind the other, which are as good as one: the quad of a value is its place / 4.
// ON: values are dropped, else copied.
template <typename T, bool ON>
__global__ __launch_bounds__(kBlock) void dropout_flat(const T *x, T *y, uint64_t n, Dropping d) {
  constexpr int V = kVec<T>, U = kFlat<T>;
  typedef typename Packed<T, V>::memory Vector;
  const uint64_t step = ON ? step_of(d) : 0;
  for (uint64_t base = (uint64_t)blockIdx.x * (kBlock * V * U); base < n; base += (uint64_t)gridDim.x * (kBlock * V * U)) {
    typename Packed<T, V>::type v[U];
    const auto place = [&](int u) { return base + (uint64_t)((u * kBlock + threadIdx.x) * V); };
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t i = place(u);
      v[u] = (T)0;
      if (i + V <= n) {
        v[u] = __builtin_nontemporal_load((const Vector *)(x + i));
      } else if (i < n) {
#pragma unroll
        for (int j = 0; j < V; j++)
          if (i + j < n) v[u][j] = x[i + j];
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t i = place(u);
      Floats<V> f = floats<V>(v[u]);
      if constexpr (ON) drop_columns(f, d, step, i / 4);
      v[u] = rounded<T>(f);
      if (i + V <= n) {
        __builtin_nontemporal_store(v[u], (Vector *)(y + i));
      } else if (i < n) {
#pragma unroll
        for (int j = 0; j < V; j++)
          if (i + j < n) y[i + j] = v[u][j];
      }
    }
  }
}

// Any rows, of `pieces` pieces of V columns each, the last of a row not always whole.  The row of the first piece that a block takes
// at once takes a division (of 32 bits where all pieces can be counted in them: one of 64 bits is as long as the draws); that
// of the others follows from it, by a comparison if a row has more pieces than a block has threads, by a product with
// 1 / pieces otherwise (exact: the numbers are below 512, and half a piece lies between a whole quotient and the next error).
template <typename T, bool ON>
__global__ __launch_bounds__(kBlock) void dropout_rows(const T *x, int64_t x_stride, T *y, int64_t y_stride, uint64_t total, uint32_t width,
                                                       uint32_t pieces, float inv_pieces, Dropping d) {
  constexpr int V = kVec<T>, U = kRagged<T>;
  const uint64_t step = ON ? step_of(d) : 0;
  for (uint64_t base = (uint64_t)blockIdx.x * (kBlock * U); base < total; base += (uint64_t)gridDim.x * (kBlock * U)) {
    typename Packed<T, V>::type v[U];
    uint64_t row[U];
    uint32_t c[U], columns[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint64_t first = base + u * kBlock;
      row[u] = total >> 32 ? first / pieces : (uint64_t)((uint32_t)first / pieces);
      const uint32_t piece = (uint32_t)(first - row[u] * pieces) + threadIdx.x;
      const uint32_t more = pieces >= kBlock ? piece >= pieces : (uint32_t)(((float)piece + 0.5f) * inv_pieces);
      row[u] += more;
      c[u] = (piece - more * pieces) * V;
      columns[u] = first + threadIdx.x < total ? width : 0; // a piece that is not there is one of a row without columns
      v[u] = load_raw<V, Rows::kLong>(x + (int64_t)row[u] * x_stride, c[u], columns[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      Floats<V> f = floats<V>(settled<V, Rows::kLong>(v[u], c[u], width));
      if constexpr (ON) drop_columns(f, d, step, row[u] * d.quads + c[u] / 4);
      store_columns<V, Rows::kLong>(y + (int64_t)row[u] * y_stride, c[u], columns[u], f);
    }
  }
}

template <typename T, bool ON> void launch(const hctr_dropout_args &a, const Dropping &d) {
  const uint32_t width = (uint32_t)a.width, pieces = div_up(a.width, kVec<T>);
  const bool flat = a.rows == 1 || (width % 4 == 0 && a.x.stride == (int64_t)a.width && a.y.stride == (int64_t)a.width);
  const uint64_t total = flat ? (a.rows * width + kVec<T> - 1) / kVec<T> : a.rows * pieces;
  const uint64_t per_block = kBlock * (flat ? kFlat<T> : kRagged<T>);
  const dim3 blocks((unsigned)std::min<uint64_t>((total + per_block - 1) / per_block, (1u << 31) / kBlock)), threads(kBlock);
  const hipStream_t s = (hipStream_t)a.stream;
  if (flat)
    hipLaunchKernelGGL((dropout_flat<T, ON>), blocks, threads, 0, s, (const T *)a.x.data, (T *)a.y.data, a.rows * width, d);
  else
    hipLaunchKernelGGL((dropout_rows<T, ON>), blocks, threads, 0, s, (const T *)a.x.data, a.x.stride, (T *)a.y.data, a.y.stride, total, width,
                       pieces, 1.f / (float)pieces, d);
  HCTR_HIP(hipGetLastError());
}

} // namespace

bool make_dropping(const hctr_drop &d, size_t width, Dropping &out) {
  HCTR_CHECK(d.p >= 0.0 && d.p <= 1.0, "the probability of dropping a value must be in 0..1");
  const double words = std::nearbyint(d.p * 4294967296.0); // that drop their value
  out.seed = d.seed;
  out.step = d.step;
  out.step_dev = d.step_dev;
  out.quads = (width + 3) / 4;
  out.scale = d.p < 1.0 ? (float)(1.0 / (1.0 - d.p)) : 0.f;
  out.last = words >= 1.0 ? (uint32_t)(words - 1.0) : 0;
  return words >= 1.0;
}

void check_matrix(const hctr_matrix &m, size_t rows, size_t width, bool out, const char *name) {
  HCTR_CHECK(m.data, std::string(name) + ": null pointer");
  HCTR_CHECK(!out || rows <= 1 || m.stride >= (int64_t)width || m.stride <= -(int64_t)width,
             std::string(name) + ": the rows of a result overlap");
}

void dropout(const hctr_dropout_args &a) {
  HCTR_CHECK(a.width >= 1 && a.width < (1u << 31), "dropout: the width must be in 1..2^31 - 1");
  HCTR_CHECK(a.dtype == HCTR_F32 || a.dtype == HCTR_BF16 || a.dtype == HCTR_F16, "dropout: unknown type");
  Dropping d;
  const bool on = make_dropping(a.drop, a.width, d);
  if (!a.rows) return;
  check_matrix(a.x, a.rows, a.width, false, "dropout: x");
  check_matrix(a.y, a.rows, a.width, true, "dropout: y");
  if (a.dtype == HCTR_F32) on ? launch<float, true>(a, d) : launch<float, false>(a, d);
  else if (a.dtype == HCTR_BF16) on ? launch<bf16_t, true>(a, d) : launch<bf16_t, false>(a, d);
  else on ? launch<f16_t, true>(a, d) : launch<f16_t, false>(a, d);
}

} // namespace hctr
