// Dropout whose mask is a function of position, seed and step (philox.h), and the argument checks of the dense operators.
#include <cmath>

#include "dense.h"

namespace hctr {
namespace {

constexpr int kBlock = 256;

// one thread per V columns of a row; ON: values are dropped, else the rows are copied
template <typename T, bool ON>
__global__ __launch_bounds__(kBlock) void dropout_rows(const T *__restrict__ x, int64_t x_stride, T *y, int64_t y_stride,
                                                       uint64_t rows, uint32_t width, uint32_t pieces, Dropping d) {
  constexpr int V = kVec<T>;
  const uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x, row = i / pieces;
  if (row >= rows) return;
  const uint32_t c = (uint32_t)(i - row * pieces) * V;
  Floats<V> f = load_columns<V, Rows::kLong>(x + (int64_t)row * x_stride, c, width);
  if constexpr (ON) drop_columns(f, d, step_of(d), row * d.quads + c / 4);
  store_columns<V, Rows::kLong>(y + (int64_t)row * y_stride, c, width, f);
}

template <typename T> void launch(const hctr_dropout_args &a, const Dropping &d, bool on) {
  const hipStream_t s = (hipStream_t)a.stream;
  const uint32_t width = (uint32_t)a.width, pieces = div_up(a.width, kVec<T>);
  const uint64_t blocks = (a.rows * pieces + kBlock - 1) / kBlock;
  HCTR_CHECK(blocks < (1ull << 31), "dropout: too many values for one call");
  const auto kernel = on ? dropout_rows<T, true> : dropout_rows<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, s, (const T *)a.x.data, a.x.stride, (T *)a.y.data, a.y.stride,
                     a.rows, width, pieces, d);
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
  if (a.dtype == HCTR_F32) launch<float>(a, d, on);
  else if (a.dtype == HCTR_BF16) launch<bf16_t>(a, d, on);
  else launch<f16_t>(a, d, on);
}

} // namespace hctr
