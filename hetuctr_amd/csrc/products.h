// What the operators made of matrix products share: results and partial sums, the choice of tiles, and the kernels around the products.
#pragma once
#include <string>

#include "../../include/hetuctr_hip.h"
#include "matmul.h"

namespace hctr {

// A result of `rows` x `columns` values; or two, one below the other, the second from row `second_from` on (to: null: not wanted).
struct Result {
  void *to[2];
  int64_t stride[2]; // elements
  uint32_t rows, columns, second_from;
  const float *scale;      // what every value is multiplied by, or null
  const uint32_t *row_of;  // where a row goes, or null: its own place
};

// columns `column` .. `column` + V - 1 of a row, or as many of them as there are
template <int V, typename T> __device__ __forceinline__ void write(T *row, uint32_t column, uint32_t columns, typename Packed<T, V>::type x) {
  if (column + V <= columns) {
    *(typename Packed<T, V>::memory *)(row + column) = x;
  } else {
#pragma unroll
    for (int e = 0; e < V - 1; e++)
      if (column + e < columns) row[column + e] = x[e];
  }
}
template <typename T> __device__ __forceinline__ void write4(T *row, uint32_t column, uint32_t columns, f32x4 v) {
  const Floats<4> f = {{v[0], v[1], v[2], v[3]}};
  write<4>(row, column, columns, rounded<T>(f));
}
// a row of a result; null: it is not wanted
template <typename T> __device__ __forceinline__ T *row_of(const Result &r, uint32_t row) {
  if (r.row_of) row = r.row_of[row];
  const bool second = row >= r.second_from;
  row -= second ? r.second_from : 0;
  T *to = (T *)(second ? r.to[1] : r.to[0]);
  return to && row < r.rows ? to + (int64_t)row * (second ? r.stride[1] : r.stride[0]) : nullptr;
}

// A product, cut along k into `splits` parts where its tiles alone would leave the card idle: each part's sums go to `partial` as floats
// ([split][rows][columns, up to a multiple of four]), and join_parts adds them up.
struct ProductArgs {
  Operand a, b;
  uint32_t rows, columns, k;
  const uint32_t *rows_there, *k_there; // device memory: how many rows, or how much of k, there is; or null: all
  uint32_t row_tiles, column_tiles, splits, band;
  float *partial; // null: the sums are the result
  bool add;       // to what `partial` holds
  Result result;
};

// 16-bit types and floats have a tile of each size.
struct Shape {
  int tile;
  uint32_t splits;
};
Shape shape_of(size_t rows, size_t columns, size_t k, int size, bool paired, bool may_split);
inline size_t parts_bytes(size_t rows, size_t columns, uint32_t splits) { return splits * rows * ((columns + 3) / 4 * 4) * sizeof(float); }

// a kAlong, b kAcross, a second matrix of b behind the first: rows x columns += a b
template <typename T> void launch_forward_product(ProductArgs &p, int tile, hipStream_t s);
// both kAcross
template <typename T> void launch_across_product(ProductArgs &p, int tile, hipStream_t s);
template <typename T> void launch_join(const ProductArgs &p, hipStream_t s);
// The threads of a block that makes a tile.  A launch has fewer than 2^32: two for each row and column of tiles, so that only results that no card
// holds have too many (of a gated layer, whose tiles of 128 are 64 columns of the result, 2^37 values).
inline uint32_t tile_threads(uint32_t row_tiles, uint32_t column_tiles, int tile, const char *what) {
  HCTR_CHECK((uint64_t)row_tiles * column_tiles * (2 * tile) < (1ull << 32), std::string(what) + ": too many tiles");
  return 2 * tile;
}

// ---- matrices that do not begin, or end their rows, at a multiple of 16 bytes, are laid out once more -------------------------
struct Layout {
  const char *at;
  int64_t stride; // bytes
};
constexpr int64_t kMaxStride = 1 << 23; // bytes: 256 rows are counted in 31 bits
inline size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }
inline size_t size_of(int dtype) { return dtype == HCTR_F32 ? 4 : 2; }
// whether tiles can be read from where the matrix is
inline bool fits(const hctr_matrix &m, size_t rows, size_t width, size_t size) {
  return (uintptr_t)m.data % 16 == 0 && width * size % 16 == 0 && (rows <= 1 || (m.stride > 0 && m.stride * (int64_t)size % 16 == 0 && m.stride * (int64_t)size <= kMaxStride));
}
inline size_t laid_out_bytes(const hctr_matrix &m, size_t rows, size_t width, size_t size) {
  return fits(m, rows, width, size) ? 0 : up(rows * up(width * size, 16), 256);
}
// `space` moves on by laid_out_bytes
Layout laid_out(const hctr_matrix &m, size_t rows, size_t width, int dtype, char *&space, hipStream_t s);
template <typename T> void launch_copy_rows(const hctr_matrix &m, size_t rows, size_t width, char *to, size_t to_stride, hipStream_t s);

// sums[c] = the sum over the `rows` (or as many as *rows_there / per, rounded up) rows of partial[row][columns], times *scale: element c of
// out[0], or c - second_from of out[1], of `count` each (null: not wanted)
struct ColumnSums {
  const float *partial;
  uint32_t rows, columns, second_from, count;
  const uint32_t *rows_there;
  uint32_t per;
  const float *scale;
  void *out[2];
};
void launch_column_sums(const ColumnSums &c, int dtype, hipStream_t s);

// element c of a bias of `n`: floats, or values of T if `narrow`; null: zeros
template <typename T> __device__ __forceinline__ float bias_at(const void *bias, bool narrow, uint32_t c, uint32_t n) {
  return !bias || c >= n ? 0.f : narrow ? (float)((const T *)bias)[c] : ((const float *)bias)[c];
}

inline void check_sizes(size_t rows, size_t width, size_t across, size_t most_across, const char *what, const char *name) {
  HCTR_CHECK(rows < (1u << 31) - 65536, std::string(what) + ": too many rows");
  HCTR_CHECK(width >= 1 && width <= (1u << 20), std::string(what) + ": the width must be in 1..2^20");
  HCTR_CHECK(across >= 1 && across <= most_across, std::string(what) + ": " + name);
}
inline void check_dtype(int t, const char *what) { HCTR_CHECK(t == HCTR_F32 || t == HCTR_BF16 || t == HCTR_F16, std::string(what) + ": unknown type"); }
inline void check_space(const void *workspace, size_t bytes, size_t need, const char *what) {
  HCTR_CHECK(!need || (workspace && (uintptr_t)workspace % 16 == 0 && bytes >= need),
             std::string(what) + ": the workspace is missing, too small or not 16-byte aligned");
}

} // namespace hctr
