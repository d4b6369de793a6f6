// The operators between the table's rows and a dense model: dropout, layer normalisation, both in one pass, their gradients.
#pragma once
#include "../../include/hetuctr_hip.h"
#include "common.h"
#include "philox.h"
#include "values.h"

namespace hctr {

// What a kernel needs to drop values: the word of row r, column c is number c % 4 of philox(r * quads + c / 4, step, seed).
struct Dropping {
  uint64_t seed, step;
  const uint64_t *step_dev; // added to step if not null
  uint64_t quads;           // of a row
  float scale;              // of what is kept
  uint32_t last;            // words up to this one drop their value
};

// V values that begin at column c (a multiple of four) of row r, quad = r * quads + c / 4: dropped, or kept and, if SCALED,
// multiplied by the scale.  A dropped value becomes zero whatever it was: it is never multiplied.
template <bool SCALED = true, int V>
__device__ __forceinline__ void drop_columns(Floats<V> &f, const Dropping &d, uint64_t step, uint64_t quad) {
#pragma unroll
  for (int q = 0; q < V / 4; q++) {
    const Quad w = philox(quad + q, step, d.seed);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float kept = SCALED ? f.v[4 * q + j] * d.scale : f.v[4 * q + j];
      f.v[4 * q + j] = w.w[j] > d.last ? kept : 0.f;
    }
  }
}

__device__ __forceinline__ uint64_t step_of(const Dropping &d) { return d.step + (d.step_dev ? *d.step_dev : 0); }

struct NormForward {
  uint64_t rows;
  uint32_t width;
  float eps, inv_width;
  const void *x, *residual; // residual: only with the sum
  void *sum, *y;            // sum: only with the residual
  int64_t x_stride, residual_stride, sum_stride, y_stride;
  const void *weight, *bias; // either may be null
  bool narrow;               // weight and bias are of the activations' type, else float
  float *mean, *rstd;        // either may be null
  Dropping drop;
};

struct NormBackward {
  uint64_t rows;
  uint32_t width;
  float inv_width;
  const void *dy, *s, *ds; // s: what was normalised; ds: the gradient it has besides, or null
  void *dx, *dresidual;    // either may be null
  int64_t dy_stride, s_stride, ds_stride, dx_stride, dresidual_stride;
  const float *mean, *rstd;
  const void *weight;
  bool narrow;
  float *partial;       // [blocks][2][width] sums for weight and bias, or null
  void *dweight, *dbias; // where blocks of their own make them (few rows); either may be null
  uint32_t row_blocks;   // blocks behind these are the columns'
  Dropping drop;
};

// The entry points of the C ABI behind their guard; the arguments are checked here.
void dropout(const hctr_dropout_args &a);
void layer_norm(const hctr_norm_args &a, bool add);
void layer_norm_backward(const hctr_norm_grad_args &a, bool add);
size_t layer_norm_workspace(size_t rows, size_t width);

void check_types(int stream, int act, int affine, bool has_affine);
// true: values are dropped (p is not, and does not round to, zero)
bool make_dropping(const hctr_drop &d, size_t width, Dropping &out);
// a matrix whose rows a kernel reads, or writes if `out`
void check_matrix(const hctr_matrix &m, size_t rows, size_t width, bool out, const char *name);

} // namespace hctr
