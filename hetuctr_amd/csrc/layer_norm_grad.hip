// The gradient of layer normalisation: of the rows, and of weight and bias.
//
// The rows' gradients need two sums over each row.  Those of weight and bias are sums over all rows: every block adds up the rows
// that it works on, writes one row of partial sums, and a second kernel adds those up in the order of the blocks, so that the
// result does not depend on which block is done first.
#include <algorithm>

#include "layer_norm.h"

namespace hctr {
namespace {

constexpr int kBlock = 256;

// One block per row at a time, which it reads twice; its sums for weight and bias lie in its row of `partial` from the first row
// on: rows of any width.
template <typename S, typename A, bool ADD, bool DROP>
__global__ __launch_bounds__(kBlock) void grad_wide(NormBackward a) {
  constexpr int V = kVec<S>;
  __shared__ float smem[kBlock / kWave];
  const uint64_t step = DROP ? step_of(a.drop) : 0;
  float *dweight = a.partial ? a.partial + (uint64_t)blockIdx.x * 2 * a.width : nullptr, *dbias = dweight + a.width;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float mean = a.mean[r], rstd = a.rstd[r];
    const auto gradient = [&](uint32_t c) { // of y, before what was dropped behind the normalisation
      Floats<V> f = load_columns<V>((const A *)a.dy + (int64_t)r * a.dy_stride, c, a.width);
      if constexpr (DROP && !ADD) drop_columns(f, a.drop, step, r * a.drop.quads + c / 4);
      return f;
    };
    const auto normal = [&](uint32_t c) {
      Floats<V> f = load_columns<V>((const S *)a.s + (int64_t)r * a.s_stride, c, a.width);
#pragma unroll
      for (int j = 0; j < V; j++) f.v[j] = (f.v[j] - mean) * rstd;
      return f;
    };
    float sum_g = 0.f, sum_gh = 0.f;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kBlock * V) {
      const Floats<V> g = gradient(c), h = normal(c), w = load_affine<V, A>(a.weight, a.narrow, c, a.width, 1.f);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float gw = g.v[j] * w.v[j];
        if (c + j < a.width) {
          sum_g += gw;
          sum_gh = fmaf(gw, h.v[j], sum_gh);
        }
      }
      if (dweight) {
        const bool first = r == blockIdx.x;
#pragma unroll
        for (int j = 0; j < V; j++)
          if (c + j < a.width) {
            dweight[c + j] = fmaf(g.v[j], h.v[j], first ? 0.f : dweight[c + j]);
            dbias[c + j] = g.v[j] + (first ? 0.f : dbias[c + j]);
          }
      }
    }
    const float mean_g = block_sum<kBlock>(sum_g, smem) * a.inv_width, mean_gh = block_sum<kBlock>(sum_gh, smem) * a.inv_width;
    for (uint32_t c = threadIdx.x * V; c < a.width; c += kBlock * V) {
      const Floats<V> g = gradient(c), h = normal(c), w = load_affine<V, A>(a.weight, a.narrow, c, a.width, 1.f);
      Floats<V> d;
#pragma unroll
      for (int j = 0; j < V; j++) d.v[j] = rstd * (fmaf(g.v[j], w.v[j], -mean_g) - h.v[j] * mean_gh);
      if constexpr (ADD) {
        if (a.ds) {
          const Floats<V> more = load_columns<V>((const S *)a.ds + (int64_t)r * a.ds_stride, c, a.width);
#pragma unroll
          for (int j = 0; j < V; j++) d.v[j] += more.v[j];
        }
        if (a.dresidual) store_columns((S *)a.dresidual + (int64_t)r * a.dresidual_stride, c, a.width, d);
        if (a.dx) {
          if constexpr (DROP) drop_columns(d, a.drop, step, r * a.drop.quads + c / 4);
          store_columns((A *)a.dx + (int64_t)r * a.dx_stride, c, a.width, d);
        }
      } else {
        store_columns((S *)a.dx + (int64_t)r * a.dx_stride, c, a.width, d);
      }
    }
  }
}

// one thread per column: the blocks' sums added up in their order
template <typename W>
__global__ __launch_bounds__(kBlock) void sum_partial(const float *__restrict__ partial, uint32_t blocks, uint32_t width,
                                                      W *dweight, W *dbias) {
  const uint32_t c = blockIdx.x * kBlock + threadIdx.x;
  if (c >= width) return;
  float w = 0.f, b = 0.f;
  for (uint32_t i = 0; i < blocks; i++) {
    w += partial[(uint64_t)i * 2 * width + c];
    b += partial[((uint64_t)i * 2 + 1) * width + c];
  }
  if (dweight) dweight[c] = (W)w;
  if (dbias) dbias[c] = (W)b;
}

constexpr unsigned kMostPartials = 1024;
unsigned partial_rows(size_t rows) { return (unsigned)std::min<size_t>(rows, kMostPartials); }

template <typename S, typename A, bool ADD, bool DROP> void launch(const NormBackward &p, hipStream_t s) {
  const unsigned blocks = p.partial ? partial_rows(p.rows) : (unsigned)std::min<uint64_t>(p.rows, 1u << 20);
  hipLaunchKernelGGL((grad_wide<S, A, ADD, DROP>), dim3(blocks), dim3(kBlock), 0, s, p);
  HCTR_HIP(hipGetLastError());
}

template <typename S, typename A> void launch_types(const NormBackward &p, bool add, bool on, hipStream_t s) {
  if (add) on ? launch<S, A, true, true>(p, s) : launch<S, A, true, false>(p, s);
  else on ? launch<S, A, false, true>(p, s) : launch<S, A, false, false>(p, s);
}

template <typename W> void launch_sum(const hctr_norm_grad_args &a, unsigned blocks, hipStream_t s) {
  hipLaunchKernelGGL(sum_partial<W>, dim3(div_up(a.width, kBlock)), dim3(kBlock), 0, s, (const float *)a.workspace, blocks,
                     (uint32_t)a.width, (W *)a.dweight, (W *)a.dbias);
  HCTR_HIP(hipGetLastError());
}

} // namespace

size_t layer_norm_workspace(size_t rows, size_t width) { return (size_t)partial_rows(rows) * 2 * width * sizeof(float); }

void layer_norm_backward(const hctr_norm_grad_args &a, bool add) {
  HCTR_CHECK(a.width >= 1 && a.width < (1u << 31), "layer norm: the width must be in 1..2^31 - 1");
  const bool columns = a.dweight || a.dbias;
  check_types(a.stream_dtype, a.act_dtype, a.affine_dtype, a.weight || columns);
  NormBackward p = {};
  const bool on = make_dropping(a.drop, a.width, p.drop);
  const hipStream_t s = (hipStream_t)a.stream;
  if (a.rows) {
    check_matrix(a.dy, a.rows, a.width, false, "layer norm: dy");
    check_matrix(a.s, a.rows, a.width, false, "layer norm: s");
    HCTR_CHECK(a.mean && a.rstd, "layer norm: mean and rstd of the forward pass are needed");
    if (!add || a.dx.data) check_matrix(a.dx, a.rows, a.width, true, "layer norm: dx");
    if (add && a.dresidual.data) check_matrix(a.dresidual, a.rows, a.width, true, "layer norm: dresidual");
    HCTR_CHECK(!columns || (a.workspace && (uintptr_t)a.workspace % 16 == 0 && a.workspace_bytes >= layer_norm_workspace(a.rows, a.width)),
               "layer norm: the workspace is missing, too small or not 16-byte aligned");
  }
  p.rows = a.rows;
  p.width = (uint32_t)a.width;
  p.inv_width = (float)(1.0 / (double)a.width);
  p.dy = a.dy.data, p.dy_stride = a.dy.stride;
  p.s = a.s.data, p.s_stride = a.s.stride;
  p.dx = a.dx.data, p.dx_stride = a.dx.stride;
  if (add) {
    p.ds = a.dsum.data, p.ds_stride = a.dsum.stride;
    p.dresidual = a.dresidual.data, p.dresidual_stride = a.dresidual.stride;
  }
  p.mean = a.mean, p.rstd = a.rstd;
  p.weight = a.weight;
  p.narrow = a.affine_dtype != HCTR_F32;
  p.partial = columns ? (float *)a.workspace : nullptr;
  if (a.rows) {
    if (a.stream_dtype == HCTR_BF16) launch_types<bf16_t, bf16_t>(p, add, on, s);
    else if (a.stream_dtype == HCTR_F16) launch_types<f16_t, f16_t>(p, add, on, s);
    else if (a.act_dtype == HCTR_BF16) launch_types<float, bf16_t>(p, add, on, s);
    else if (a.act_dtype == HCTR_F16) launch_types<float, f16_t>(p, add, on, s);
    else launch_types<float, float>(p, add, on, s);
  }
  if (!columns) return;
  const unsigned blocks = partial_rows(a.rows);
  if (a.affine_dtype == HCTR_F32) launch_sum<float>(a, blocks, s);
  else if (a.affine_dtype == HCTR_BF16) launch_sum<bf16_t>(a, blocks, s);
  else launch_sum<f16_t>(a, blocks, s);
}

} // namespace hctr
