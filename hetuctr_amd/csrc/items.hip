// Softmax cross entropy over many items and its gradient: argument checks, workspaces, the launches, what is not a product.
#include "items.h"

#include <algorithm>

#include "dense.h"
#include "few_rows.h"
#include "items_tail.h"

namespace hctr {
namespace {

__global__ __launch_bounds__(256) void count_rows(const int64_t *target, int64_t ignored, const float *dloss, uint32_t rows, uint2 *chunks) {
  __shared__ uint32_t counts[4], sizes[4];
  uint32_t count = 0, most = 0;
  for (uint32_t i = threadIdx.x; i < kChunk; i += 256) {
    const uint32_t r = blockIdx.x * kChunk + i;
    const bool taken = r < rows && target[r] != ignored;
    count += taken;
    if (taken && dloss) most = max(most, size_bits(dloss[r]));
  }
#pragma unroll
  for (int mask = 32; mask; mask /= 2) {
    count += (uint32_t)__shfl_xor((int)count, mask);
    most = max(most, (uint32_t)__shfl_xor((int)most, mask));
  }
  if (lane_id() == 0) counts[threadIdx.x / kWave] = count, sizes[threadIdx.x / kWave] = most;
  __syncthreads();
  if (threadIdx.x == 0) chunks[blockIdx.x] = make_uint2(counts[0] + counts[1] + counts[2] + counts[3], max(max(sizes[0], sizes[1]), max(sizes[2], sizes[3])));
}

// The tiles' parts of 8 rows joined by 128 groups of threads, each of which takes every 128th tile; then the groups', in pairs.
constexpr uint32_t kJoinRows = 8, kJoinGroups = 128;
__global__ __launch_bounds__(kJoinRows *kJoinGroups) void join_tails(const float2 *parts, uint32_t tiles, uint32_t rows, const float *hit, Taken taken, float *loss, float *lse) {
  constexpr uint32_t LOADS = 4;
  __shared__ Tail tails[kJoinGroups][kJoinRows];
  const uint32_t there = *taken.count, x = threadIdx.x % kJoinRows, y = threadIdx.x / kJoinRows, r = blockIdx.x * kJoinRows + x;
  if (blockIdx.x * kJoinRows >= there) return;
  Tail t = {-kInfinity, 0.f};
  for (uint32_t i = y; i < tiles; i += kJoinGroups * LOADS) {
    float2 v[LOADS];
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) v[k] = r < there && i + k * kJoinGroups < tiles ? parts[(uint64_t)(i + k * kJoinGroups) * rows + r] : make_float2(-kInfinity, 0.f);
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) t = join(t, Tail{v[k].x, v[k].y});
  }
  tails[y][x] = t;
  for (uint32_t n = kJoinGroups / 2; n; n /= 2) {
    __syncthreads();
    if (y < n) tails[y][x] = join(tails[y][x], tails[y + n][x]);
  }
  if (y || r >= there) return;
  t = tails[0][x];
  const float log_sum = logf(t.sum), nan = __builtin_nanf("");
  const bool item = taken.target[r] != kNoItem;
  const uint32_t to = taken.row_of[r];
  loss[to] = item ? log_sum + (t.most - hit[r]) : nan;
  if (lse) lse[to] = item ? log_sum + t.most : nan;
}

struct RowsSpace { // of the rows that take part, in the workspace
  size_t taken, chunks, x, bytes;
};
RowsSpace rows_space(size_t rows, size_t width, size_t size) {
  RowsSpace r;
  r.taken = 256 + 4 * up(rows * 4, 256);
  r.chunks = rows > kChunk ? up(div_up(rows, kChunk) * sizeof(uint2), 256) : 0;
  r.x = up(rows * up(width * size, 16), 256);
  r.bytes = r.taken + r.chunks + r.x;
  return r;
}

// Rows that take part, at the workspace's beginning, which moves on
template <typename T> TakeRows take(const hctr_matrix &x, const int64_t *target, int64_t ignored, size_t rows, size_t width, size_t items, const float *dloss, char *&space,
                                    hipStream_t s) {
  const RowsSpace need = rows_space(rows, width, sizeof(T));
  const size_t each = up(rows * 4, 256);
  TakeRows t = {};
  t.x = x.data, t.x_stride = x.stride;
  t.target = target, t.ignored = ignored;
  t.rows = (uint32_t)rows, t.width = (uint32_t)width, t.items = (uint32_t)items;
  char *at = space + 256;
  t.taken = {(uint32_t *)space, (float *)space + 4, (uint32_t *)at, (uint32_t *)(at + each), (float *)(at + 2 * each), (float *)(at + 3 * each)};
  t.to = space + need.taken + need.chunks;
  t.to_stride = (uint32_t)(up(width * sizeof(T), 16) / sizeof(T));
  if (need.chunks) {
    uint2 *chunks = (uint2 *)(space + need.taken);
    t.chunks = chunks;
    hipLaunchKernelGGL(count_rows, dim3(div_up(rows, kChunk)), dim3(256), 0, s, target, ignored, dloss, (uint32_t)rows, chunks);
    HCTR_HIP(hipGetLastError());
  }
  space += need.bytes;
  return t;
}
Operand taken_rows(const TakeRows &t, size_t size) { return {{(const char *)t.to, nullptr}, (int64_t)(t.to_stride * size), t.rows, 0, 0}; }

struct ForwardPlan {
  int tile;
  size_t hit, parts, weight, bytes;
};
ForwardPlan plan_of(const hctr_items_args &a) {
  ForwardPlan p = {};
  if (!a.rows) return p;
  const size_t size = size_of(a.dtype);
  p.tile = a.rows <= kFewRows ? 0 : shape_of(a.rows, a.items, a.width, (int)size, false, false).tile;
  p.hit = up(a.rows * 4, 256);
  p.parts = up(div_up(a.items, p.tile ? p.tile : kFewItems) * a.rows * sizeof(float2), 256);
  p.weight = p.tile ? laid_out_bytes(a.weight, a.items, a.width, size) : 0;
  p.bytes = rows_space(a.rows, a.width, size).bytes + p.hit + p.parts + p.weight;
  return p;
}

template <typename T> void forward(const hctr_items_args &a) {
  const ForwardPlan plan = plan_of(a);
  const hipStream_t s = (hipStream_t)a.stream;
  char *space = (char *)a.workspace;
  TakeRows t = take<T>(a.x, a.target, a.ignore_index, a.rows, a.width, a.items, nullptr, space, s);
  t.loss = a.loss, t.lse = a.lse;
  launch_take_rows<T>(t, s);
  ItemsProduct p = {};
  p.hit = (float *)space, space += plan.hit;
  p.parts = (float2 *)space, space += plan.parts;
  p.rows = t.rows, p.width = t.width, p.items = t.items, p.band = 8;
  p.bias = a.bias, p.narrow = a.bias_dtype != HCTR_F32;
  p.taken = t.taken;
  p.x = taken_rows(t, sizeof(T));
  p.few_x = t.to, p.few_stride = t.to_stride;
  p.loose_weight = a.weight.data, p.loose_stride = a.weight.stride;
  if (plan.tile) {
    const Layout w = laid_out(a.weight, a.items, a.width, a.dtype, space, s);
    p.weight = {{w.at, nullptr}, w.stride, p.items, 0, 0};
  }
  launch_items_forward<T>(p, plan.tile, s);
  hipLaunchKernelGGL(join_tails, dim3(div_up(a.rows, kJoinRows)), dim3(kJoinRows * kJoinGroups), 0, s, (const float2 *)p.parts, p.column_tiles, p.rows, (const float *)p.hit,
                     p.taken, a.loss, a.lse);
  HCTR_HIP(hipGetLastError());
}

// What is held of d at a time: large enough for every product to fill the card, and to make the sums that dx is joined from a small part
// of what is moved.
constexpr size_t kPieceBytes = (size_t)512 << 20;

struct BackwardPlan {
  size_t piece, pieces, d_stride;
  int tile;
  Shape dx, dweight;
  size_t rows, d, acc, parts, sums, weight, bytes;
};
BackwardPlan plan_of(const hctr_items_grad_args &a) {
  BackwardPlan p = {};
  const size_t size = size_of(a.dtype), rows = std::max<size_t>(a.rows, 1);
  p.piece = std::min(up(a.items, 64), std::min<size_t>(kMaxStride / size, std::max<size_t>(2048, kPieceBytes / (rows * size) / 256 * 256)));
  p.pieces = (a.items + p.piece - 1) / p.piece;
  p.d_stride = p.piece;
  const size_t some = std::min(a.items, p.piece);
  p.tile = a.rows <= kFewRows ? 0 : shape_of(a.rows, some, a.width, (int)size, false, false).tile;
  if (a.rows) {
    p.rows = rows_space(a.rows, a.width, size).bytes;
    p.d = up(a.rows * p.d_stride * size, 256);
  }
  if (a.dx.data && a.rows) {
    p.dx = shape_of(a.rows, a.width, some, (int)size, false, true);
    if (p.dx.splits > 1 || p.pieces > 1) p.acc = up(parts_bytes(a.rows, a.width, p.dx.splits), 256);
  }
  // (the slopes of few rows, too, may come from a matrix that is laid out anew: dx takes it)
  if (a.rows && (p.tile || a.dx.data)) p.weight = laid_out_bytes(a.weight, some, a.width, size);
  if (a.dweight.data) {
    p.dweight = shape_of(some, a.width, a.rows, (int)size, false, true);
    if (p.dweight.splits > 1) p.parts = up(parts_bytes(some, a.width, p.dweight.splits), 256);
  }
  if (a.dbias) p.sums = up((p.tile ? div_up(a.rows, p.tile) : 1) * p.d_stride * sizeof(float), 256);
  p.bytes = p.rows + p.d + p.acc + p.parts + p.sums + p.weight;
  return p;
}

template <typename T> void backward(const hctr_items_grad_args &a) {
  const BackwardPlan plan = plan_of(a);
  const hipStream_t s = (hipStream_t)a.stream;
  constexpr size_t size = sizeof(T);
  char *space = (char *)a.workspace;
  TakeRows t = {};
  if (a.rows) {
    t = take<T>(a.x, a.target, a.ignore_index, a.rows, a.width, a.items, a.dloss, space, s);
    t.dloss = a.dloss, t.lse_in = a.lse;
    t.dx = a.dx.data, t.dx_stride = a.dx.stride;
    t.scaled = !std::is_same_v<T, float>;
    launch_take_rows<T>(t, s);
  }
  char *d = space, *acc = d + plan.d, *parts = acc + plan.acc, *sums = parts + plan.parts, *rest = sums + plan.sums;
  const uint32_t *count = t.taken.count;
  const float *back = t.taken.scale ? t.taken.scale + 1 : nullptr;
  const Operand slopes = {{d, nullptr}, (int64_t)(plan.d_stride * size), 0, 0, 0};
  ProductArgs q = {}; // dx
  for (size_t i = 0; i < plan.pieces; i++) {
    const size_t first = i * plan.piece, some = std::min(a.items - first, plan.piece);
    const hctr_matrix weight = {(char *)a.weight.data + (int64_t)first * a.weight.stride * (int64_t)size, a.weight.stride};
    Layout w = {};
    if (a.rows) {
      ItemsProduct p = {};
      if (plan.tile || a.dx.data) {
        char *to = rest;
        w = laid_out(weight, some, a.width, a.dtype, to, s);
        p.weight = {{w.at, nullptr}, w.stride, (uint32_t)some, 0, 0};
      }
      p.rows = t.rows, p.width = t.width, p.items = (uint32_t)some, p.first = (uint32_t)first, p.band = 8;
      p.narrow = a.bias_dtype != HCTR_F32;
      p.bias = a.bias ? (const char *)a.bias + first * (p.narrow ? size : 4) : nullptr;
      p.taken = t.taken;
      p.x = taken_rows(t, size);
      p.few_x = t.to, p.few_stride = t.to_stride;
      p.loose_weight = weight.data, p.loose_stride = weight.stride;
      p.d = d, p.d_stride = (uint32_t)plan.d_stride;
      p.sums = a.dbias ? (float *)sums : nullptr;
      launch_items_gradient<T>(p, plan.tile, s);
    }
    if (a.dbias) {
      const size_t rows_each = plan.tile ? plan.tile : kFewRows, wide = a.bias_dtype == HCTR_F32 ? 4 : size;
      launch_column_sums({(const float *)sums, (uint32_t)((a.rows + rows_each - 1) / rows_each), (uint32_t)plan.d_stride, ~0u, (uint32_t)some, count, (uint32_t)rows_each, back,
                          {(char *)a.dbias + first * wide, nullptr}}, a.bias_dtype, s);
    }
    if (a.dx.data && a.rows) {
      q = {};
      q.a = slopes, q.a.rows = t.rows;
      q.b = {{w.at, nullptr}, w.stride, t.width, ~0u, (uint32_t)some};
      q.rows = t.rows, q.columns = t.width, q.k = (uint32_t)some;
      q.rows_there = count;
      q.splits = plan.dx.splits, q.band = 8;
      q.partial = plan.acc ? (float *)acc : nullptr;
      q.add = i > 0;
      q.result = {{a.dx.data, nullptr}, {a.dx.stride, 0}, q.rows, q.columns, ~0u, back, t.taken.row_of};
      launch_forward_product<T>(q, plan.dx.tile, s);
    }
    if (a.dweight.data) {
      const hctr_matrix dweight = {(char *)a.dweight.data + (int64_t)first * a.dweight.stride * (int64_t)size, a.dweight.stride};
      ProductArgs v = {};
      v.a = slopes, v.a.rows = (uint32_t)some;
      v.b = taken_rows(t, size), v.b.rows = (uint32_t)a.width;
      v.rows = (uint32_t)some, v.columns = (uint32_t)a.width, v.k = (uint32_t)a.rows;
      v.k_there = count;
      v.splits = plan.dweight.splits, v.band = 8;
      v.partial = plan.parts ? (float *)parts : nullptr;
      v.result = {{dweight.data, nullptr}, {dweight.stride, 0}, v.rows, v.columns, ~0u, back, nullptr};
      launch_across_product<T>(v, plan.dweight.tile, s);
      if (v.partial) launch_join<T>(v, s);
    }
  }
  if (q.partial) launch_join<T>(q, s);
}

template <typename A> void check(const A &a) {
  check_dtype(a.dtype, "linear cross entropy");
  check_sizes(a.rows, a.width, a.items, ((size_t)1 << 31) - 65536, "linear cross entropy", "there must be 1 to 2^31 - 65536 items");
}

} // namespace

size_t linear_cross_entropy_workspace(const hctr_items_args &a) {
  check(a);
  return plan_of(a).bytes;
}
size_t linear_cross_entropy_backward_workspace(const hctr_items_grad_args &a) {
  check(a);
  return plan_of(a).bytes;
}

void linear_cross_entropy(const hctr_items_args &a) {
  check(a);
  HCTR_CHECK(!a.bias || a.bias_dtype == HCTR_F32 || a.bias_dtype == a.dtype, "linear cross entropy: the bias is of the matrices' type or float");
  if (!a.rows) return;
  check_matrix(a.x, a.rows, a.width, false, "linear cross entropy: x");
  check_matrix(a.weight, a.items, a.width, false, "linear cross entropy: weight");
  HCTR_CHECK(a.target && a.loss, "linear cross entropy: target or loss: null pointer");
  check_space(a.workspace, a.workspace_bytes, plan_of(a).bytes, "linear cross entropy");
  if (a.dtype == HCTR_F32) forward<float>(a);
  else if (a.dtype == HCTR_BF16) forward<bf16_t>(a);
  else forward<f16_t>(a);
}

void linear_cross_entropy_backward(const hctr_items_grad_args &a) {
  check(a);
  HCTR_CHECK(!(a.bias || a.dbias) || a.bias_dtype == HCTR_F32 || a.bias_dtype == a.dtype, "linear cross entropy: the bias is of the matrices' type or float");
  if (a.rows) {
    check_matrix(a.x, a.rows, a.width, false, "linear cross entropy: x");
    check_matrix(a.weight, a.items, a.width, false, "linear cross entropy: weight");
    HCTR_CHECK(a.target && a.dloss && a.lse, "linear cross entropy: target, dloss or lse: null pointer");
    if (a.dx.data) check_matrix(a.dx, a.rows, a.width, true, "linear cross entropy: dx");
  }
  if (a.dweight.data) check_matrix(a.dweight, a.items, a.width, true, "linear cross entropy: dweight");
  check_space(a.workspace, a.workspace_bytes, plan_of(a).bytes, "linear cross entropy");
  if (a.dtype == HCTR_F32) backward<float>(a);
  else if (a.dtype == HCTR_BF16) backward<bf16_t>(a);
  else backward<f16_t>(a);
}

} // namespace hctr
