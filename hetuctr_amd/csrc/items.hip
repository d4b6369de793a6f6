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

// The tiles' parts of ROWS rows joined by the other threads, each of which takes every so many tiles' parts of a row; then theirs, in pairs.  The target's
// logit is one of those that went into the sum, to the bit, and the largest adds 1 to it: no loss is below zero.
struct JoinTails {
  const float2 *parts;
  uint32_t tiles, rows;
  Taken taken;
  float *loss, *lse;
};
template <uint32_t ROWS> __global__ __launch_bounds__(256) void join_tails(JoinTails p) {
  constexpr uint32_t GROUPS = 256 / ROWS, LOADS = 8;
  __shared__ Tail tails[GROUPS][ROWS];
  const uint32_t there = *p.taken.count, x = threadIdx.x % ROWS, y = threadIdx.x / ROWS, row0 = blockIdx.x * ROWS, r = row0 + x;
  if (row0 >= there) return;
  Tail t = {kLowest, 0.f};
  for (uint32_t i = y; i < p.tiles; i += GROUPS * LOADS) {
    float2 v[LOADS];
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) v[k] = r < there && i + k * GROUPS < p.tiles ? p.parts[(uint64_t)(i + k * GROUPS) * p.rows + r] : make_float2(kLowest, 0.f);
#pragma unroll
    for (uint32_t k = 0; k < LOADS; k++) t = join(t, Tail{v[k].x, v[k].y});
  }
  tails[y][x] = t;
  for (uint32_t n = GROUPS / 2; n; n /= 2) {
    __syncthreads();
    if (y < n) tails[y][x] = join(tails[y][x], tails[y + n][x]);
  }
  if (y || r >= there) return;
  t = tails[0][x];
  const float log_sum = log2f(t.sum), hit = p.taken.target[r] == kNoItem ? __builtin_nanf("") : p.taken.hits[r];
  const uint32_t to = p.taken.row_of[r];
  p.loss[to] = (log_sum + (t.most - hit)) * kLog2;
  if (p.lse) p.lse[to] = hit != hit ? hit : (log_sum + t.most) * kLog2;
}

// of the workspace
struct RowsSpace {
  size_t each, taken, chunks, x, bias, bytes; // each: of a number for every row
};
RowsSpace rows_space(size_t rows, size_t width, size_t items, size_t size) {
  RowsSpace r;
  r.each = up(rows, kFilled) * 4;
  r.taken = 256 + 4 * r.each;
  r.chunks = rows > kChunk ? up(div_up(rows, kChunk) * sizeof(uint2), 256) : 0;
  r.x = up(rows * up(width * size, 16), 256);
  r.bias = up(items, kFilled) * sizeof(float);
  r.bytes = r.taken + r.chunks + r.x + r.bias;
  return r;
}

// Rows that take part, at the workspace's beginning, which moves on
template <typename T, typename A> TakeRows take(const A &a, const float *dloss, char *&space, hipStream_t s) {
  const size_t rows = a.rows, width = a.width, items = a.items;
  const RowsSpace need = rows_space(rows, width, items, sizeof(T));
  const size_t each = need.each;
  TakeRows t = {};
  t.x = a.x.data, t.x_stride = a.x.stride;
  t.target = a.target, t.ignored = a.ignore_index;
  t.bias = a.bias, t.narrow = a.bias_dtype != HCTR_F32;
  t.rows = (uint32_t)rows, t.width = (uint32_t)width, t.items = (uint32_t)items;
  char *at = space + 256;
  t.taken = {(uint32_t *)space, (float *)space + 4, (uint32_t *)at, (uint32_t *)(at + each), (float *)(at + 2 * each), (float *)(at + 3 * each), (float *)(at + 3 * each),
             (float *)(space + need.taken + need.chunks + need.x)};
  t.to = space + need.taken + need.chunks;
  t.to_stride = (uint32_t)(up(width * sizeof(T), 16) / sizeof(T));
  if (need.chunks) {
    uint2 *chunks = (uint2 *)(space + need.taken);
    t.chunks = chunks;
    hipLaunchKernelGGL(count_rows, dim3(div_up(rows, kChunk)), dim3(256), 0, s, a.target, a.ignore_index, dloss, (uint32_t)rows, chunks);
    HCTR_HIP(hipGetLastError());
  }
  space += need.bytes;
  return t;
}
Operand taken_rows(const TakeRows &t, size_t size) { return {{(const char *)t.to, nullptr}, (int64_t)(t.to_stride * size), t.rows, 0, 0}; }

// Narrow matrices of 16 bits hold their rows in registers; few rows take the weights past the LDS; others go by tiles, but for those that
// are few and long: a block for 32 rows shares out k among its waves (us, 35 rows of 8086 columns, 712 items: 67 by tiles, 36 so,
// float 307 and 72).
enum class Way { kFew, kNarrow, kTiles };
Way way_of(size_t rows, size_t width, size_t items, size_t size) {
  if (size == 2 && width <= kNarrow) return Way::kNarrow;
  if (rows <= kFewRows) return Way::kFew;
  return (size_t)div_up(rows, 64) * div_up(items, 64) <= 64 && width * size >= 32 * kStepBytes ? Way::kFew : Way::kTiles;
}

struct ForwardPlan {
  Way way;
  int tile;
  size_t tiles, parts, weight, bytes; // tiles: along the items
};
ForwardPlan plan_of(const hctr_items_args &a) {
  ForwardPlan p = {};
  if (!a.rows) return p;
  const size_t size = size_of(a.dtype);
  p.way = way_of(a.rows, a.width, a.items, size);
  if (p.way == Way::kTiles) p.tile = shape_of(a.rows, a.items, a.width, (int)size, false, false).tile;
  p.tiles = p.way == Way::kNarrow ? narrow_ranges(a.rows, a.items, a.width, false) : div_up(a.items, p.tile ? p.tile : 16 * few_groups(a.rows, a.items));
  p.parts = up(p.tiles * a.rows * sizeof(float2), 256);
  p.weight = p.way == Way::kFew ? 0 : laid_out_bytes(a.weight, a.items, a.width, size);
  p.bytes = rows_space(a.rows, a.width, a.items, size).bytes + p.parts + p.weight;
  return p;
}

ItemsNarrow narrow_of(const TakeRows &t, const Layout &weight) {
  ItemsNarrow n = {};
  n.x = (const char *)t.to, n.x_stride = t.to_stride * 2;
  n.weight = weight.at, n.weight_stride = weight.stride;
  n.rows = t.rows, n.width = t.width, n.items = t.items;
  n.taken = t.taken;
  return n;
}

template <typename T> void forward(const hctr_items_args &a) {
  const ForwardPlan plan = plan_of(a);
  const hipStream_t s = (hipStream_t)a.stream;
  char *space = (char *)a.workspace;
  TakeRows t = take<T>(a, nullptr, space, s);
  t.loss = a.loss, t.lse = a.lse;
  launch_take_rows<T>(t, s);
  float2 *parts = (float2 *)space;
  space += plan.parts;
  Layout w = {};
  if (plan.way != Way::kFew) w = laid_out(a.weight, a.items, a.width, a.dtype, space, s);
  if (plan.way == Way::kNarrow) {
    if constexpr (sizeof(T) == 2) {
      ItemsNarrow n = narrow_of(t, w);
      n.ranges = (uint32_t)plan.tiles;
      n.parts = parts;
      launch_narrow_forward<T>(n, s);
    }
  } else {
    ItemsProduct p = {};
    p.parts = parts;
    p.rows = t.rows, p.width = t.width, p.items = t.items, p.band = 8;
    p.taken = t.taken;
    p.x = taken_rows(t, sizeof(T));
    p.few_x = t.to, p.few_stride = t.to_stride;
    p.loose_weight = a.weight.data, p.loose_stride = a.weight.stride;
    p.weight = {{w.at, nullptr}, w.stride, p.items, 0, 0};
    launch_items_forward<T>(p, plan.tile, s);
  }
  // (few rows: more blocks)
  const JoinTails j = {parts, (uint32_t)plan.tiles, t.rows, t.taken, a.loss, a.lse};
  if (t.rows <= 1024) hipLaunchKernelGGL((join_tails<2>), dim3(div_up(t.rows, 2)), dim3(256), 0, s, j);
  else hipLaunchKernelGGL((join_tails<8>), dim3(div_up(t.rows, 8)), dim3(256), 0, s, j);
  HCTR_HIP(hipGetLastError());
}

// What is held of d at a time, at most: large enough for every product to fill the card, and to make the sums that dx is joined from a small part
// of what is moved.  For that it is d of kPieceItems items at least, however many rows there are.
constexpr size_t kPieceItems = 2048, kPieceBytes = (size_t)512 << 20;

struct BackwardPlan {
  Way way;
  size_t dx_ranges, dweight_ranges; // of the narrow way
  size_t piece, pieces, d_stride;
  int tile;
  Shape dx, dweight;
  size_t rows, d, acc, parts, sums, weight, bytes;
};
BackwardPlan plan_of(const hctr_items_grad_args &a) {
  BackwardPlan p = {};
  const size_t size = size_of(a.dtype), rows = std::max<size_t>(a.rows, 1);
  p.way = way_of(a.rows, a.width, a.items, size);
  if (a.rows && p.way == Way::kNarrow) {
    p.rows = rows_space(a.rows, a.width, a.items, size).bytes;
    p.weight = laid_out_bytes(a.weight, a.items, a.width, size);
    p.dx_ranges = narrow_ranges(a.rows, a.items, a.width, true);
    p.dweight_ranges = narrow_ranges(a.items, a.rows, a.width, true);
    if (a.dx.data) p.acc = up(parts_bytes(a.rows, a.width, (uint32_t)p.dx_ranges), 256);
    if (a.dweight.data && p.dweight_ranges > 1) p.parts = up(parts_bytes(a.items, a.width, (uint32_t)p.dweight_ranges), 256);
    if (a.dbias) p.sums = up(p.dweight_ranges * a.items * sizeof(float), 256);
    p.bytes = p.rows + p.acc + p.parts + p.sums + p.weight;
    return p;
  }
  p.piece = std::min(up(a.items, 64), std::min<size_t>(kMaxStride / size, std::max<size_t>(kPieceItems, kPieceBytes / (rows * size) / 256 * 256)));
  p.pieces = (a.items + p.piece - 1) / p.piece;
  p.d_stride = p.piece;
  const size_t some = std::min(a.items, p.piece);
  p.tile = p.way == Way::kFew ? 0 : shape_of(a.rows, some, a.width, (int)size, false, false).tile;
  if (a.rows) {
    p.rows = rows_space(a.rows, a.width, a.items, size).bytes;
    p.d = up(a.rows * p.d_stride * size, 256);
  }
  if (a.dx.data && a.rows) {
    p.dx = shape_of(a.rows, a.width, some, (int)size, false, true);
    if (p.dx.splits > 1 || p.pieces > 1) p.acc = up(parts_bytes(a.rows, a.width, p.dx.splits), 256);
  }
  // (few rows do not need the weights laid out for their slopes, but dx does)
  if (a.rows && (p.tile || a.dx.data)) p.weight = laid_out_bytes(a.weight, some, a.width, size);
  if (a.dweight.data) {
    p.dweight = shape_of(some, a.width, a.rows, (int)size, false, true);
    if (p.dweight.splits > 1) p.parts = up(parts_bytes(some, a.width, p.dweight.splits), 256);
  }
  if (a.dbias) p.sums = up(div_up(a.rows, p.tile ? p.tile : kFewRows) * p.d_stride * sizeof(float), 256);
  p.bytes = p.rows + p.d + p.acc + p.parts + p.sums + p.weight;
  return p;
}

// Narrow rows: nothing is held of d; the items' sums are made beside the weight's gradient.
template <typename T> void backward_narrow(const hctr_items_grad_args &a, const BackwardPlan &plan, const TakeRows &t, char *space) {
  if constexpr (sizeof(T) == 2) {
    const hipStream_t s = (hipStream_t)a.stream;
    char *acc = space, *parts = acc + plan.acc, *sums = parts + plan.parts, *rest = sums + plan.sums;
    ItemsNarrow n = narrow_of(t, laid_out(a.weight, a.items, a.width, a.dtype, rest, s));
    const auto join = [&](const ItemsNarrow &n, uint32_t rows, const uint32_t *there) {
      ProductArgs q = {};
      q.rows = rows, q.columns = n.width, q.splits = n.ranges, q.partial = n.partial, q.rows_there = there, q.result = n.result;
      launch_join<T>(q, s);
    };
    if (a.dx.data) {
      n.ranges = (uint32_t)plan.dx_ranges;
      n.partial = (float *)acc;
      n.result = {{a.dx.data, nullptr}, {a.dx.stride, 0}, t.rows, t.width, ~0u, t.taken.scale + 1, t.taken.row_of};
      launch_narrow_dx<T>(n, s);
      join(n, t.rows, t.taken.count);
    }
    if (a.dweight.data || a.dbias) {
      n.ranges = (uint32_t)plan.dweight_ranges;
      n.partial = plan.parts ? (float *)parts : nullptr;
      n.sums = a.dbias ? (float *)sums : nullptr;
      n.result = {{a.dweight.data, nullptr}, {a.dweight.stride, 0}, t.items, t.width, ~0u, t.taken.scale + 1, nullptr};
      launch_narrow_dweight<T>(n, s);
      if (n.partial) join(n, t.items, nullptr);
      if (n.sums) launch_column_sums({n.sums, n.ranges, t.items, ~0u, t.items, nullptr, 1, t.taken.scale + 1, {a.dbias, nullptr}}, a.bias_dtype, s);
    }
  }
}

template <typename T> void backward(const hctr_items_grad_args &a) {
  const BackwardPlan plan = plan_of(a);
  const hipStream_t s = (hipStream_t)a.stream;
  constexpr size_t size = sizeof(T);
  char *space = (char *)a.workspace;
  TakeRows t = {};
  if (a.rows) {
    t = take<T>(a, a.dloss, space, s);
    t.dloss = a.dloss, t.lse_in = a.lse;
    t.dx = a.dx.data, t.dx_stride = a.dx.stride;
    t.scaled = !std::is_same_v<T, float>;
    launch_take_rows<T>(t, s);
    if (plan.way == Way::kNarrow) return backward_narrow<T>(a, plan, t, space);
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
  HCTR_CHECK(a.rows <= (1u << 26), "linear cross entropy: too many rows"); // 32 threads each, in a launch
}

} // namespace

// As many blocks as the card holds at a time, of eight tiles of 64 rows at least.
uint32_t narrow_ranges(size_t owned, size_t through, size_t width, bool gradient) {
  const size_t owners = (owned + 255) / (gradient && width > 64 ? 192 : 256), tiles = (through + 63) / 64;
  return (uint32_t)std::max<size_t>(1, std::min((size_t)256 * narrow_share(width, gradient) / std::max<size_t>(1, owners), tiles / 8));
}

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
