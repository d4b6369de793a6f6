#include "clip.h"

#include <algorithm>
#include <vector>

#include "products.h"

namespace hctr {
namespace {

constexpr int kBlock = 256;
// Pieces of 16 bytes that a thread has under way: a block takes a chunk of LOADS * 4 KiB of one gradient at a time.  Eight where there are few
// chunks, whose blocks make the norm for themselves as well, four where there are many (us, 28.8 MB in 17 gradients 17.9 with eight, 20.8
// with four; 4.1 GB 2130 and 2031).
constexpr uint64_t chunk_bytes(int loads) { return (uint64_t)kBlock * 16 * loads; }
constexpr int kFewLoads = 8, kManyLoads = 4;
// Blocks of a call in all, which stay: each leaves one sum, and every block that scales adds them all up for itself, in the same order.
constexpr uint32_t kMostBlocks = 2048;
constexpr int kMostEntries = 128; // gradients that the arguments of one launch name

struct Entries {
  const void *values[kMostEntries];
  void *into[kMostEntries];
  uint64_t count[kMostEntries];
  uint32_t first[kMostEntries]; // chunk
  uint8_t dtype[kMostEntries];
  uint32_t entries, chunks;
};

template <typename F> __device__ __forceinline__ void with_entry(const Entries &e, uint32_t chunk, F &&f) {
  uint32_t low = 0, high = e.entries; // the last entry whose first chunk is not behind this one
  while (high - low > 1) {
    const uint32_t middle = (low + high) / 2;
    const bool behind = e.first[middle] > chunk;
    low = behind ? low : middle, high = behind ? middle : high;
  }
  const uint32_t in = chunk - e.first[low];
  if (e.dtype[low] == HCTR_F32) f((const float *)e.values[low], (float *)e.into[low], e.count[low], in);
  else if (e.dtype[low] == HCTR_BF16) f((const bf16_t *)e.values[low], (bf16_t *)e.into[low], e.count[low], in);
  else f((const f16_t *)e.values[low], (f16_t *)e.into[low], e.count[low], in);
}

// f(piece, place, how many of its values are there) for the LOADS pieces of 16 bytes that a thread has of a chunk, all loaded first;
// meanwhile(): what is done while they are under way
template <int LOADS, bool ONCE, typename T, typename M, typename F> __device__ __forceinline__ void pieces_of(const T *values, uint64_t count, uint32_t chunk, M &&meanwhile, F &&f) {
  constexpr int V = kVec<T>;
  typedef typename Packed<T, V>::memory Loose;
  const uint64_t base = (uint64_t)chunk * (chunk_bytes(LOADS) / sizeof(T)) + threadIdx.x * V;
  typename Packed<T, V>::type v[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    const uint64_t at = base + (uint64_t)i * (kBlock * V);
    v[i] = (T)0;
    if (at + V <= count) {
      v[i] = ONCE ? __builtin_nontemporal_load((const Loose *)(values + at)) : *(const Loose *)(values + at);
    } else if (at < count) {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (at + j < count) v[i][j] = values[at + j];
    }
  }
  meanwhile();
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    const uint64_t at = base + (uint64_t)i * (kBlock * V);
    if (at < count) f(v[i], at, at + V <= count ? (uint32_t)V : (uint32_t)(count - at));
  }
}

// v over the block, the same in all threads
__device__ __forceinline__ double block_total(double v) {
  __shared__ double sums[kBlock / kWave];
#pragma unroll
  for (int mask = 32; mask; mask /= 2) v += __shfl_xor(v, mask);
  if (lane_id() == 0) sums[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kBlock / kWave; i++) v += sums[i];
  return v;
}

// Bound by memory: 4.1 GB 675 us, 6.1 TB/s.  In 64 bits a square cannot leave the range, and the sums' order does not matter to a float's
// precision; for 16-bit values the conversions take about half of the time that the memory leaves.
template <int LOADS> __global__ __launch_bounds__(kBlock) void sum_squares(Entries e, double *sums) {
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < e.chunks; chunk += gridDim.x)
    with_entry(e, chunk, [&](const auto *values, auto *, uint64_t count, uint32_t in) {
      pieces_of<LOADS, false>(values, count, in, [] {}, [&](const auto &v, uint64_t, uint32_t) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(v) / sizeof(*values)); j++) {
          const double d = (double)(float)v[j];
          sum = __builtin_fma(d, d, sum);
        }
      });
    });
  sum = block_total(sum);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

__device__ __forceinline__ double total_norm(const double *sums, uint32_t count) {
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < count; i += kBlock) sum += sums[i];
  return sqrt(block_total(sum));
}

// the norm, as a float and for scale_gradients; either may be null
__global__ __launch_bounds__(kBlock) void finish_norm(const double *sums, uint32_t count, const float *given, float *norm, double *whole) {
  const double n = given ? (double)*given : total_norm(sums, count);
  if (threadIdx.x) return;
  if (norm) *norm = (float)n;
  if (whole) *whole = n;
}

// Bound by memory: 4.1 GB read and written 1390 us, 5.9 TB/s.  The chunks are taken in the other direction than by sum_squares: what was read last is still in the last cache.  The norm is `given`, or
// `whole`, or made of the sums by every block.
template <int LOADS> __global__ __launch_bounds__(kBlock) void scale_gradients(Entries e, const double *sums, uint32_t count, const float *given, const double *whole, float max_norm, float *norm) {
  bool known = false, same = false;
  float factor = 1.f;
  // (the block's first values are under way by then)
  const auto find = [&] {
    if (known) return;
    known = true;
    const double n = given ? (double)*given : whole ? *whole : total_norm(sums, count);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    same = n <= (double)max_norm;
    factor = same ? 1.f : (float)((double)max_norm / n);
  };
  for (uint32_t i = blockIdx.x; i < e.chunks; i += gridDim.x)
    with_entry(e, e.chunks - 1 - i, [&](const auto *values, auto *into, uint64_t total, uint32_t in) {
      if (same && values == into) return;
      pieces_of<LOADS, true>(values, total, in, find, [&](const auto &v, uint64_t at, uint32_t there) {
        if (same && values == into) return;
        typedef std::remove_const_t<std::remove_pointer_t<decltype(into)>> T;
        constexpr int V = kVec<T>;
        Floats<V> f = floats<V>(v);
        if (!same)
#pragma unroll
          for (int j = 0; j < V; j++) f.v[j] *= factor;
        const auto x = rounded<T>(f);
        if (there == V) {
          __builtin_nontemporal_store(x, (typename Packed<T, V>::memory *)(into + at));
        } else {
#pragma unroll
          for (int j = 0; j < V; j++)
            if ((uint32_t)j < there) into[at + j] = x[j];
        }
      });
    });
}

bool many(const hctr_clip_args &a) {
  uint64_t bytes = 0;
  for (size_t i = 0; i < a.count; i++) bytes += a.gradients[i].count * size_of(a.gradients[i].dtype);
  return bytes > 4 * kMostBlocks * chunk_bytes(kFewLoads);
}
uint64_t chunks_of(const hctr_gradient &g, bool many) {
  const uint64_t each = chunk_bytes(many ? kManyLoads : kFewLoads);
  return (g.count * size_of(g.dtype) + each - 1) / each;
}

// Launches: of up to kMostEntries gradients and 2^31 chunks each
template <typename F> void in_launches(const hctr_clip_args &a, bool many, F &&f) {
  Entries e;
  e.entries = e.chunks = 0;
  for (size_t i = 0; i < a.count; i++) {
    const hctr_gradient &g = a.gradients[i];
    if (!g.count) continue;
    const uint64_t chunks = chunks_of(g, many);
    if (e.entries == kMostEntries || (e.entries && e.chunks + chunks >= (1u << 31))) {
      f(e);
      e.entries = e.chunks = 0;
    }
    const uint32_t k = e.entries++;
    e.values[k] = g.values, e.into[k] = g.into, e.count[k] = g.count, e.dtype[k] = (uint8_t)g.dtype, e.first[k] = e.chunks;
    e.chunks += (uint32_t)chunks;
  }
  if (e.entries) f(e);
}
size_t launches_of(const hctr_clip_args &a, bool many) {
  size_t n = 0, entries = 0;
  uint64_t chunks = 0;
  for (size_t i = 0; i < a.count; i++) {
    if (!a.gradients[i].count) continue;
    const uint64_t more = chunks_of(a.gradients[i], many);
    if (entries == kMostEntries || (entries && chunks + more >= (1u << 31))) n++, entries = 0, chunks = 0;
    entries++, chunks += more;
  }
  return n + (entries > 0);
}
uint32_t most_blocks(size_t launches) { return std::max<uint32_t>(64, kMostBlocks / (uint32_t)std::max<size_t>(1, launches)); }

void check(const hctr_clip_args &a) {
  HCTR_CHECK(a.gradients || !a.count, "clip gradients: null pointer");
  for (size_t i = 0; i < a.count; i++) {
    const hctr_gradient &g = a.gradients[i];
    check_dtype(g.dtype, "clip gradients");
    HCTR_CHECK(g.count <= (1ull << 44), "clip gradients: a gradient has more than 2^44 values");
  }
}

// No result, the norm among them, may lie where another result, another gradient or the norm that is given does: blocks read these while others write.
void check_places(const hctr_clip_args &a) {
  struct Span {
    uintptr_t from, to;
    bool written;
  };
  std::vector<Span> spans;
  spans.reserve(2 * a.count + 2);
  for (size_t i = 0; i < a.count; i++) {
    const hctr_gradient &g = a.gradients[i];
    if (!g.count) continue;
    HCTR_CHECK(g.values && g.into, "clip gradients: null pointer");
    const size_t bytes = g.count * size_of(g.dtype);
    spans.push_back({(uintptr_t)g.into, (uintptr_t)g.into + bytes, true});
    if (g.values != g.into) spans.push_back({(uintptr_t)g.values, (uintptr_t)g.values + bytes, false});
  }
  if (a.given) spans.push_back({(uintptr_t)a.given, (uintptr_t)a.given + sizeof(float), false});
  if (a.norm && a.norm != a.given) spans.push_back({(uintptr_t)a.norm, (uintptr_t)a.norm + sizeof(float), true});
  const auto before = [](const Span &x, const Span &y) { return x.from < y.from; };
  if (!std::is_sorted(spans.begin(), spans.end(), before)) std::sort(spans.begin(), spans.end(), before);
  uintptr_t read = 0, written = 0; // where what was seen so far ends
  for (const Span &s : spans) {
    HCTR_CHECK(s.from >= written && (!s.written || s.from >= read), "clip gradients: a result lies where another gradient or result, or the norm, does");
    if (s.written) written = std::max(written, s.to);
    else read = std::max(read, s.to);
  }
}

} // namespace

size_t gradient_workspace(const hctr_clip_args &a) {
  check(a);
  const size_t launches = launches_of(a, many(a));
  return (launches * most_blocks(launches) + 1) * sizeof(double); // the sums, and the norm
}

void gradient_norm(const hctr_clip_args &a, bool clip) {
  check(a);
  HCTR_CHECK(!clip || a.max_norm >= 0.f, "clip gradients: max_norm must not be negative");
  HCTR_CHECK(clip || a.norm, "gradient norm: null pointer");
  if (clip) check_places(a);
  else
    for (size_t i = 0; i < a.count; i++) HCTR_CHECK(!a.gradients[i].count || a.gradients[i].values, "gradient norm: null pointer");
  const bool much = many(a);
  const size_t launches = launches_of(a, much);
  const bool sums_wanted = !clip || !a.given;
  if (sums_wanted) check_space(a.workspace, a.workspace_bytes, gradient_workspace(a), "clip gradients");
  const hipStream_t s = (hipStream_t)a.stream;
  const uint32_t most = most_blocks(launches);
  double *sums = (double *)a.workspace;
  uint32_t count = 0;
  if (sums_wanted)
    in_launches(a, much, [&](const Entries &e) {
      const uint32_t blocks = std::min(e.chunks, most);
      if (much) hipLaunchKernelGGL((sum_squares<kManyLoads>), dim3(blocks), dim3(kBlock), 0, s, e, sums + count);
      else hipLaunchKernelGGL((sum_squares<kFewLoads>), dim3(blocks), dim3(kBlock), 0, s, e, sums + count);
      HCTR_HIP(hipGetLastError());
      count += blocks;
    });
  float *norm = a.norm == a.given ? nullptr : a.norm;
  // Few chunks: the blocks that scale make the norm themselves, a launch less (28.8 MB in 17 gradients: 17.9 us, with three launches 20.6).  Many:
  // a block for each, without that work, moves more at a time than blocks that stay (4.1 GB: 1787 us for blocks that stay, 1445).
  double *whole = clip && much && !a.given ? sums + launches * most : nullptr;
  if ((norm || whole) && (!clip || !launches || whole)) {
    hipLaunchKernelGGL(finish_norm, dim3(1), dim3(kBlock), 0, s, (const double *)sums, count, clip ? a.given : nullptr, norm, whole);
    HCTR_HIP(hipGetLastError());
    if (whole) norm = nullptr;
  }
  if (!clip) return;
  in_launches(a, much, [&](const Entries &e) {
    if (much)
      hipLaunchKernelGGL((scale_gradients<kManyLoads>), dim3(std::min(e.chunks, 1u << 23)), dim3(kBlock), 0, s, e, (const double *)sums, count, a.given, (const double *)whole,
                         a.max_norm, norm);
    else
      hipLaunchKernelGGL((scale_gradients<kFewLoads>), dim3(std::min(e.chunks, kMostBlocks)), dim3(kBlock), 0, s, e, (const double *)sums, count, a.given, (const double *)whole,
                         a.max_norm, norm);
    HCTR_HIP(hipGetLastError());
    norm = nullptr;
  });
}

} // namespace hctr
