// Rows of a table looked up by token, and what a table learns from them.
//
//   lookup    y[n][d] = keep(n, d) * c * W[t_n][d]
//   gradient  G[k][d] = c * sum over n with t_n = k of keep(n, d) * g[n][d]
//   Adam      torch-fused Adam of W with G, which is never written
//
// c = scale / (1 - p); keep is the dropout's decision for element n * D + d
// (counter_mask.cuh), always true without dropout. Tokens that name no row
// give rows of zeros and no gradient. Arithmetic in 32-bit floats, one
// rounding to the element type at the end.
//
// The gradient goes by sorted tokens (token_order.cuh): the sorted list is cut
// into chunks of equal length, a group of lanes sums the gradient rows of its
// chunk in order and hands each finished row to the epilogue (a store, or
// Adam). A row whose tokens lie in several chunks leaves partial sums that a
// second kernel adds in chunk order. No float atomics: the result is the same
// on every run.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "clad3dgs_b200.h"
#include "counter_mask.cuh"
#include "element_types.cuh"
#include "gaussian_math.cuh"
#include "token_order.cuh"

namespace clad3dgs {
int fail(int code, const std::string& message);  // gaussian_step.cu

// Reads (and clears) the word set by indices outside their table.
cudaError_t token_fault(bool clear, unsigned* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, tokens::g_token_fault, sizeof(*word));
  if (e == cudaSuccess && clear && *word) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbol(tokens::g_token_fault, &zero, sizeof(zero));
  }
  return e;
}

namespace {

using tokens::Index;

constexpr int kThreads = 256;

// How a [.][width] array is cut: vectors of V elements, `lanes` of them side
// by side in one group (a power of two, 32 at most), `slices` groups a row.
struct Cut {
  int lanes;
  int64_t slices;
};

Cut cut_of(int64_t width, int vec) {
  const int64_t vectors = width / vec;
  Cut c{1, 0};
  while (c.lanes < 32 && c.lanes < vectors) c.lanes *= 2;
  c.slices = (vectors + c.lanes - 1) / c.lanes;
  return c;
}

// keep decisions of V elements that begin at element e, as factors 0 or 1.
template <int V>
__device__ __forceinline__ void draw(const CounterMask& mask, unsigned long long offset,
                                     int64_t e, bool (&keep)[V]) {
  uint4 words = mask_words(mask, offset, e / 4);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j > 0 && (e + j) % 4 == 0) words = mask_words(mask, offset, (e + j) / 4);
    keep[j] = mask.keeps(word_of(words, unsigned(e + j) % 4));
  }
}

template <class T, int V, bool kDrop>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(int64_t n, int64_t width, Cut cut, const T* __restrict__ table,
                  int64_t table_stride, Index index, float factor, CounterMask mask,
                  T* __restrict__ out) {
  const unsigned long long offset = kDrop ? mask_offset(mask) : 0;
  const int lane = threadIdx.x % cut.lanes;
  const int64_t groups = int64_t(gridDim.x) * kThreads / cut.lanes;
  for (int64_t job = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / cut.lanes;
       job < n * cut.slices; job += groups) {
    const int64_t i = job / cut.slices;
    const int64_t column = ((job - i * cut.slices) * cut.lanes + lane) * V;
    if (column >= width) continue;
    const uint32_t row = tokens::row_of(index, i);
    Vec<T, V> v{};
    if (row < index.rows) {
      v = *reinterpret_cast<const Vec<T, V>*>(table + row * table_stride + column);
      bool keep[V];
      if (kDrop) draw<V>(mask, offset, i * width + column, keep);
#pragma unroll
      for (int j = 0; j < V; ++j)
        v.v[j] = from_float<T>(!kDrop || keep[j] ? to_float(v.v[j]) * factor : 0.f);
    }
    *reinterpret_cast<Vec<T, V>*>(out + i * width + column) = v;
  }
}

// What becomes of a finished row's gradient.
template <class T>
struct Store {
  T* out;

  template <int V>
  __device__ __forceinline__ void operator()(int64_t at, const float (&sum)[V]) const {
    Vec<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.v[j] = from_float<T>(sum[j]);
    *reinterpret_cast<Vec<T, V>*>(out + at) = v;
  }
};

struct Adam {
  float *table, *first, *second;
  float step;
  double inv_bias2;

  template <int V>
  __device__ __forceinline__ void operator()(int64_t at, const float (&sum)[V]) const {
    constexpr int W = V < 4 ? V : 4;
#pragma unroll
    for (int h = 0; h < V; h += W) {
      auto* p = reinterpret_cast<Vec<float, W>*>(table + at + h);
      auto* m = reinterpret_cast<Vec<float, W>*>(first + at + h);
      auto* v = reinterpret_cast<Vec<float, W>*>(second + at + h);
      Vec<float, W> pv = *p, mv = *m, vv = *v;
#pragma unroll
      for (int j = 0; j < W; ++j)
        torch_adam(pv.v[j], mv.v[j], vv.v[j], sum[h + j], step, inv_bias2);
      *p = pv;
      *m = mv;
      *v = vv;
    }
  }
};

template <class T>
struct Sums {
  int64_t n, rows, width;
  Cut cut;
  int chunk;  // tokens of one group
  const T* grad;
  int64_t stride;
  const uint2* order;
  float factor;
  CounterMask mask;
  float* partial;  // [2 * chunks][width]: a chunk's first row, its last row
};

template <int V>
__device__ __forceinline__ void keep_partial(float* to, const float (&sum)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int h = 0; h < V; h += W) {
    Vec<float, W> v;
#pragma unroll
    for (int j = 0; j < W; ++j) v.v[j] = sum[h + j];
    *reinterpret_cast<Vec<float, W>*>(to + h) = v;
  }
}

template <int V>
__device__ __forceinline__ void add_partial(const float* from, float (&sum)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int h = 0; h < V; h += W) {
    const Vec<float, W> v = *reinterpret_cast<const Vec<float, W>*>(from + h);
#pragma unroll
    for (int j = 0; j < W; ++j) sum[h + j] += v.v[j];
  }
}

template <int V>
__device__ __forceinline__ void times(float (&sum)[V], float factor) {
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] *= factor;
}

template <class T, int V, bool kDrop, class End>
__global__ void __launch_bounds__(kThreads) sum_kernel(const Sums<T> a, const End end) {
  const unsigned long long offset = kDrop ? mask_offset(a.mask) : 0;
  const int64_t job = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / a.cut.lanes;
  const int64_t chunk = job / a.cut.slices;
  const int64_t column =
      ((job - chunk * a.cut.slices) * a.cut.lanes + threadIdx.x % a.cut.lanes) * V;
  const int64_t begin = chunk * a.chunk;
  if (begin >= a.n || column >= a.width) return;
  const int64_t stop = begin + a.chunk < a.n ? begin + a.chunk : a.n;
  uint32_t row = a.order[begin].x;
  bool before = begin > 0 && a.order[begin - 1].x == row;  // the row began in another chunk
  float sum[V] = {};
  for (int64_t i = begin; i < stop; ++i) {
    const uint2 token = a.order[i];
    if (token.x != row) {
      if (before) {
        keep_partial<V>(a.partial + 2 * chunk * a.width + column, sum);
      } else {
        times<V>(sum, a.factor);
        end.template operator()<V>(row * a.width + column, sum);
      }
      before = false;
      row = token.x;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] = 0.f;
    }
    if (row >= a.rows) return;
    const Vec<T, V> g =
        *reinterpret_cast<const Vec<T, V>*>(a.grad + token.y * a.stride + column);
    bool keep[V];
    if (kDrop) draw<V>(a.mask, offset, token.y * a.width + column, keep);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!kDrop || keep[j]) sum[j] += to_float(g.v[j]);
  }
  const bool after = stop < a.n && a.order[stop].x == row;
  if (before || after) {
    keep_partial<V>(a.partial + (2 * chunk + (before ? 0 : 1)) * a.width + column, sum);
  } else {
    times<V>(sum, a.factor);
    end.template operator()<V>(row * a.width + column, sum);
  }
}

// Rows whose tokens lie in several chunks: the group of the chunk a row begins
// in adds the others' partial sums in their order.
template <class T, int V, class End>
__global__ void __launch_bounds__(kThreads) join_kernel(const Sums<T> a, const End end) {
  const int64_t job = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / a.cut.lanes;
  int64_t chunk = job / a.cut.slices;
  const int64_t column =
      ((job - chunk * a.cut.slices) * a.cut.lanes + threadIdx.x % a.cut.lanes) * V;
  const int64_t begin = chunk * a.chunk, stop = begin + a.chunk;
  if (stop >= a.n || column >= a.width) return;
  const uint32_t row = a.order[stop - 1].x;
  if (row >= a.rows || a.order[stop].x != row) return;
  if (begin > 0 && a.order[begin - 1].x == row) return;  // began earlier
  float sum[V] = {};
  add_partial<V>(a.partial + (2 * chunk + 1) * a.width + column, sum);
  for (int64_t at = stop; at < a.n && a.order[at].x == row; at += a.chunk)
    add_partial<V>(a.partial + 2 * ++chunk * a.width + column, sum);
  times<V>(sum, a.factor);
  end.template operator()<V>(row * a.width + column, sum);
}

// Rows that no token names: a gradient of zero. One warp takes 32 rows, each
// lane looks one of them up in the order.
template <class T, int V, class End>
__global__ void __launch_bounds__(kThreads) rest_kernel(const Sums<T> a, const End end) {
  const int64_t first = (blockIdx.x * int64_t(kThreads) + threadIdx.x) / 32 * 32;
  if (first >= a.rows) return;
  const int lane = threadIdx.x & 31;
  const int64_t mine = first + lane;
  bool named = true;
  if (mine < a.rows) {
    int64_t low = 0, high = a.n;
    while (low < high) {
      const int64_t middle = (low + high) / 2;
      if (a.order[middle].x < mine) low = middle + 1;
      else high = middle;
    }
    named = low < a.n && a.order[low].x == mine;
  }
  unsigned left = __ballot_sync(~0u, !named);
  const float zero[V] = {};
  while (left) {
    const int64_t row = first + __ffs(left) - 1;
    left &= left - 1;
    for (int64_t column = lane * V; column < a.width; column += 32 * V)
      end.template operator()<V>(row * a.width + column, zero);
  }
}

int chunk_of(int64_t n) { return n > 0 ? 32 : 32; }

int64_t chunks_of(int64_t n) { return (n + chunk_of(n) - 1) / chunk_of(n); }

unsigned grid_of(int64_t threads) { return unsigned((threads + kThreads - 1) / kThreads); }

template <class T, int V, class End>
cudaError_t run_sums(Sums<T> a, const End& end, bool drop, cudaStream_t stream) {
  a.cut = cut_of(a.width, V);
  if (a.n > 0) {
    const unsigned grid = grid_of(chunks_of(a.n) * a.cut.slices * a.cut.lanes);
    if (drop) sum_kernel<T, V, true, End><<<grid, kThreads, 0, stream>>>(a, end);
    else sum_kernel<T, V, false, End><<<grid, kThreads, 0, stream>>>(a, end);
    join_kernel<T, V, End><<<grid, kThreads, 0, stream>>>(a, end);
  }
  rest_kernel<T, V, End><<<grid_of((a.rows + 31) / 32 * 32), kThreads, 0, stream>>>(a, end);
  return cudaGetLastError();
}

// Vector length: the longest that every row of every array starts on.
template <class T, class End>
cudaError_t pick_sums(const Sums<T>& a, const End& end, int bytes, bool drop,
                      cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (bytes >= 16) return run_sums<T, 8, End>(a, end, drop, stream);
    if (bytes >= 8) return run_sums<T, 4, End>(a, end, drop, stream);
    if (bytes >= 4) return run_sums<T, 2, End>(a, end, drop, stream);
  } else {
    if (bytes >= 16) return run_sums<T, 4, End>(a, end, drop, stream);
    if (bytes >= 8) return run_sums<T, 2, End>(a, end, drop, stream);
  }
  return run_sums<T, 1, End>(a, end, drop, stream);
}

template <class T, int V>
cudaError_t run_lookup(int64_t n, int64_t width, const void* table, int64_t stride,
                       const Index& index, float factor, const CounterMask& mask, bool drop,
                       void* out, cudaStream_t stream) {
  const Cut cut = cut_of(width, V);
  const int64_t threads = n * cut.slices * cut.lanes;
  const unsigned grid =
      unsigned(std::min<int64_t>((threads + kThreads - 1) / kThreads, int64_t(1) << 20));
  auto* kernel = drop ? lookup_kernel<T, V, true> : lookup_kernel<T, V, false>;
  kernel<<<grid, kThreads, 0, stream>>>(n, width, cut, static_cast<const T*>(table), stride,
                                        index, factor, mask, static_cast<T*>(out));
  return cudaGetLastError();
}

template <class T>
cudaError_t pick_lookup(int64_t n, int64_t width, const void* table, int64_t stride,
                        const Index& index, float factor, const CounterMask& mask, bool drop,
                        void* out, cudaStream_t stream) {
  const int bytes = common_bytes(uint64_t(width * sizeof(T)) | uint64_t(stride * sizeof(T)) |
                                 uint64_t(table) | uint64_t(out));
  auto go = [&](auto run) {
    return run(n, width, table, stride, index, factor, mask, drop, out, stream);
  };
  if constexpr (sizeof(T) == 2) {
    if (bytes >= 16) return go(run_lookup<T, 8>);
    if (bytes >= 8) return go(run_lookup<T, 4>);
    if (bytes >= 4) return go(run_lookup<T, 2>);
  } else {
    if (bytes >= 16) return go(run_lookup<T, 4>);
    if (bytes >= 8) return go(run_lookup<T, 2>);
  }
  return go(run_lookup<T, 1>);
}

int refuse(const char* what, const char* why) {
  return fail(CLAD3DGS_INVALID_ARGUMENT, std::string(what) + ": " + why);
}

int status(const char* what, cudaError_t e) {
  return e == cudaSuccess
             ? CLAD3DGS_OK
             : fail(CLAD3DGS_CUDA_ERROR, std::string(what) + ": " + cudaGetErrorString(e));
}

constexpr int64_t kMostTokens = (int64_t(1) << 31) - 1;  // positions and rows are 32-bit

// The checks every entry shares; null if they pass.
const char* problem(int64_t n, int64_t rows, int64_t width, int type, double scale, double p) {
  if (n < 0 || rows < 0 || width < 0) return "negative size";
  if (n > kMostTokens || rows > kMostTokens) return "more than 2^31 - 1 tokens or rows";
  if (width > 0 && (n > (int64_t(1) << 60) / width || rows > (int64_t(1) << 60) / width))
    return "too many elements";
  if (type < CLAD3DGS_F32 || type > CLAD3DGS_BF16) return "unknown element type";
  if (!std::isfinite(scale)) return "scale must be finite";
  if (!(p >= 0.0 && p <= 1.0)) return "p must lie in [0, 1]";
  return nullptr;
}

float factor_of(double scale, double p) { return p < 1.0 ? float(scale / (1.0 - p)) : 0.f; }

template <class T>
Sums<T> sums_of(int64_t n, int64_t rows, int64_t width, const void* grad, int64_t stride,
                const uint32_t* order, double scale, double p, uint64_t seed, uint64_t offset,
                const int64_t* offset_device, void* workspace) {
  Sums<T> a;
  a.n = n;
  a.rows = rows;
  a.width = width;
  a.chunk = chunk_of(n);
  a.grad = static_cast<const T*>(grad);
  a.stride = stride;
  a.order = reinterpret_cast<const uint2*>(order);
  a.factor = factor_of(scale, p);
  a.mask = counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device));
  a.partial = static_cast<float*>(workspace);
  return a;
}

size_t partial_bytes(int64_t n, int64_t width) {
  return size_t(2 * chunks_of(n)) * width * sizeof(float);
}

const char* sums_problem(int64_t n, int64_t rows, int64_t width, const void* grad,
                         int64_t stride, const uint32_t* order, const void* workspace,
                         size_t bytes) {
  if (n > 0 && width > 0 && (!grad || !order || !workspace)) return "null array";
  if (stride < 0) return "bad row stride";
  if (n > 0 && bytes < partial_bytes(n, width)) return "workspace too small";
  if (uint64_t(workspace) % 16 || uint64_t(order) % 8) return "unaligned workspace or order";
  return nullptr;
}

}  // namespace
}  // namespace clad3dgs

using namespace clad3dgs;

extern "C" size_t clad3dgs_token_order_workspace(int64_t n, int64_t rows) {
  if (n <= 0 || rows < 0 || n > kMostTokens || rows > kMostTokens) return 0;
  return tokens::sort_plan(n, rows).bytes();
}

extern "C" int clad3dgs_token_order(int64_t n, int64_t rows, const void* index, int index_bits,
                                    int has_padding, int64_t padding, uint32_t* order,
                                    void* workspace, size_t workspace_bytes,
                                    cudaStream_t stream) {
  const char* what = "token order";
  if (const char* why = problem(n, rows, 0, CLAD3DGS_F32, 1.0, 0.0)) return refuse(what, why);
  if (index_bits != 32 && index_bits != 64) return refuse(what, "indices are 32 or 64 bits");
  if (n == 0) return CLAD3DGS_OK;
  if (!index || !order || !workspace) return refuse(what, "null array");
  if (uint64_t(workspace) % 256 || uint64_t(order) % 8)
    return refuse(what, "unaligned workspace or order");
  if (workspace_bytes < tokens::sort_plan(n, rows).bytes())
    return refuse(what, "workspace too small");
  const tokens::Index x{index, index_bits == 64, has_padding != 0, padding, rows};
  return status(what, tokens::sort_tokens(n, x, reinterpret_cast<uint2*>(order), workspace,
                                          stream));
}

extern "C" int clad3dgs_embedding_lookup(int type, int64_t n, int64_t rows, int64_t width,
                                         const void* table, int64_t table_stride,
                                         const void* index, int index_bits, int has_padding,
                                         int64_t padding, double scale, double p, uint64_t seed,
                                         uint64_t offset, const int64_t* offset_device,
                                         void* out, cudaStream_t stream) {
  const char* what = "embedding lookup";
  if (const char* why = problem(n, rows, width, type, scale, p)) return refuse(what, why);
  if (index_bits != 32 && index_bits != 64) return refuse(what, "indices are 32 or 64 bits");
  if (n == 0 || width == 0) return CLAD3DGS_OK;
  if ((!table && rows > 0) || !index || !out) return refuse(what, "null array");
  if (table_stride < 0) return refuse(what, "bad row stride");
  const tokens::Index x{index, index_bits == 64, has_padding != 0, padding, rows};
  const CounterMask mask =
      counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device));
  auto go = [&](auto pick) {
    return pick(n, width, table, table_stride, x, factor_of(scale, p), mask, p > 0.0, out,
                stream);
  };
  return status(what, type == CLAD3DGS_F32   ? go(pick_lookup<float>)
                      : type == CLAD3DGS_F16 ? go(pick_lookup<__half>)
                                             : go(pick_lookup<__nv_bfloat16>));
}

extern "C" size_t clad3dgs_embedding_workspace(int64_t n, int64_t width) {
  if (n <= 0 || width <= 0 || n > kMostTokens || n > (int64_t(1) << 60) / width) return 0;
  return partial_bytes(n, width);
}

extern "C" int clad3dgs_embedding_gradient(int type, int64_t n, int64_t rows, int64_t width,
                                           const void* grad, int64_t grad_stride,
                                           const uint32_t* order, double scale, double p,
                                           uint64_t seed, uint64_t offset,
                                           const int64_t* offset_device, void* out,
                                           void* workspace, size_t workspace_bytes,
                                           cudaStream_t stream) {
  const char* what = "embedding gradient";
  if (const char* why = problem(n, rows, width, type, scale, p)) return refuse(what, why);
  if (rows == 0 || width == 0) return CLAD3DGS_OK;
  if (const char* why = sums_problem(n, rows, width, grad, grad_stride, order, workspace,
                                     workspace_bytes))
    return refuse(what, why);
  if (!out) return refuse(what, "null array");
  auto go = [&](auto zero) {
    using T = decltype(zero);
    const int bytes = common_bytes(uint64_t(width * sizeof(T)) |
                                   uint64_t(grad_stride * sizeof(T)) | uint64_t(grad) |
                                   uint64_t(out));
    return pick_sums(sums_of<T>(n, rows, width, grad, grad_stride, order, scale, p, seed, offset,
                                offset_device, workspace),
                     Store<T>{static_cast<T*>(out)}, bytes, p > 0.0, stream);
  };
  return status(what, type == CLAD3DGS_F32   ? go(float())
                      : type == CLAD3DGS_F16 ? go(__half())
                                             : go(__nv_bfloat16()));
}

extern "C" int clad3dgs_embedding_consume_torch_adam(
    int type, int64_t n, int64_t rows, int64_t width, const void* grad, int64_t grad_stride,
    const uint32_t* order, double scale, double p, uint64_t seed, uint64_t offset,
    const int64_t* offset_device, float* table, float* first, float* second, double rate,
    TorchAdamConfig config, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const char* what = "embedding consume";
  if (const char* why = problem(n, rows, width, type, scale, p)) return refuse(what, why);
  if (!(std::isfinite(rate) && rate >= 0.0 && config.bias1 > 0.f && config.bias1 <= 1.f &&
        config.bias2_sqrt > 0.f && config.bias2_sqrt <= 1.f))
    return refuse(what, "invalid Adam configuration");
  if (rows == 0 || width == 0) return CLAD3DGS_OK;
  if (const char* why = sums_problem(n, rows, width, grad, grad_stride, order, workspace,
                                     workspace_bytes))
    return refuse(what, why);
  if (!table || !first || !second) return refuse(what, "null array");
  const Adam adam{table, first, second, float(rate / double(config.bias1)),
                  1.0 / double(config.bias2_sqrt)};
  auto go = [&](auto zero) {
    using T = decltype(zero);
    int bytes = common_bytes(uint64_t(width * sizeof(T)) | uint64_t(grad_stride * sizeof(T)) |
                             uint64_t(grad));
    // Vectors of V gradients meet V floats, moved 16 bytes at a time.
    const int floats =
        common_bytes(uint64_t(table) | uint64_t(first) | uint64_t(second));
    if (floats < 16) bytes = std::min(bytes, floats / 4 * int(sizeof(T)));
    return pick_sums(sums_of<T>(n, rows, width, grad, grad_stride, order, scale, p, seed, offset,
                                offset_device, workspace),
                     adam, bytes, p > 0.0, stream);
  };
  return status(what, type == CLAD3DGS_F32   ? go(float())
                      : type == CLAD3DGS_F16 ? go(__half())
                                             : go(__nv_bfloat16()));
}
