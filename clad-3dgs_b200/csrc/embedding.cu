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
// The gradient goes by sorted tokens (token_order.cuh), its sums and what
// becomes of them are in row_sums.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "clad3dgs_b200.h"
#include "counter_mask.cuh"
#include "element_types.cuh"
#include "launch.cuh"
#include "row_sums.cuh"
#include "token_order.cuh"

namespace clad3dgs {
// gaussian_step.cu
int fail(int code, const std::string& message);
cudaError_t fault_word(unsigned** word);

namespace sums {
CLAD3DGS_ROW_SUMS(extern, float)           // row_sums_f32.cu
CLAD3DGS_ROW_SUMS(extern, __half)          // row_sums_f16.cu
CLAD3DGS_ROW_SUMS(extern, __nv_bfloat16)   // row_sums_bf16.cu
}  // namespace sums

namespace {

using tokens::Index;

constexpr int kThreads = 256;

// The output's elements: table elements times the factor, dropped ones at zero.
template <class T, int V, bool kDrop>
__device__ __forceinline__ Vec<T, V> finish(const Vec<T, V>& x, const bool (&keep)[V],
                                            float factor) {
  float f[V];
  unpack<T, V>(x, f);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = !kDrop || keep[j] ? f[j] * factor : 0.f;
  return pack<T, V>(f);
}

// A lookup is bound by writing its output (the index and the table's rows come on
// top; small tables stay in L2). Threads take consecutive vectors of 16 bytes of
// the output, whatever rows they belong to, so that stores are whole lines, U of
// them each, all asked for before the first is stored. 1.1M rows of 48 floats
// from 4096: 39 us (5.5 TB/s; groups of lanes a row 50, one vector a thread
// 147); 16384 of 2048 bf16 from 131072, of which they name 6900: 20 us (4.8 TB/s).
template <class T, class Division, int V, int U, bool kDrop>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(typename Division::Number total, const Division vectors,
                  const T* table, int64_t table_stride, Index index, float factor,
                  const __grid_constant__ CounterMask mask, T* __restrict__ out) {
  using Number = typename Division::Number;
  wait_before();
  const unsigned long long offset = kDrop ? mask_offset(mask) : 0;
  const Number first = Number(blockIdx.x) * (U * kThreads) + threadIdx.x;
  int64_t raw[U];
  Number column[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Number at = first + u * kThreads;
    const Number i = vectors.quotient(at);
    column[u] = (at - i * vectors.divisor) * V;
    raw[u] = at < total ? tokens::raw_index(index, i) : 0;
  }
  Vec<T, V> v[U];
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    v[u] = {};
    if (first + u * kThreads < total) {
      const uint32_t row = tokens::row_of(index, raw[u], &bad);
      if (row < index.rows)
        v[u] = *reinterpret_cast<const Vec<T, V>*>(table + row * table_stride + column[u]);
    }
  }
  tokens::report(index, bad);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Number at = first + u * kThreads;
    if (at >= total) return;
    bool keep[V];
    if (kDrop) mask_vector<V, Number>(mask, offset, uint64_t(at) * V, keep);
    *reinterpret_cast<Vec<T, V>*>(out + int64_t(at) * V) =
        finish<T, V, kDrop>(v[u], keep, factor);
  }
}

// Rows that do not start on 16 bytes: V consecutive elements of the output a
// thread from single loads (neighbours hit the same lines); bound by their
// instructions (100003 x 77 f16 with dropout: 14 us, the call's launch included,
// against 98 with one element a thread). A vector touches
// two rows at most, or any number of rows shorter than itself (kShort).
template <class T, class Division, int V, bool kShort, bool kDrop>
__global__ void __launch_bounds__(kThreads)
    lookup_odd_kernel(typename Division::Number total, const Division width,
                      const T* table, int64_t table_stride, Index index,
                      float factor, const __grid_constant__ CounterMask mask,
                      T* __restrict__ out) {
  using Number = typename Division::Number;
  wait_before();
  const unsigned long long offset = kDrop ? mask_offset(mask) : 0;
  const Number at = (Number(blockIdx.x) * kThreads + threadIdx.x) * V;
  if (at >= total) return;
  Number i = width.quotient(at), column = at - i * width.divisor;
  Vec<T, V> v{};
  bool bad = false;
  uint32_t row = tokens::row_of(index, tokens::raw_index(index, i), &bad);
  if constexpr (kShort) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (at + j < total) {
        if (column == width.divisor) {
          column = 0;
          row = tokens::row_of(index, tokens::raw_index(index, ++i), &bad);
        }
        if (row < index.rows) v.v[j] = table[row * table_stride + column];
        ++column;
      }
    }
  } else {
    // Elements before `border` from this row, the others from the next.
    const int border = width.divisor - column < V ? int(width.divisor - column) : V;
    const int count = total - at < V ? int(total - at) : V;
    uint32_t next = uint32_t(index.rows);
    if (border < count) next = tokens::row_of(index, tokens::raw_index(index, i + 1), &bad);
    const T* here = table + row * table_stride + column;
    const T* there = table + next * table_stride - border;
    const int until = row < index.rows ? (border < count ? border : count) : 0;
    const int from = next < index.rows ? border : V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j < until) v.v[j] = here[j];
      else if (j >= from && j < count) v.v[j] = there[j];
    }
  }
  tokens::report(index, bad);
  bool keep[V];
  if (kDrop) mask_vector<V, Number>(mask, offset, uint64_t(at), keep);
  v = finish<T, V, kDrop>(v, keep, factor);
  if (at + V <= total) {
    *reinterpret_cast<Vec<T, V>*>(out + at) = v;
  } else {
    for (int j = 0; j < V; ++j)
      if (at + j < total) out[at + j] = v.v[j];
  }
}

struct Lookup {
  int64_t n, width;
  const void* table;
  int64_t stride;
  Index index;
  float factor;
  CounterMask mask;
  bool drop;
  void* out;
  cudaStream_t stream;
};

unsigned grid_of(int64_t work, int64_t each) { return unsigned((work + each - 1) / each); }

template <class T, class Division>
cudaError_t run_lookup(const Lookup& a, bool aligned) {
  using Number = typename Division::Number;
  constexpr int V = 16 / sizeof(T);
  const T* table = static_cast<const T*>(a.table);
  T* out = static_cast<T*>(a.out);
  if (aligned) {
    // Two vectors a thread where a warp's belong to one row, whose index is
    // read once (16384 x 2048 bf16: 19.7 us, 22.7 with four), else four, to have
    // more of the indices on their way (1.1M x 48 f32: 39 us, 46 with two).
    const int64_t vectors = a.width / V, total = a.n * vectors;
    const bool wide = vectors >= 32;
    auto* kernel = wide ? (a.drop ? lookup_kernel<T, Division, V, 2, true>
                                  : lookup_kernel<T, Division, V, 2, false>)
                        : (a.drop ? lookup_kernel<T, Division, V, 4, true>
                                  : lookup_kernel<T, Division, V, 4, false>);
    return launch_after(kernel, grid_of(total, (wide ? 2 : 4) * kThreads), kThreads, 0, a.stream,
        Number(total), Division(vectors), table, a.stride, a.index, a.factor, a.mask, out);
  }
  const int64_t total = a.n * a.width;
  auto go = [&](auto* kernel, int each) {
    return launch_after(kernel, grid_of(total, int64_t(each) * kThreads), kThreads, 0, a.stream,
        Number(total), Division(a.width), table, a.stride, a.index, a.factor, a.mask, out);
  };
  if (uint64_t(out) % 16)
    return a.drop ? go(lookup_odd_kernel<T, Division, 1, true, true>, 1)
                  : go(lookup_odd_kernel<T, Division, 1, true, false>, 1);
  if (a.width < V)
    return a.drop ? go(lookup_odd_kernel<T, Division, V, true, true>, V)
                  : go(lookup_odd_kernel<T, Division, V, true, false>, V);
  return a.drop ? go(lookup_odd_kernel<T, Division, V, false, true>, V)
                : go(lookup_odd_kernel<T, Division, V, false, false>, V);
}

template <class T>
cudaError_t pick_lookup(const Lookup& a) {
  const bool aligned =
      common_bytes(uint64_t(a.width * sizeof(T)) | uint64_t(a.stride * sizeof(T)) |
                   uint64_t(a.table) | uint64_t(a.out)) == 16;
  return Narrow::fits(a.n * a.width + 16 * kThreads) ? run_lookup<T, Narrow>(a, aligned)
                                                     : run_lookup<T, Wide>(a, aligned);
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

float factor_of(double scale, double p) { return p < 1.0 ? float(scale / (1.0 - p)) : 0.f; }

// The checks every entry shares; null if they pass.
const char* problem(int64_t n, int64_t rows, int64_t width, int type, double scale, double p) {
  if (n < 0 || rows < 0 || width < 0) return "negative size";
  if (n > kMostTokens || rows > kMostTokens) return "more than 2^31 - 1 tokens or rows";
  if (width > 0 && (n > (int64_t(1) << 60) / width || rows > (int64_t(1) << 60) / width))
    return "too many elements";
  if (type < CLAD3DGS_F32 || type > CLAD3DGS_BF16) return "unknown element type";
  if (!(p >= 0.0 && p <= 1.0)) return "p must lie in [0, 1]";
  if (!std::isfinite(scale) || !std::isfinite(factor_of(scale, p)))
    return "scale / (1 - p) must be finite in 32 bits";
  return nullptr;
}

size_t round_up(size_t bytes) { return (bytes + 255) / 256 * 256; }

// What the gradient and Adam entries share: the tokens, checked, and sorted into
// the front of the workspace unless their order is given.
struct Tokens {
  int64_t n, rows, width;
  Index index;
  int index_bits;
  const uint32_t* order;
  char* workspace;
  size_t bytes;

  bool sorts() const { return !order && n > 0 && !sums::few(n, rows, width); }
  size_t order_bytes() const {
    return sorts() ? round_up(size_t(n) * sizeof(uint2)) +
                         round_up(tokens::sort_plan(n, rows).bytes())
                   : 0;
  }
  size_t need(bool consume) const {
    return order_bytes() + sums::workspace_bytes(n, rows, width, consume);
  }
  const char* problem(const void* grad, int64_t stride, bool consume) const {
    if (n > 0 && !grad) return "null array";
    if (stride < 0) return "bad row stride";
    if (n > 0 && !order) {
      if (!index.data) return "null array";
      if (index_bits != 32 && index_bits != 64) return "indices are 32 or 64 bits";
    }
    if (need(consume) > 0 && !workspace) return "null array";
    if (bytes < need(consume)) return "workspace too small";
    if (uint64_t(workspace) % 256 || uint64_t(order) % 8) return "unaligned workspace or order";
    return nullptr;
  }
  float* partial() const { return reinterpret_cast<float*>(workspace + order_bytes()); }
  // The arguments of the sums; sorts first where it has to.
  template <class T>
  cudaError_t prepare(sums::Args<T>* a, const void* grad, int64_t stride,
                      const CounterMask& mask, float factor, const tokens::Fill& fill,
                      cudaStream_t stream) const {
    a->n = n;
    a->rows = rows;
    a->width = width;
    a->grad = static_cast<const T*>(grad);
    a->stride = stride;
    a->order = reinterpret_cast<const uint2*>(order);
    a->factor = factor;
    a->mask = mask;
    a->partial = partial();
    if (!sorts()) return cudaSuccess;
    uint2* sorted = reinterpret_cast<uint2*>(workspace);
    a->order = sorted;
    return tokens::sort_tokens(n, index, sorted, workspace + round_up(size_t(n) * sizeof(uint2)),
                               fill, stream);
  }
};

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
  const size_t need = tokens::sort_plan(n, rows).bytes();
  if (!index || !order || (need > 0 && !workspace)) return refuse(what, "null array");
  if (uint64_t(workspace) % 256 || uint64_t(order) % 8)
    return refuse(what, "unaligned workspace or order");
  if (workspace_bytes < need) return refuse(what, "workspace too small");
  tokens::Index x{index, index_bits == 64, has_padding != 0, padding, rows};
  if (const cudaError_t e = fault_word(&x.fault); e != cudaSuccess) return status(what, e);
  return status(what, tokens::sort_tokens(n, x, reinterpret_cast<uint2*>(order), workspace,
                                          tokens::Fill{}, stream));
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
  tokens::Index x{index, index_bits == 64, has_padding != 0, padding, rows};
  if (const cudaError_t e = fault_word(&x.fault); e != cudaSuccess) return status(what, e);
  const Lookup a{n, width, table, table_stride, x, factor_of(scale, p),
                 counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device)),
                 p > 0.0, out, stream};
  return status(what, type == CLAD3DGS_F32   ? pick_lookup<float>(a)
                      : type == CLAD3DGS_F16 ? pick_lookup<__half>(a)
                                             : pick_lookup<__nv_bfloat16>(a));
}

extern "C" size_t clad3dgs_embedding_workspace(int64_t n, int64_t rows, int64_t width,
                                               int consume, int ordered) {
  if (n <= 0 || problem(n, rows, width, CLAD3DGS_F32, 1.0, 0.0)) return 0;
  const uint32_t given = 0;
  const Tokens tokens{n, rows, width, Index{}, 64, ordered ? &given : nullptr, nullptr, 0};
  return tokens.need(consume != 0);
}

extern "C" int clad3dgs_embedding_gradient(int type, int64_t n, int64_t rows, int64_t width,
                                           const void* grad, int64_t grad_stride,
                                           const void* index, int index_bits, int has_padding,
                                           int64_t padding, const uint32_t* order, double scale,
                                           double p, uint64_t seed, uint64_t offset,
                                           const int64_t* offset_device, void* out,
                                           void* workspace, size_t workspace_bytes,
                                           cudaStream_t stream) {
  const char* what = "embedding gradient";
  if (const char* why = problem(n, rows, width, type, scale, p)) return refuse(what, why);
  if (rows == 0 || width == 0) return CLAD3DGS_OK;
  Tokens tokens{n, rows, width, Index{index, index_bits == 64, has_padding != 0, padding, rows},
                      index_bits, order, static_cast<char*>(workspace), workspace_bytes};
  if (const char* why = tokens.problem(grad, grad_stride, false)) return refuse(what, why);
  if (!out) return refuse(what, "null array");
  if (const cudaError_t e = fault_word(&tokens.index.fault); e != cudaSuccess)
    return status(what, e);
  const CounterMask mask =
      counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device));
  auto go = [&](auto zero) {
    using T = decltype(zero);
    sums::Args<T> a{};
    const cudaError_t e =
        tokens.prepare(&a, grad, grad_stride, mask, factor_of(scale, p), tokens::Fill{}, stream);
    return e == cudaSuccess ? sums::gradient(a, tokens.index, static_cast<T*>(out), p > 0.0, stream) : e;
  };
  return status(what, type == CLAD3DGS_F32   ? go(float())
                      : type == CLAD3DGS_F16 ? go(__half())
                                             : go(__nv_bfloat16()));
}

extern "C" int clad3dgs_embedding_consume_torch_adam(
    int type, int64_t n, int64_t rows, int64_t width, const void* grad, int64_t grad_stride,
    const void* index, int index_bits, int has_padding, int64_t padding, const uint32_t* order,
    double scale, double p, uint64_t seed, uint64_t offset, const int64_t* offset_device,
    float* table, float* first, float* second, double rate, TorchAdamConfig config,
    void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const char* what = "embedding consume";
  if (const char* why = problem(n, rows, width, type, scale, p)) return refuse(what, why);
  if (!(std::isfinite(rate) && rate >= 0.0 && config.bias1 > 0.f && config.bias1 <= 1.f &&
        config.bias2_sqrt > 0.f && config.bias2_sqrt <= 1.f))
    return refuse(what, "invalid Adam configuration");
  if (rows == 0 || width == 0) return CLAD3DGS_OK;
  Tokens tokens{n, rows, width, Index{index, index_bits == 64, has_padding != 0, padding, rows},
                      index_bits, order, static_cast<char*>(workspace), workspace_bytes};
  if (const char* why = tokens.problem(grad, grad_stride, true)) return refuse(what, why);
  if (!table || !first || !second) return refuse(what, "null array");
  if (const cudaError_t e = fault_word(&tokens.index.fault); e != cudaSuccess)
    return status(what, e);
  const sums::Adam adam{table, first, second, float(rate / double(config.bias1)),
                        1.0 / double(config.bias2_sqrt)};
  const CounterMask mask =
      counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device));
  auto go = [&](auto zero) {
    using T = decltype(zero);
    sums::Args<T> a{};
    cudaError_t e = cudaSuccess;
    tokens::Fill fill;
    if (n > 0 && !sums::few(n, rows, width)) {
      // The slots are cleared by the sort, if there is one and they are few.
      const sums::Kept kept(tokens.partial(), n, rows, width);
      if (tokens.sorts() && tokens::sort_clears(n, rows, rows))
        fill = {reinterpret_cast<uint4*>(kept.slots),
                int64_t(sums::slot_bytes(rows) / sizeof(uint4))};
      else
        e = kept.clear(rows, stream);
    }
    if (e == cudaSuccess)
      e = tokens.prepare(&a, grad, grad_stride, mask, factor_of(scale, p), fill, stream);
    return e == cudaSuccess ? sums::consume(a, tokens.index, adam, p > 0.0, stream) : e;
  };
  return status(what, type == CLAD3DGS_F32   ? go(float())
                      : type == CLAD3DGS_F16 ? go(__half())
                                             : go(__nv_bfloat16()));
}
