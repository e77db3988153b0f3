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
#include "row_sums.cuh"
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

// A lookup moves rows through registers: bound by writing the output, the index
// and the table's rows (small ones stay in L2) come on top. Groups of lanes take
// a row each, C vectors of 16 bytes a lane; a thread asks for the rows of U
// tokens before it stores the first, so that four to six loads are in flight.
template <class T, int V, int C, int U, bool kDrop>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(int64_t n, int64_t width, int lanes, int64_t slices,
                  const T* __restrict__ table, int64_t table_stride, Index index, float factor,
                  CounterMask mask, T* __restrict__ out) {
  const unsigned long long offset = kDrop ? mask_offset(mask) : 0;
  const int64_t block = blockIdx.x / slices;
  const int lane = threadIdx.x % lanes, groups = kThreads / lanes;
  const int apart = lanes * V;
  const int64_t column = (blockIdx.x - block * slices) * (apart * C) + lane * V;
  const int64_t first = block * (groups * U) + threadIdx.x / lanes;
  int64_t raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    raw[u] = first + u * groups < n ? tokens::raw_index(index, first + u * groups) : 0;
  Vec<T, V> v[U][C];
  uint32_t row[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    row[u] = first + u * groups < n ? tokens::row_of(index, raw[u]) : uint32_t(index.rows);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      v[u][c] = {};
      if (row[u] < index.rows && column + c * apart < width)
        v[u][c] = *reinterpret_cast<const Vec<T, V>*>(table + row[u] * table_stride + column +
                                                      c * apart);
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * groups;
    if (i >= n) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int64_t at = i * width + column + c * apart;
      if (column + c * apart >= width) break;
      bool keep[V];
      if (kDrop) mask_vector<V>(mask, offset, at, keep);
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[u][c].v[j] = from_float<T>(!kDrop || keep[j] ? to_float(v[u][c].v[j]) * factor : 0.f);
      if (row[u] >= index.rows) v[u][c] = {};
      *reinterpret_cast<Vec<T, V>*>(out + at) = v[u][c];
    }
  }
}

// Rows that do not start on 16 bytes: a thread fills V consecutive elements of
// the output, whatever rows they belong to, from single loads (adjacent
// threads read adjacent elements, which the L1 cache gathers).
template <class T, class Number, int V, bool kDrop>
__global__ void __launch_bounds__(kThreads)
    lookup_flat_kernel(Number total, Number width, const T* __restrict__ table,
                       int64_t table_stride, Index index, float factor, CounterMask mask,
                       T* __restrict__ out) {
  const unsigned long long offset = kDrop ? mask_offset(mask) : 0;
  const Number at = (Number(blockIdx.x) * kThreads + threadIdx.x) * V;
  if (at >= total) return;
  Number i = at / width, column = at - i * width;
  uint32_t row = tokens::row_of(index, tokens::raw_index(index, i));
  Vec<T, V> v{};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (at + j < total) {
      if (column == width) {
        column = 0;
        row = tokens::row_of(index, tokens::raw_index(index, ++i));
      }
      if (row < index.rows) v.v[j] = table[row * table_stride + column];
      ++column;
    }
  }
  bool keep[V];
  if (kDrop) mask_vector<V>(mask, offset, at, keep);
#pragma unroll
  for (int j = 0; j < V; ++j)
    v.v[j] = from_float<T>(!kDrop || keep[j] ? to_float(v.v[j]) * factor : 0.f);
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

template <class T, int V, int C, int U>
cudaError_t run_rows(const Lookup& a) {
  int64_t padded;
  const int lanes = sums::lanes_of(a.width / V, C, &padded);
  const int64_t slices = padded / (lanes * C), tokens = kThreads / lanes * U;
  const unsigned grid = unsigned((a.n + tokens - 1) / tokens * slices);
  auto* kernel = a.drop ? lookup_kernel<T, V, C, U, true> : lookup_kernel<T, V, C, U, false>;
  kernel<<<grid, kThreads, 0, a.stream>>>(a.n, a.width, lanes, slices,
                                          static_cast<const T*>(a.table), a.stride, a.index,
                                          a.factor, a.mask, static_cast<T*>(a.out));
  return cudaGetLastError();
}

template <class T, class Number, int V>
cudaError_t run_flat(const Lookup& a) {
  const int64_t total = a.n * a.width;
  const unsigned grid = unsigned((total + kThreads * V - 1) / (kThreads * V));
  auto* kernel =
      a.drop ? lookup_flat_kernel<T, Number, V, true> : lookup_flat_kernel<T, Number, V, false>;
  kernel<<<grid, kThreads, 0, a.stream>>>(Number(total), Number(a.width),
                                          static_cast<const T*>(a.table), a.stride, a.index,
                                          a.factor, a.mask, static_cast<T*>(a.out));
  return cudaGetLastError();
}

template <class T>
cudaError_t run_lookup(const Lookup& a) {
  constexpr int V = 16 / sizeof(T);
  const int bytes = common_bytes(uint64_t(a.width * sizeof(T)) | uint64_t(a.stride * sizeof(T)) |
                                 uint64_t(a.table) | uint64_t(a.out));
  if (bytes >= 16) {
    switch (sums::vectors_of_lane(a.n, a.width, V)) {
      case 4: return run_rows<T, V, 4, 1>(a);
      case 3: return run_rows<T, V, 3, 2>(a);
      default: return run_rows<T, V, 1, 4>(a);
    }
  }
  if (uint64_t(a.out) % 16) return run_flat<T, int64_t, 1>(a);
  // Divisions of 32-bit numbers while every element number fits one.
  return a.n * a.width < (int64_t(1) << 32) - kThreads * V ? run_flat<T, uint32_t, V>(a)
                                                           : run_flat<T, int64_t, V>(a);
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
sums::Args<T> sums_of(int64_t n, int64_t rows, int64_t width, const void* grad, int64_t stride,
                      const uint32_t* order, double scale, double p, uint64_t seed,
                      uint64_t offset, const int64_t* offset_device, void* workspace) {
  sums::Args<T> a{};
  a.n = n;
  a.rows = rows;
  a.width = width;
  a.grad = static_cast<const T*>(grad);
  a.stride = stride;
  a.order = reinterpret_cast<const uint2*>(order);
  a.factor = factor_of(scale, p);
  a.mask = counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device));
  a.partial = static_cast<float*>(workspace);
  return a;
}

const char* sums_problem(int64_t n, int64_t rows, int64_t width, const void* grad,
                         int64_t stride, const uint32_t* order, const void* workspace,
                         size_t bytes) {
  if (n > 0 && width > 0 && (!grad || !order || !workspace)) return "null array";
  if (stride < 0) return "bad row stride";
  if (n > 0 && bytes < sums::workspace_bytes(n, width)) return "workspace too small";
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
  const size_t need = tokens::sort_plan(n, rows).bytes();
  if (!index || !order || (need > 0 && !workspace)) return refuse(what, "null array");
  if (uint64_t(workspace) % 256 || uint64_t(order) % 8)
    return refuse(what, "unaligned workspace or order");
  if (workspace_bytes < need) return refuse(what, "workspace too small");
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
  const Lookup a{n, width, table, table_stride, x, factor_of(scale, p),
                 counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device)),
                 p > 0.0, out, stream};
  return status(what, type == CLAD3DGS_F32   ? run_lookup<float>(a)
                      : type == CLAD3DGS_F16 ? run_lookup<__half>(a)
                                             : run_lookup<__nv_bfloat16>(a));
}

extern "C" size_t clad3dgs_embedding_workspace(int64_t n, int64_t width) {
  if (n <= 0 || width <= 0 || n > kMostTokens || n > (int64_t(1) << 60) / width) return 0;
  return sums::workspace_bytes(n, width);
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
    const uint64_t row = uint64_t(width * sizeof(T));
    const int bytes =
        common_bytes(row | uint64_t(grad_stride * sizeof(T)) | uint64_t(grad));
    return sums::run<T, T>(sums_of<T>(n, rows, width, grad, grad_stride, order, scale, p, seed,
                                      offset, offset_device, workspace),
                           sums::Store<T>{static_cast<T*>(out)}, bytes,
                           common_bytes(row | uint64_t(out)), p > 0.0, stream);
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
  const sums::Adam adam{table, first, second, float(rate / double(config.bias1)),
                  1.0 / double(config.bias2_sqrt)};
  auto go = [&](auto zero) {
    using T = decltype(zero);
    const int bytes = common_bytes(uint64_t(width * sizeof(T)) |
                                   uint64_t(grad_stride * sizeof(T)) | uint64_t(grad));
    return sums::run<T, float>(sums_of<T>(n, rows, width, grad, grad_stride, order, scale, p,
                                          seed, offset, offset_device, workspace),
                               adam, bytes,
                               common_bytes(uint64_t(width * sizeof(float)) | uint64_t(table) |
                                            uint64_t(first) | uint64_t(second)),
                               p > 0.0, stream);
  };
  return status(what, type == CLAD3DGS_F32   ? go(float())
                      : type == CLAD3DGS_F16 ? go(__half())
                                             : go(__nv_bfloat16()));
}
