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

// How a row is cut: vectors of V elements, `lanes` of them side by side in one
// group (a power of two, 32 at most), `slices` groups a row.
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
      if (kDrop) mask_vector<V>(mask, offset, i * width + column, keep);
#pragma unroll
      for (int j = 0; j < V; ++j)
        v.v[j] = from_float<T>(!kDrop || keep[j] ? to_float(v.v[j]) * factor : 0.f);
    }
    *reinterpret_cast<Vec<T, V>*>(out + i * width + column) = v;
  }
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
