// Dropout from a counter-based generator, with a mask that is never stored.
//
//   y[e] = keep(e) ? x[e] / (1 - p) : 0      (rows form: keep(e / width))
//
// The map is linear and its own adjoint, so the backward pass is the same
// kernel on the gradient with the same seed and offset. A dropped element
// gives +0 whatever it held (infinities and NaN too). Arithmetic in 32 bits,
// one rounding to the element type.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "clad3dgs_b200.h"
#include "counter_mask.cuh"
#include "element_types.cuh"
#include "launch.cuh"

namespace clad3dgs {
int fail(int code, const std::string& message);  // gaussian_step.cu

namespace {

constexpr int kThreads = 256;

// Bound by moving the elements once each way, and nearly as much by the
// generator: twenty products of 32 x 32 bits for four elements, at a quarter of
// the rate of other instructions. Every access is a vector of 16 bytes.

// x with the dropped elements at zero and the others times the factor.
template <class T, int V>
__device__ __forceinline__ Vec<T, V> drop(const Vec<T, V>& x, const bool (&keep)[V],
                                          float factor) {
  float f[V];
  unpack<T, V>(x, f);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = keep[j] ? f[j] * factor : 0.f;
  return pack<T, V>(f);
}

// Packed rows: element numbers are addresses. Blocks stay and take a vector a
// round: the first two rounds' products that hang on the offset alone are made
// once, and with 64 warps an SM the next vectors arrive while these are drawn
// for (16384 x 4096 bf16: 61 us, 66 with eight blocks of 256 threads, 72 to 80
// with a block for every one, two or four vectors a thread; the words alone
// take 37 us, the copy alone 42).
constexpr int kStayThreads = 1024, kStayBlocks = 2;

template <class T, class Number, int V>
__global__ void __launch_bounds__(kStayThreads, kStayBlocks)
    packed_kernel(int64_t vectors, int rest, const T* x, T* y, float factor,
                  const __grid_constant__ CounterMask mask) {
  wait_before();
  const unsigned long long offset = mask_offset(mask);
  const int64_t first = int64_t(blockIdx.x) * kStayThreads + threadIdx.x;
  for (int64_t i = first; i < vectors; i += int64_t(gridDim.x) * kStayThreads) {
    const Vec<T, V> v = reinterpret_cast<const Vec<T, V>*>(x)[i];
    bool keep[V];
    mask_vector<V, Number>(mask, offset, i * V, keep);
    reinterpret_cast<Vec<T, V>*>(y)[i] = drop<T, V>(v, keep, factor);
  }
  if (first < rest) {  // elements behind the last vector
    const int64_t at = vectors * V + first;
    const uint4 words = mask_words(mask, offset, Number(at / 4));
    const bool keep[1] = {mask.keeps(word_of(words, unsigned(at % 4)))};
    reinterpret_cast<Vec<T, 1>*>(y)[at] =
        drop<T, 1>(reinterpret_cast<const Vec<T, 1>*>(x)[at], keep, factor);
  }
}

// Rows of whole vectors, with any stride that keeps them aligned; `vectors` a
// row. kRows: one decision for each row.
template <class T, class Division, int V, int U, bool kRows>
__global__ void __launch_bounds__(kThreads)
    aligned_rows_kernel(typename Division::Number total, const Division vectors, const T* x,
                        int64_t x_stride, T* y, int64_t y_stride, float factor,
                        const __grid_constant__ CounterMask mask) {
  using Number = typename Division::Number;
  wait_before();
  const unsigned long long offset = mask_offset(mask);
  const Number first = Number(blockIdx.x) * (U * kThreads) + threadIdx.x;
  Vec<T, V> v[U];
  Number row[U], column[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Number at = first + u * kThreads;
    row[u] = vectors.quotient(at);
    column[u] = (at - row[u] * vectors.divisor) * V;
    if (at < total) v[u] = *reinterpret_cast<const Vec<T, V>*>(x + row[u] * x_stride + column[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (first + u * kThreads >= total) return;
    bool keep[V];
    if constexpr (kRows) {
      const bool kept =
          mask.keeps(word_of(mask_words(mask, offset, row[u] / 4), unsigned(row[u] % 4)));
#pragma unroll
      for (int j = 0; j < V; ++j) keep[j] = kept;
    } else {
      mask_vector<V>(mask, offset, uint64_t(first + u * kThreads) * V, keep);
    }
    v[u] = drop<T, V>(v[u], keep, factor);
    *reinterpret_cast<Vec<T, V>*>(y + row[u] * y_stride + column[u]) = v[u];
  }
}

// Any rows: V consecutive elements a thread, loaded one by one (neighbours hit
// the same lines) and stored as a vector where the output is packed and
// aligned (kPacked).
template <class T, class Division, int V, bool kRows, bool kPacked>
__global__ void __launch_bounds__(kThreads)
    any_rows_kernel(typename Division::Number total, const Division width, const T* x,
                    int64_t x_stride, T* y, int64_t y_stride, float factor,
                    const __grid_constant__ CounterMask mask) {
  using Number = typename Division::Number;
  wait_before();
  const unsigned long long offset = mask_offset(mask);
  const Number at = (Number(blockIdx.x) * kThreads + threadIdx.x) * V;
  if (at >= total) return;
  const Number row = width.quotient(at), column = at - row * width.divisor;
  Vec<T, V> v;
  {
    Number r = row, c = column;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (c == width.divisor) c = 0, ++r;
      if (at + j < total) v.v[j] = x[r * x_stride + c];
      ++c;
    }
  }
  bool keep[V];
  if constexpr (kRows) {
    Number r = row, c = column;
    uint4 words = mask_words(mask, offset, r / 4);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (c == width.divisor) {
        c = 0;
        if (++r % 4 == 0) words = mask_words(mask, offset, r / 4);
      }
      keep[j] = mask.keeps(word_of(words, unsigned(r % 4)));
      ++c;
    }
  } else {
    mask_vector<V, Number>(mask, offset, at, keep);
  }
  v = drop<T, V>(v, keep, factor);
  if (kPacked && at + V <= total) {
    *reinterpret_cast<Vec<T, V>*>(y + at) = v;
    return;
  }
  Number r = row, c = column;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (c == width.divisor) c = 0, ++r;
    if (at + j < total) y[r * y_stride + c] = v.v[j];
    ++c;
  }
}

struct Call {
  int64_t rows, width;
  const void* x;
  int64_t x_stride;
  void* y;
  int64_t y_stride;
  float factor;
  CounterMask mask;
  bool by_row;
  cudaStream_t stream;
};

unsigned grid_of(int64_t work, int64_t each) { return unsigned((work + each - 1) / each); }

template <class T, class Division>
cudaError_t launch_rows(const Call& a, bool aligned) {
  using Number = typename Division::Number;
  constexpr int V = 16 / sizeof(T), U = 2;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  if (aligned) {
    const int64_t vectors = a.width / V, total = a.rows * vectors;
    auto* kernel = a.by_row ? aligned_rows_kernel<T, Division, V, U, true>
                            : aligned_rows_kernel<T, Division, V, U, false>;
    return launch_after(kernel, grid_of(total, U * kThreads), kThreads, 0, a.stream,
        Number(total), Division(vectors), x, a.x_stride, y, a.y_stride, a.factor, a.mask);
  }
  const int64_t total = a.rows * a.width;
  const bool packed = (a.y_stride == a.width || a.rows == 1) && uint64_t(y) % 16 == 0;
  auto* kernel = packed ? (a.by_row ? any_rows_kernel<T, Division, V, true, true>
                                    : any_rows_kernel<T, Division, V, false, true>)
                        : (a.by_row ? any_rows_kernel<T, Division, V, true, false>
                                    : any_rows_kernel<T, Division, V, false, false>);
  return launch_after(kernel, grid_of(total, V * kThreads), kThreads, 0, a.stream,
        Number(total), Division(a.width), x, a.x_stride, y, a.y_stride, a.factor, a.mask);
}

template <class T>
cudaError_t launch(const Call& a) {
  constexpr int V = 16 / sizeof(T);
  const int64_t n = a.rows * a.width;
  const bool packed = a.rows == 1 || (a.x_stride == a.width && a.y_stride == a.width);
  const bool based = (uint64_t(a.x) | uint64_t(a.y)) % 16 == 0;
  // Rows of one element are decided one by one either way.
  if (packed && based && (!a.by_row || a.width == 1)) {
    auto* kernel =
        n < (int64_t(1) << 34) ? packed_kernel<T, uint32_t, V> : packed_kernel<T, uint64_t, V>;
    const unsigned blocks = std::max(1u, grid_of(n / V, kStayThreads));
    return launch_after(kernel, std::min(blocks, 148u * kStayBlocks), kStayThreads, 0, a.stream,
                        n / V, int(n % V), static_cast<const T*>(a.x), static_cast<T*>(a.y),
                        a.factor, a.mask);
  }
  const bool aligned =
      based && a.width % V == 0 && (a.rows == 1 || (a.x_stride % V == 0 && a.y_stride % V == 0));
  return Narrow::fits(n + 2 * V * kThreads) ? launch_rows<T, Narrow>(a, aligned)
                                            : launch_rows<T, Wide>(a, aligned);
}

}  // namespace
}  // namespace clad3dgs

using namespace clad3dgs;

extern "C" int clad3dgs_dropout(int type, int64_t rows, int64_t width, const void* x,
                                int64_t x_stride, void* y, int64_t y_stride, double p,
                                uint64_t seed, uint64_t offset, const int64_t* offset_device,
                                int by_row, cudaStream_t stream) {
  if (rows < 0 || width < 0) return fail(CLAD3DGS_INVALID_ARGUMENT, "dropout: negative size");
  if (!(p >= 0.0 && p <= 1.0))
    return fail(CLAD3DGS_INVALID_ARGUMENT, "dropout: p must lie in [0, 1]");
  if (type < CLAD3DGS_F32 || type > CLAD3DGS_BF16)
    return fail(CLAD3DGS_INVALID_ARGUMENT, "dropout: unknown element type");
  if (rows == 0 || width == 0) return CLAD3DGS_OK;
  if (rows > (int64_t(1) << 62) / width)
    return fail(CLAD3DGS_INVALID_ARGUMENT, "dropout: too many elements");
  if (!x || !y) return fail(CLAD3DGS_INVALID_ARGUMENT, "dropout: null array");
  if (x_stride < 0 || (rows > 1 && y_stride < width))
    return fail(CLAD3DGS_INVALID_ARGUMENT, "dropout: bad row stride");
  const Call a{rows, width, x, x_stride, y, y_stride,
               p < 1.0 ? float(1.0 / (1.0 - p)) : 0.f,
               counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device)),
               by_row != 0, stream};
  const cudaError_t e = type == CLAD3DGS_F32   ? launch<float>(a)
                        : type == CLAD3DGS_F16 ? launch<__half>(a)
                                               : launch<__nv_bfloat16>(a);
  return e == cudaSuccess
             ? CLAD3DGS_OK
             : fail(CLAD3DGS_CUDA_ERROR, std::string("dropout: ") + cudaGetErrorString(e));
}
