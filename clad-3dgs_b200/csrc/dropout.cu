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

namespace clad3dgs {
int fail(int code, const std::string& message);  // gaussian_step.cu

namespace {

constexpr int kThreads = 256;

template <class T, bool kRows>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(int64_t n, int64_t width, const T* x, int64_t x_stride, T* y,
                   int64_t y_stride, float factor, CounterMask mask) {
  const unsigned long long offset = mask_offset(mask);
  const int64_t blocks = (n + 3) / 4;
  for (int64_t b = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; b < blocks;
       b += (int64_t)gridDim.x * blockDim.x) {
    uint4 words = make_uint4(0, 0, 0, 0);
    if (!kRows) words = mask_words(mask, offset, b);
    int64_t row = 4 * b / width, column = 4 * b - row * width;
    const int count = int(n - 4 * b < 4 ? n - 4 * b : 4);
    for (int j = 0; j < count; ++j) {
      const uint32_t word =
          kRows ? word_of(mask_words(mask, offset, row / 4), row % 4) : word_of(words, j);
      const float v = to_float(x[row * x_stride + column]) * factor;
      y[row * y_stride + column] = from_float<T>(mask.keeps(word) ? v : 0.f);
      if (++column == width) column = 0, ++row;
    }
  }
}

template <class T>
cudaError_t launch(int64_t rows, int64_t width, const void* x, int64_t x_stride, void* y,
                   int64_t y_stride, double p, uint64_t seed, uint64_t offset,
                   const int64_t* offset_device, bool by_row, cudaStream_t stream) {
  const int64_t n = rows * width;
  const CounterMask mask =
      counter_mask(p, seed, offset, reinterpret_cast<const long long*>(offset_device));
  const float factor = float(1.0 / (1.0 - p));
  const unsigned grid =
      unsigned(std::min<int64_t>((n / 4 + kThreads) / kThreads, int64_t(1) << 20));
  auto* kernel = by_row ? dropout_kernel<T, true> : dropout_kernel<T, false>;
  kernel<<<grid, kThreads, 0, stream>>>(n, width, static_cast<const T*>(x), x_stride,
                                        static_cast<T*>(y), y_stride, factor, mask);
  return cudaGetLastError();
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
  cudaError_t e;
  switch (type) {
    case CLAD3DGS_F32:
      e = launch<float>(rows, width, x, x_stride, y, y_stride, p, seed, offset, offset_device,
                        by_row != 0, stream);
      break;
    case CLAD3DGS_F16:
      e = launch<__half>(rows, width, x, x_stride, y, y_stride, p, seed, offset, offset_device,
                         by_row != 0, stream);
      break;
    default:
      e = launch<__nv_bfloat16>(rows, width, x, x_stride, y, y_stride, p, seed, offset,
                                offset_device, by_row != 0, stream);
  }
  return e == cudaSuccess
             ? CLAD3DGS_OK
             : fail(CLAD3DGS_CUDA_ERROR, std::string("dropout: ") + cudaGetErrorString(e));
}
