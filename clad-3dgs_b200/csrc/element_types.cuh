// Element types of the table operators and the dropout: conversions to and
// from the 32-bit floats that every kernel computes in, and vectors of
// consecutive elements moved as one load or store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace clad3dgs {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V consecutive elements; 16 bytes at most.
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// Largest power of two (16 at most) that divides every value given.
inline int common_bytes(uint64_t a) {
  int b = 16;
  while (b > 1 && a % b) b /= 2;
  return b;
}

}  // namespace clad3dgs
