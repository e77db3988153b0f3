// Element types of the table operators and the dropout: conversions to and
// from the 32-bit floats that every kernel computes in, and vectors of
// consecutive elements moved as one load or store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

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

// A vector to floats and back, two 16-bit elements an instruction.
template <class T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& from, float (&to)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) to[j] = to_float(from.v[j]);
}

template <class T, int V>
__device__ __forceinline__ Vec<T, V> pack(const float (&from)[V]) {
  Vec<T, V> to;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2*>(&to.v[j]) = __floats2half2_rn(from[j], from[j + 1]);
      else
        *reinterpret_cast<__nv_bfloat162*>(&to.v[j]) =
            __floats2bfloat162_rn(from[j], from[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) to.v[j] = from_float<T>(from[j]);
  }
  return to;
}

// Largest power of two (16 at most) that divides the value (of several: their
// bitwise or).
inline int common_bytes(uint64_t a) {
  int b = 16;
  while (b > 1 && a % b) b /= 2;
  return b;
}

// Quotient and remainder by a number that the host knows (Granlund and
// Montgomery, "Division by invariant integers using multiplication", PLDI'94):
// a high product, a sum and a shift for dividends below 2^31 (Narrow), the
// division itself for larger ones (Wide).
struct Narrow {
  using Number = uint32_t;
  uint32_t divisor, factor, shift;

  explicit Narrow(int64_t d) : divisor(uint32_t(d)), shift(0) {
    while ((uint64_t(1) << shift) < uint64_t(d)) ++shift;
    factor = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - uint64_t(d))) / uint64_t(d) + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return (__umulhi(n, factor) + n) >> shift;
  }
  static bool fits(int64_t most) { return most < (int64_t(1) << 31); }
};

struct Wide {
  using Number = int64_t;
  int64_t divisor;

  explicit Wide(int64_t d) : divisor(d) {}
  __device__ __forceinline__ int64_t quotient(int64_t n) const { return n / divisor; }
};

}  // namespace clad3dgs
