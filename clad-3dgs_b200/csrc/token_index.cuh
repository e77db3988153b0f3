// The indices by which tokens name the rows of a table.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace clad3dgs {
namespace tokens {

// Set when a kernel met an index outside its table that is not the padding: a
// word in every file that includes this, read by take_token_fault.
constexpr unsigned kFaultTokenRange = 256u;
static __device__ unsigned int g_token_fault = 0;

// The indices a caller gives.
struct Index {
  const void* data;
  bool wide;  // int64, else int32
  bool has_padding;
  int64_t padding;
  int64_t rows;
};

__device__ __forceinline__ int64_t raw_index(const Index& x, int64_t i) {
  return x.wide ? static_cast<const int64_t*>(x.data)[i]
                : int64_t(static_cast<const int32_t*>(x.data)[i]);
}

// The row that an index names, or `rows` for none; *bad is set for an index
// outside the table that is not the padding.
__device__ __forceinline__ uint32_t row_of(const Index& x, int64_t t, bool* bad) {
  const bool inside = uint64_t(t) < uint64_t(x.rows);
  const bool padding = x.has_padding && t == x.padding;
  *bad |= !inside && !padding;
  return uint32_t(inside && !padding ? t : x.rows);
}

// Once a thread, for all its indices: an atomic between two of them would hold
// back the loads behind it.
__device__ __forceinline__ void report(bool bad) {
  if (bad) atomicOr(&g_token_fault, kFaultTokenRange);
}

// Adds this file's fault word to *word, and clears it if asked to.
static inline cudaError_t take_token_fault(bool clear, unsigned* word) {
  unsigned mine = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&mine, g_token_fault, sizeof(mine));
  if (e == cudaSuccess && clear && mine) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbol(g_token_fault, &zero, sizeof(zero));
  }
  *word |= mine;
  return e;
}

}  // namespace tokens
}  // namespace clad3dgs
