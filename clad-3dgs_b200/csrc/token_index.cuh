// The indices by which tokens name the rows of a table.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace clad3dgs {
namespace tokens {

// Set in the fault word when a kernel met an index outside its table that is not
// the padding.
constexpr unsigned kFaultTokenRange = 256u;

// The indices a caller gives.
struct Index {
  const void* data;
  bool wide;  // int64, else int32
  bool has_padding;
  int64_t padding;
  int64_t rows;
  unsigned* fault = nullptr;  // the device's fault word, for kernels that read indices
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
__device__ __forceinline__ void report(const Index& x, bool bad) {
  if (bad) atomicOr(x.fault, kFaultTokenRange);
}

}  // namespace tokens
}  // namespace clad3dgs
