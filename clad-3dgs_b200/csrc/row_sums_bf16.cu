// Row sums and their Adam pass for gradients of type __nv_bfloat16 (row_sums.cuh).
#include "row_sums.cuh"

namespace clad3dgs {
namespace sums {
CLAD3DGS_ROW_SUMS(, __nv_bfloat16)
}  // namespace sums
}  // namespace clad3dgs
