// Row sums and their Adam pass for gradients of type float (row_sums.cuh).
#include "row_sums.cuh"

namespace clad3dgs {
namespace sums {
CLAD3DGS_ROW_SUMS(, float)
}  // namespace sums
}  // namespace clad3dgs
