// Row kernels of the residual joins: stream of float, branch of __half.
#include "residual_rows.cuh"

namespace lutb {
LUTB_JOIN_ROWS(float, __half)
}  // namespace lutb
