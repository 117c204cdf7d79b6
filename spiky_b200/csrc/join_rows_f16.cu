// Row kernels of the residual joins: stream of __half, branch of __half.
#include "residual_rows.cuh"

namespace lutb {
LUTB_JOIN_ROWS(__half, __half)
}  // namespace lutb
