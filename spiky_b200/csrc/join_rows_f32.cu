// Row kernels of the residual joins: stream of float, branch of float.
#include "residual_rows.cuh"

namespace lutb {
LUTB_JOIN_ROWS(float, float)
}  // namespace lutb
