// Row kernels of the residual joins: stream of float, branch of __nv_bfloat16.
#include "residual_rows.cuh"

namespace lutb {
LUTB_JOIN_ROWS(float, __nv_bfloat16)
}  // namespace lutb
