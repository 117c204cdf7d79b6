// Row kernels of the residual joins: stream of __nv_bfloat16, branch of __nv_bfloat16.
#include "residual_rows.cuh"

namespace lutb {
LUTB_JOIN_ROWS(__nv_bfloat16, __nv_bfloat16)
}  // namespace lutb
