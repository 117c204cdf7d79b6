// Joins of a block with the residual stream, as their kernels see them:
//   t = drop(f), n = after-norm of t (affine), h = skip x + branch gate n, y = before-norm of h (affine);
// alone, h is x (the norm before a block).
#pragma once

#include "residual.cuh"

namespace lutb {

struct JoinArgs {
    const void *x, *f, *gate, *aw, *ab, *bw, *bb;
    void *h, *y;
    float4 *stats;   // per row: mean and reciprocal deviation of the after-norm, of the before-norm
    const int64_t *random;
    uint64_t site;
    DropRule drop;
    int64_t rows, width, gate_rows;   // gate_rows: rows that share a gate row, 0 without gate
    int32_t after, before;            // LUTB_NORM_*
    int32_t params_f32, gate_f32;     // else of the branch's type
    int32_t alone;                    // no branch: the norm before a block
    float eps, skip, branch;
    // backward
    const void *dh, *dy;
    void *dx, *df, *dgate;
    // Sums over rows: a block's own sums [4][blocks][width] (those asked for), and [chunks][width] for the gate; see JoinSplit
    float *sums[4];   // daw, dab, dbw, dbb
    float *gate_sums;
    int32_t gate_direct;   // a chunk is a whole gate row: written to dgate
    int64_t chunk_rows, chunks, group_rows, per_group;
};

// Rows are dealt to blocks in chunks of neighbouring rows that lie within one group of rows with a common gate row (one group where no
// gate is summed), so that a block's sum for a gate row ends with the chunk.  Nothing depends on which block is first.
struct JoinSplit {
    int64_t group_rows, per_group, chunk_rows, chunks;
    int blocks;
};

template <class F>
__device__ __forceinline__ float join_param(const void *p, bool f32, int64_t at, float none) {
    if (p == nullptr) return none;
    return f32 ? static_cast<const float *>(p)[at] : to_f32(static_cast<const F *>(p)[at]);
}

}  // namespace lutb
