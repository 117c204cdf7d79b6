// A block's output into the residual stream, with the dropout on it, the norm after it, its gate and scales, and the norm before the next
// block, forward and backward; without a block the norm alone.
#include <math.h>

#include "residual_rows.cuh"

namespace lutb {

// The kernels of this file take rows of any width and any number of rows, the entry points give them those that the row kernels (residual_rows.cuh)
// do not: a block a row, which goes through the row once for each sum and reads it from L1 and L2 after the first time, and forms the mask
// again each time.  2048 x 16392 fp32 with both norms, gate and dropout: forward 0.50 ms, backward 1.6 (the row kernels at 16384: 0.12 and
// 0.25; plain torch operations 7.2 for both).
constexpr int kRowThreads = 256;

// The sum over the block's threads, in every thread, the same order for all.
__device__ __forceinline__ float block_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kRowThreads / 32; k++) s += scratch[k];
    return s;
}

// fn(column, stays) for this thread's elements of a row: eight columns at a time, the same columns whatever the row (so that a row's sums
// do not depend on where it lies).  Eight columns take two blocks of the generator where a row does not begin with one.
template <class Fn>
__device__ __forceinline__ void each(const JoinArgs &a, int64_t row, const DropKey &key, Fn fn) {
    const int64_t at = row * a.width;
    const int off = (int)(at & 7);
    for (int64_t c0 = threadIdx.x * 8ll; c0 < a.width; c0 += kRowThreads * 8ll) {
        uint32_t kept = 0xffu;
        if (a.drop.on) {
            const uint64_t b = (uint64_t)(at + c0) >> 3;
            kept = keep_bits(b, key, a.drop);
            if (off) kept = kept >> off | keep_bits(b + 1, key, a.drop) << (8 - off);
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c0 + j < a.width) fn(c0 + j, kept >> j & 1);
    }
}

template <class X, class F>
struct JoinRow {
    const JoinArgs &a;
    const int64_t at, gate_at;
    float mean = 0.0f, r = 1.0f;   // of the after-norm
    __device__ JoinRow(const JoinArgs &args, int64_t row)
        : a(args), at(row * args.width), gate_at(args.gate_rows ? row / args.gate_rows * args.width : 0) {}
    __device__ float branch(int64_t c, uint32_t stays) const { return stays ? to_f32(static_cast<const F *>(a.f)[at + c]) * (a.drop.on ? a.drop.scale : 1.0f) : 0.0f; }
    __device__ float scaled(int64_t c, uint32_t stays) const { return (branch(c, stays) - mean) * r; }
    __device__ float normed(int64_t c, uint32_t stays) const {
        return scaled(c, stays) * join_param<F>(a.aw, a.params_f32, c, 1.0f) + join_param<F>(a.ab, a.params_f32, c, 0.0f);
    }
    __device__ float gate(int64_t c) const { return a.branch * join_param<F>(a.gate, a.gate_f32, gate_at + c, 1.0f); }
    __device__ float stream(int64_t c, uint32_t stays) const {
        const float x = to_f32(static_cast<const X *>(a.x)[at + c]);
        return a.alone ? x : a.skip * x + gate(c) * normed(c, stays);
    }
};

template <class X, class F>
__global__ void __launch_bounds__(kRowThreads) join_forward_kernel(const JoinArgs a) {
    __shared__ float scratch[kRowThreads / 32];
    const DropKey key = a.drop.on ? drop_key(a.random, a.site) : DropKey{};
    const float width = (float)a.width;
    for (int64_t row = blockIdx.x * a.chunk_rows, end = min(row + a.chunk_rows, a.rows); row < end; row++) {
        JoinRow<X, F> j(a, row);
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (a.after != LUTB_NORM_NONE) {
            float s = 0.0f;
            if (a.after == LUTB_NORM_LAYER) {
                each(a, row, key, [&](int64_t c, uint32_t k) { s += j.branch(c, k); });
                st.x = block_sum(s, scratch) / width;
            }
            s = 0.0f;
            each(a, row, key, [&](int64_t c, uint32_t k) {
                const float d = j.branch(c, k) - st.x;
                s += d * d;
            });
            st.y = 1.0f / sqrtf(block_sum(s, scratch) / width + a.eps);
            j.mean = st.x;
            j.r = st.y;
        }
        if (a.before != LUTB_NORM_NONE) {
            float s = 0.0f;
            if (a.before == LUTB_NORM_LAYER) {
                each(a, row, key, [&](int64_t c, uint32_t k) { s += j.stream(c, k); });
                st.z = block_sum(s, scratch) / width;
            }
            s = 0.0f;
            each(a, row, key, [&](int64_t c, uint32_t k) {
                const float d = j.stream(c, k) - st.z;
                s += d * d;
            });
            st.w = 1.0f / sqrtf(block_sum(s, scratch) / width + a.eps);
        }
        each(a, row, key, [&](int64_t c, uint32_t k) {
            const float h = j.stream(c, k);
            if (a.h) static_cast<X *>(a.h)[j.at + c] = from_f32<X>(h);
            if (a.y)
                static_cast<F *>(a.y)[j.at + c] = from_f32<F>((h - st.z) * st.w * join_param<F>(a.bw, a.params_f32, c, 1.0f) +
                                                              join_param<F>(a.bb, a.params_f32, c, 0.0f));
        });
        if (a.stats && threadIdx.x == 0) a.stats[row] = st;
    }
}

// Per row: u = dy bw, dh' = dh + q (u - [mean u] - zh mean(u zh)); dn = branch gate dh', v = dn aw, dt = r (v - [mean v] - xh mean(v xh)).  The
// block's sums over its rows lie in its own slices of the workspace.
template <class X, class F>
__global__ void __launch_bounds__(kRowThreads) join_backward_kernel(const JoinArgs a) {
    __shared__ float scratch[kRowThreads / 32];
    const DropKey key = a.drop.on ? drop_key(a.random, a.site) : DropKey{};
    const float width = (float)a.width;
    float *sums[4];
    for (int k = 0; k < 4; k++) {
        sums[k] = a.sums[k] ? a.sums[k] + blockIdx.x * a.width : nullptr;
        if (sums[k])
            for (int64_t c = threadIdx.x; c < a.width; c += kRowThreads) sums[k][c] = 0.0f;
    }
    const X *dh_in = static_cast<const X *>(a.dh);
    const F *dy_in = static_cast<const F *>(a.dy);
    const bool gate_summed = a.dgate && a.gate_rows > 1;
    for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const int64_t group = chunk / a.per_group, begin = group * a.group_rows + (chunk - group * a.per_group) * a.chunk_rows;
        const int64_t end = min(begin + a.chunk_rows, min((group + 1) * a.group_rows, a.rows));
        float *const gate_sums = gate_summed ? a.gate_sums + (a.gate_direct ? (int64_t)blockIdx.x : chunk) * a.width : nullptr;
        if (gate_summed)
            for (int64_t c = threadIdx.x; c < a.width; c += kRowThreads) gate_sums[c] = 0.0f;
        __syncthreads();
        for (int64_t row = begin; row < end; row++) {
            JoinRow<X, F> j(a, row);
            const float4 st = a.stats ? a.stats[row] : make_float4(0.0f, 1.0f, 0.0f, 1.0f);
            j.mean = st.x;
            j.r = st.y;
            float c1 = 0.0f, c2 = 0.0f;
            if (a.dy) {
                float s1 = 0.0f, s2 = 0.0f;
                each(a, row, key, [&](int64_t c, uint32_t k) {
                    const float u = to_f32(dy_in[j.at + c]) * join_param<F>(a.bw, a.params_f32, c, 1.0f);
                    s1 += u * ((j.stream(c, k) - st.z) * st.w);
                    s2 += u;
                });
                c1 = block_sum(s1, scratch) / width;
                if (a.before == LUTB_NORM_LAYER) c2 = block_sum(s2, scratch) / width;
            }
            auto stream_gradient = [&](int64_t c, float zh) {
                float d = dh_in ? to_f32(dh_in[j.at + c]) : 0.0f;
                if (a.dy) d += st.w * (to_f32(dy_in[j.at + c]) * join_param<F>(a.bw, a.params_f32, c, 1.0f) - c2 - zh * c1);
                return d;
            };
            auto scaled_stream = [&](int64_t c, uint32_t k) { return a.dy ? (j.stream(c, k) - st.z) * st.w : 0.0f; };
            float m1 = 0.0f, m2 = 0.0f;
            if (a.after != LUTB_NORM_NONE && a.df) {
                float s1 = 0.0f, s2 = 0.0f;
                each(a, row, key, [&](int64_t c, uint32_t k) {
                    const float v = j.gate(c) * stream_gradient(c, scaled_stream(c, k)) * join_param<F>(a.aw, a.params_f32, c, 1.0f);
                    s1 += v;
                    s2 += v * j.scaled(c, k);
                });
                m2 = block_sum(s2, scratch) / width;
                if (a.after == LUTB_NORM_LAYER) m1 = block_sum(s1, scratch) / width;
            }
            each(a, row, key, [&](int64_t c, uint32_t k) {
                const float zh = scaled_stream(c, k), d = stream_gradient(c, zh);
                if (a.dy) {
                    const float g = to_f32(dy_in[j.at + c]);
                    if (sums[2]) sums[2][c] += g * zh;
                    if (sums[3]) sums[3][c] += g;
                }
                if (a.dx) static_cast<X *>(a.dx)[j.at + c] = from_f32<X>(a.alone ? d : a.skip * d);
                if (a.alone) return;
                if (a.dgate) {
                    const float dg = a.branch * d * j.normed(c, k);
                    if (gate_summed)
                        gate_sums[c] += dg;
                    else if (a.gate_f32)
                        static_cast<float *>(a.dgate)[j.gate_at + c] = dg;
                    else
                        static_cast<F *>(a.dgate)[j.gate_at + c] = from_f32<F>(dg);
                }
                const float dn = j.gate(c) * d, xh = a.after == LUTB_NORM_NONE ? 0.0f : j.scaled(c, k);
                if (sums[0]) sums[0][c] += dn * xh;
                if (sums[1]) sums[1][c] += dn;
                if (a.df) {
                    const float dt = a.after == LUTB_NORM_NONE ? dn : j.r * (dn * join_param<F>(a.aw, a.params_f32, c, 1.0f) - m1 - xh * m2);
                    static_cast<F *>(a.df)[j.at + c] = from_f32<F>(k ? dt * (a.drop.on ? a.drop.scale : 1.0f) : 0.0f);
                }
            });
        }
        if (gate_summed && a.gate_direct) {
            for (int64_t c0 = threadIdx.x * 8ll; c0 < a.width; c0 += kRowThreads * 8ll)   // (this thread's columns)
                for (int64_t c = c0; c < min(c0 + 8, a.width); c++) {
                    if (a.gate_f32)
                        static_cast<float *>(a.dgate)[group * a.width + c] = gate_sums[c];
                    else
                        static_cast<F *>(a.dgate)[group * a.width + c] = from_f32<F>(gate_sums[c]);
                }
            __syncthreads();   // (the next chunk clears them by other threads)
        }
    }
}

// The blocks' sums into the gradients: 32 lanes of V columns a block, whose warps share the partial sums; always the same order.
struct SumList {
    const float *from[5];
    void *to[5];
    int64_t parts[5];   // partial sums of an output row
    int32_t f32[5];
    int32_t count;      // lists of one row each; the gate's rows follow
};
template <class F, int V>
__global__ void __launch_bounds__(1024) join_sums_kernel(const SumList l, int64_t width) {
    __shared__ float all[32][32 * V + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, k = min((int)blockIdx.y, l.count);
    const int64_t first = (int64_t)blockIdx.x * (32 * V), c = first + lane * V, out_row = (int)blockIdx.y - k;
    const float *from = l.from[k] + out_row * l.parts[k] * width + c;
    constexpr int kAhead = 8;   // loads on their way
    float s[V];
#pragma unroll
    for (int e = 0; e < V; e++) s[e] = 0.0f;
    if (c < width) {
        const int64_t parts = l.parts[k], step = (int64_t)warps * width;
        int64_t p = warp;
        auto load = [&](int64_t at, float *v) {
            if constexpr (V == 4) {
                const float4 q = __ldcs(reinterpret_cast<const float4 *>(from + at));
                v[0] = q.x;
                v[1] = q.y;
                v[2] = q.z;
                v[3] = q.w;
            } else {
                v[0] = __ldcs(from + at);
            }
        };
        for (; p + (kAhead - 1) * warps < parts; p += kAhead * warps) {
            float v[kAhead][V];
#pragma unroll
            for (int a = 0; a < kAhead; a++) load(p * width + a * step, v[a]);
#pragma unroll
            for (int a = 0; a < kAhead; a++)
#pragma unroll
                for (int e = 0; e < V; e++) s[e] += v[a][e];
        }
        for (; p < parts; p += warps) {
            float v[V];
            load(p * width, v);
#pragma unroll
            for (int e = 0; e < V; e++) s[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < V; e++) all[warp][lane * V + e] = s[e];
    __syncthreads();
    for (int at = warp; at < 32 * V; at += warps) {   // a warp a column
        float sum = lane < warps ? all[lane][at] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0 && first + at < width) {
            if (l.f32[k])
                static_cast<float *>(l.to[k])[out_row * width + first + at] = sum;
            else
                static_cast<F *>(l.to[k])[out_row * width + first + at] = from_f32<F>(sum);
        }
    }
}
// Wide rows: four columns a lane and as many warps as have four partial sums each; narrow ones: one column and all warps, so that there are more
// blocks (1024 columns of 592 sums, three lists: 96 blocks).
template <class F>
static int launch_sums(const SumList &l, int64_t out_rows, int64_t width, cudaStream_t stream) {
    int64_t parts = 1;
    for (int k = 0; k < 5; k++) parts = l.parts[k] > parts ? l.parts[k] : parts;
    int warps = 4;
    while (warps < 32 && 4 * warps < parts) warps *= 2;
    KernelScope scope(K_JOIN_SUMS, stream);
    if (width % 4 == 0 && width >= 4096)
        join_sums_kernel<F, 4><<<dim3((unsigned)((width + 127) / 128), (unsigned)out_rows), 32 * warps, 0, stream>>>(l, width);
    else
        join_sums_kernel<F, 1><<<dim3((unsigned)((width + 31) / 32), (unsigned)out_rows), 32 * warps, 0, stream>>>(l, width);
    LUTB_LAUNCH_CHECK();
    return LUTB_OK;
}

// `at_once`: rows that a block takes together.
static JoinSplit join_split(int64_t rows, int64_t group_rows, int64_t blocks_wanted, int at_once) {
    const int64_t groups = rows / group_rows;
    JoinSplit best{};
    int64_t best_rounds = INT64_MAX;
    for (int64_t turns = 1; turns <= 4; turns++) {   // chunks a block takes one after another
        int64_t k = turns * blocks_wanted / groups;
        k = k < 1 ? 1 : k > group_rows ? group_rows : k;
        const int64_t steps = ((group_rows + k - 1) / k + at_once - 1) / at_once, chunk_rows = steps * at_once;
        k = (group_rows + chunk_rows - 1) / chunk_rows;
        const int64_t chunks = groups * k, rounds = (chunks + blocks_wanted - 1) / blocks_wanted * steps;
        if (rounds < best_rounds) {
            best_rounds = rounds;
            best = {group_rows, k, chunk_rows, chunks, (int)(chunks < blocks_wanted ? chunks : blocks_wanted)};
        }
    }
    return best;
}

// fn(X{}, F{}) for the element types of the stream and the branch
template <class Fn>
static auto by_types(const lutb_join_cfg *c, Fn fn) {
    if (c->branch_type == LUTB_BF16) return c->stream_type == LUTB_F32 ? fn(float(), __nv_bfloat16()) : fn(__nv_bfloat16(), __nv_bfloat16());
    if (c->branch_type == LUTB_F16) return c->stream_type == LUTB_F32 ? fn(float(), __half()) : fn(__half(), __half());
    return fn(float(), float());
}

int resident_clusters(const void *kernel, const RowShape &s, size_t smem) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmemPerBlock - kBackwardStatic) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(s.cluster * 64));
    config.blockDim = dim3((unsigned)s.threads);
    config.dynamicSmemBytes = smem;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = (unsigned)s.cluster;
    attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

// Gives the shape its stages (the most of three with which as many threads as registers allow are resident, or, forward, 384 an SM; two or one
// otherwise) and returns how many teams of blocks the device holds: a cluster beyond those would run in a second round.  Threads by registers:
// 512 an SM, 384 of the forward kernel with four groups (kForwardBlocks), 640 of a norm's backward pass in blocks, which takes 90
// (32768 x 1024 bf16 52 us with 512, 48 with 640).
static int64_t resident(const lutb_join_cfg *cfg, bool backward, bool vec, bool alone, RowShape &s) {
    const DeviceInfo info = device_info();
    const int sm = info.sm_count > 0 ? info.sm_count : 148;   // (no device: a size can be asked for all the same)
    const size_t own = backward ? (s.kind == TEAM_WARP ? kBackwardStatic : kBackwardTeamStatic) : vec ? kForwardVecStatic : kForwardStatic;
    const int threads = backward ? (alone && s.kind == TEAM_BLOCK ? 640 : 512) : !alone && s.kind == TEAM_WARP && s.groups == 4 ? 384 : 512;
    const int most = threads / s.threads, wanted = backward ? most : 384 / s.threads > 1 ? 384 / s.threads : 1;
    int blocks = 1;
    size_t dynamic = 0;
    for (s.stages = 3; s.stages >= 1; s.stages--) {
        dynamic = by_types(cfg, [&](auto xt, auto ft) { return join_rows_smem<decltype(xt), decltype(ft)>(backward, vec, s, alone, cfg->gate_rows == 1); });
        blocks = dynamic > kMaxSmemPerBlock - kBackwardStatic ? 0 : (int)(kMaxSmemPerBlock / (dynamic + own));
        if (blocks >= wanted || (s.stages == 2 && blocks >= 1) || s.stages == 1) break;
    }
    blocks = blocks < 1 ? 1 : blocks < most ? blocks : most;
    if (s.cluster == 1) return (int64_t)sm * blocks;
    // (asking takes some twenty microseconds: the last answer for each pair of types is kept)
    struct Asked {
        int device, threads, cluster, clusters;
        size_t smem;
    };
    static thread_local Asked kept[2][9] = {};
    Asked &k = kept[backward][cfg->stream_type * 3 + cfg->branch_type];
    if (info.sm_count > 0 && (k.clusters == 0 || k.device != info.device || k.threads != s.threads || k.cluster != s.cluster || k.smem != dynamic))
        k = {info.device, s.threads, s.cluster,
             by_types(cfg, [&](auto xt, auto ft) { return join_rows_clusters<decltype(xt), decltype(ft)>(backward, s, dynamic); }), dynamic};
    return info.sm_count > 0 && k.clusters > 0 ? k.clusters : sm * blocks / s.cluster;
}
static bool row_kernels(const lutb_join_cfg *cfg) { return cfg->width <= kRowMaxWidth && cfg->rows <= kRowMaxRows; }

// How the rows are dealt, and to what shape of block (unless rows are too wide or too many for the row kernels).
static JoinSplit split_forward(const lutb_join_cfg *cfg, bool vec, bool alone, RowShape &s) {
    const int have = device_info().sm_count;
    if (!row_kernels(cfg)) return join_split(cfg->rows, cfg->rows, (have > 0 ? have : 148) * 8ll, 1);
    s = forward_shape(cfg->width, vec);
    const int64_t blocks = resident(cfg, false, vec, alone, s);
    return join_split(cfg->rows, cfg->rows, blocks, s.teams);
}
static JoinSplit split_backward(const lutb_join_cfg *cfg, bool gate_gradient, bool vec, bool alone, RowShape &s) {
    const int64_t group_rows = gate_gradient && cfg->gate_rows > 1 ? cfg->gate_rows : cfg->rows;
    const int have = device_info().sm_count;
    if (!row_kernels(cfg)) return join_split(cfg->rows, group_rows, (have > 0 ? have : 148) * 4ll, 1);
    s = backward_shape(cfg->width);
    const int64_t blocks = resident(cfg, true, vec, alone, s);
    return join_split(cfg->rows, group_rows, blocks, s.teams);
}
// Rows of workspace for the gate's sums: one a chunk, or where a chunk is a whole gate row none (the kernel for wide rows: one a block).
static int64_t gate_sum_rows(const lutb_join_cfg *cfg, const JoinSplit &s) {
    return cfg->gate_rows <= 1 ? 0 : s.per_group > 1 ? s.chunks : row_kernels(cfg) ? 0 : s.blocks;
}
static void take_split(JoinArgs &a, const JoinSplit &s) {
    a.group_rows = s.group_rows;
    a.per_group = s.per_group;
    a.chunk_rows = s.chunk_rows;
    a.chunks = s.chunks;
}

int launch_rows(const void *kernel, std::atomic<uint32_t> &opted, const JoinArgs &a, const RowShape &s, int clusters, size_t smem, cudaStream_t stream) {
    if (smem > kPlainSmem - kBackwardStatic) {
        const int device = device_info().device;
        const uint32_t bit = device < 32 ? 1u << device : 0;
        if (!(opted.load(std::memory_order_relaxed) & bit)) {
            LUTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmemPerBlock - kBackwardStatic));
            opted.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    JoinArgs args = a;
    RowShape shape = s;
    void *params[2] = {&args, &shape};
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(clusters * s.cluster));
    config.blockDim = dim3((unsigned)s.threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    if (s.cluster > 1) {
        attribute[0].id = cudaLaunchAttributeClusterDimension;
        attribute[0].val.clusterDim.x = (unsigned)s.cluster;
        attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
        config.attrs = attribute;
        config.numAttrs = 1;
    }
    LUTB_CUDA(cudaLaunchKernelExC(&config, kernel, params));
    return LUTB_OK;
}

static bool all_aligned(uintptr_t to, std::initializer_list<const void *> list) {
    uintptr_t all = 0;
    for (const void *p : list) all |= reinterpret_cast<uintptr_t>(p);
    return all % to == 0;
}

static int check_join(const lutb_join_cfg *c) {
    LUTB_REQUIRE(c != nullptr, LUTB_ERR_NULL, "cfg is NULL");
    auto type_ok = [](int t) { return t == LUTB_F32 || t == LUTB_BF16 || t == LUTB_F16; };
    LUTB_REQUIRE(type_ok(c->stream_type) && type_ok(c->branch_type), LUTB_ERR_MODE, "unknown element type");
    LUTB_REQUIRE(c->stream_type == c->branch_type || c->stream_type == LUTB_F32, LUTB_ERR_MODE,
                 "the branch must have the stream's type, or the stream must be float32");
    LUTB_REQUIRE(c->param_type == LUTB_F32 || c->param_type == c->branch_type, LUTB_ERR_MODE, "norm parameters must be float32 or of the branch's type");
    LUTB_REQUIRE(c->gate_type == LUTB_F32 || c->gate_type == c->branch_type, LUTB_ERR_MODE, "a gate must be float32 or of the branch's type");
    LUTB_REQUIRE(c->rows >= 0, LUTB_ERR_SHAPE, "rows < 0");
    LUTB_REQUIRE(c->width > 0 && c->width <= INT32_MAX, LUTB_ERR_SHAPE, "width must be between 1 and 2^31 - 1");
    LUTB_REQUIRE(c->rows <= INT64_MAX / 16 / c->width, LUTB_ERR_SHAPE, "too many rows");
    LUTB_REQUIRE(c->after >= LUTB_NORM_NONE && c->after <= LUTB_NORM_LAYER && c->before >= LUTB_NORM_NONE && c->before <= LUTB_NORM_LAYER,
                 LUTB_ERR_MODE, "unknown norm");
    LUTB_REQUIRE(c->gate_rows >= 0 && (c->gate_rows == 0 || c->rows % c->gate_rows == 0), LUTB_ERR_SHAPE, "rows must be a multiple of gate_rows");
    LUTB_REQUIRE(c->eps > 0.0f && isfinite(c->eps), LUTB_ERR_SHAPE, "eps must be positive");
    LUTB_REQUIRE(isfinite(c->skip_scale) && isfinite(c->branch_scale), LUTB_ERR_SHAPE, "scales must be finite");
    LUTB_REQUIRE(c->dropout >= 0.0 && c->dropout <= 1.0, LUTB_ERR_SHAPE, "dropout probability must be between 0 and 1");
    LUTB_REQUIRE(c->site >= 0, LUTB_ERR_SHAPE, "site < 0");
    return LUTB_OK;
}

static bool aligned(const void *p, int type) { return reinterpret_cast<uintptr_t>(p) % (type == LUTB_F32 ? 4 : 2) == 0; }

static JoinArgs join_args(const lutb_join_cfg *c) {
    JoinArgs a{};
    a.site = (uint64_t)c->site;
    a.drop = drop_rule(c->dropout);
    a.rows = c->rows;
    a.width = c->width;
    a.after = c->after;
    a.before = c->before;
    a.params_f32 = c->param_type == LUTB_F32;
    a.gate_f32 = c->gate_type == LUTB_F32;
    a.eps = c->eps;
    a.skip = c->skip_scale;
    a.branch = c->branch_scale;
    return a;
}

int join_wait_errors(int *count_out) {
    int all = 0, one = 0;
    int (*const each[5])(int *) = {join_rows_wait_errors<float, float>, join_rows_wait_errors<__nv_bfloat16, __nv_bfloat16>,
                                   join_rows_wait_errors<__half, __half>, join_rows_wait_errors<float, __nv_bfloat16>, join_rows_wait_errors<float, __half>};
    for (auto read : each) {
        if (int rc = read(&one)) return rc;
        all += one;
    }
    *count_out = all;
    return LUTB_OK;
}

}  // namespace lutb

extern "C" int lutb_join_forward(const lutb_join_cfg *cfg, const void *x, const void *f, const void *gate, const void *after_weight,
                                 const void *after_bias, const void *before_weight, const void *before_bias, const int64_t *random,
                                 void *h, void *y, float *stats, void *stream) {
    using namespace lutb;
    if (int rc = check_join(cfg)) return rc;
    if (cfg->rows == 0) return LUTB_OK;
    LUTB_REQUIRE(x != nullptr, LUTB_ERR_NULL, "x is required");
    LUTB_REQUIRE(f != nullptr || (gate == nullptr && cfg->after == LUTB_NORM_NONE && cfg->dropout == 0.0 && h == nullptr), LUTB_ERR_NULL,
                 "a join without branch has no gate, no norm after it, no dropout and no stream output");
    LUTB_REQUIRE(f == nullptr || h != nullptr, LUTB_ERR_NULL, "h is required");
    LUTB_REQUIRE((y != nullptr) == (cfg->before != LUTB_NORM_NONE) && (f != nullptr || y != nullptr), LUTB_ERR_NULL, "y goes with the norm before the next block");
    LUTB_REQUIRE((gate != nullptr) == (cfg->gate_rows > 0), LUTB_ERR_NULL, "gate goes with gate_rows");
    LUTB_REQUIRE(cfg->dropout == 0.0 || random != nullptr, LUTB_ERR_NULL, "random is required for dropout");
    LUTB_REQUIRE(aligned(x, cfg->stream_type) && aligned(h, cfg->stream_type) && aligned(f, cfg->branch_type) && aligned(y, cfg->branch_type) &&
                     aligned(gate, cfg->gate_type) && aligned(after_weight, cfg->param_type) && aligned(after_bias, cfg->param_type) &&
                     aligned(before_weight, cfg->param_type) && aligned(before_bias, cfg->param_type),
                 LUTB_ERR_ALIGN, "arrays must be aligned to their elements");
    LUTB_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 16 == 0 && reinterpret_cast<uintptr_t>(random) % 8 == 0, LUTB_ERR_ALIGN,
                 "stats must be 16-byte aligned, random 8-byte aligned");
    JoinArgs a = join_args(cfg);
    a.x = x; a.f = f; a.gate = gate; a.aw = after_weight; a.ab = after_bias; a.bw = before_weight; a.bb = before_bias;
    a.h = h; a.y = y; a.stats = reinterpret_cast<float4 *>(stats); a.random = random; a.gate_rows = cfg->gate_rows;
    const bool vec = cfg->width % kRowElems == 0 && all_aligned(16, {x, f, gate, after_weight, after_bias, before_weight, before_bias}) && all_aligned(32, {h, y});
    RowShape shape{};
    const JoinSplit split = split_forward(cfg, vec, f == nullptr, shape);
    a.alone = f == nullptr;
    take_split(a, split);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return by_types(cfg, [&](auto xt, auto ft) -> int {
        KernelScope scope(K_JOIN_FORWARD, s);
        if (row_kernels(cfg)) return join_rows<decltype(xt), decltype(ft)>(false, vec, a, shape, split.blocks, s);
        join_forward_kernel<decltype(xt), decltype(ft)><<<split.blocks, kRowThreads, 0, s>>>(a);
        LUTB_LAUNCH_CHECK();
        return (int)LUTB_OK;
    });
}

extern "C" size_t lutb_join_backward_workspace(const lutb_join_cfg *cfg) {
    using namespace lutb;
    if (check_join(cfg) || cfg->rows == 0) return 0;
    size_t floats = 0;
    for (int vec = 0; vec < 2; vec++)
        for (int kind = 0; kind < 3; kind++) {   // a join, one whose gate has a gradient, a norm alone
            RowShape shape{};
            const bool gated = kind == 1;
            const JoinSplit split = split_backward(cfg, gated, vec != 0, kind == 2, shape);
            const size_t need = (size_t)(4 * split.blocks + (gated ? gate_sum_rows(cfg, split) : 0)) * cfg->width;
            floats = need > floats ? need : floats;
        }
    return floats * sizeof(float);
}

extern "C" int lutb_join_backward(const lutb_join_cfg *cfg, const void *x, const void *f, const void *gate, const void *after_weight,
                                  const void *after_bias, const void *before_weight, const int64_t *random, const float *stats,
                                  const void *dh, const void *dy, void *dx, void *df, void *dgate, void *d_after_weight, void *d_after_bias,
                                  void *d_before_weight, void *d_before_bias, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace lutb;
    if (int rc = check_join(cfg)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    LUTB_REQUIRE((gate != nullptr) == (cfg->gate_rows > 0) && (gate != nullptr || dgate == nullptr), LUTB_ERR_NULL, "gate goes with gate_rows");
    LUTB_REQUIRE(cfg->after != LUTB_NORM_NONE || (d_after_weight == nullptr && d_after_bias == nullptr), LUTB_ERR_MODE, "there is no norm after the block");
    LUTB_REQUIRE(dy != nullptr || cfg->rows == 0 || (d_before_weight == nullptr && d_before_bias == nullptr), LUTB_ERR_NULL,
                 "the gradients of the norm before the next block come from dy");
    LUTB_REQUIRE(dy == nullptr || cfg->before != LUTB_NORM_NONE, LUTB_ERR_MODE, "dy goes with the norm before the next block");
    void *const wanted[4] = {d_after_weight, d_after_bias, d_before_weight, d_before_bias};
    if (cfg->rows == 0) {
        const size_t bytes = (size_t)cfg->width * (cfg->param_type == LUTB_F32 ? 4 : 2);
        for (void *p : wanted)
            if (p) LUTB_CUDA(cudaMemsetAsync(p, 0, bytes, s));
        return LUTB_OK;
    }
    LUTB_REQUIRE(dh != nullptr || dy != nullptr, LUTB_ERR_NULL, "a gradient is required");
    LUTB_REQUIRE(stats != nullptr || (cfg->after == LUTB_NORM_NONE && dy == nullptr), LUTB_ERR_NULL, "stats are required for norms");
    LUTB_REQUIRE(x != nullptr || dy == nullptr, LUTB_ERR_NULL, "x is required for the norm before the next block");
    const bool alone = f == nullptr && cfg->before != LUTB_NORM_NONE;
    LUTB_REQUIRE(!alone || (gate == nullptr && cfg->after == LUTB_NORM_NONE && cfg->dropout == 0.0 && df == nullptr && dy != nullptr && dh == nullptr), LUTB_ERR_NULL,
                 "a norm alone has no gate, no norm after it, no dropout and no gradients of these");
    LUTB_REQUIRE(f != nullptr || alone || (cfg->after == LUTB_NORM_NONE && dgate == nullptr), LUTB_ERR_NULL, "f is required for its norm and for the gate's gradient");
    LUTB_REQUIRE(cfg->dropout == 0.0 || random != nullptr, LUTB_ERR_NULL, "random is required for dropout");
    LUTB_REQUIRE(aligned(x, cfg->stream_type) && aligned(dh, cfg->stream_type) && aligned(dx, cfg->stream_type) && aligned(f, cfg->branch_type) &&
                     aligned(dy, cfg->branch_type) && aligned(df, cfg->branch_type) && aligned(gate, cfg->gate_type) && aligned(dgate, cfg->gate_type) &&
                     aligned(after_weight, cfg->param_type) && aligned(after_bias, cfg->param_type) && aligned(before_weight, cfg->param_type),
                 LUTB_ERR_ALIGN, "arrays must be aligned to their elements");
    for (void *p : wanted) LUTB_REQUIRE(aligned(p, cfg->param_type), LUTB_ERR_ALIGN, "arrays must be aligned to their elements");
    LUTB_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 16 == 0 && reinterpret_cast<uintptr_t>(random) % 8 == 0, LUTB_ERR_ALIGN,
                 "stats must be 16-byte aligned, random 8-byte aligned");
    JoinArgs a = join_args(cfg);
    a.x = x; a.f = f; a.gate = gate; a.aw = after_weight; a.ab = after_bias; a.bw = before_weight; a.gate_rows = cfg->gate_rows;
    a.stats = reinterpret_cast<float4 *>(const_cast<float *>(stats)); a.random = random;
    a.dh = dh; a.dy = dy; a.dx = dx; a.df = df; a.dgate = dgate;
    const bool gate_summed = dgate != nullptr && cfg->gate_rows > 1;
    const bool vec = cfg->width % kRowElems == 0 &&
                     all_aligned(16, {x, f, gate, after_weight, after_bias, before_weight, dh, dy}) && all_aligned(32, {dx, df, dgate});
    RowShape shape{};
    const JoinSplit split = split_backward(cfg, dgate != nullptr, vec, alone, shape);
    a.alone = alone;
    take_split(a, split);
    a.gate_direct = gate_summed && split.per_group == 1;
    SumList l{};
    float *at = static_cast<float *>(workspace);
    size_t need = 0;
    for (int k = 0; k < 4; k++) {
        if (!wanted[k]) continue;
        a.sums[k] = at + need;
        l.from[l.count] = a.sums[k]; l.to[l.count] = wanted[k]; l.parts[l.count] = split.blocks; l.f32[l.count] = a.params_f32;
        l.count++;
        need += (size_t)split.blocks * cfg->width;
    }
    if (gate_summed) {
        a.gate_sums = at + need;
        l.from[l.count] = a.gate_sums; l.to[l.count] = dgate; l.parts[l.count] = split.per_group; l.f32[l.count] = a.gate_f32;
        need += (size_t)gate_sum_rows(cfg, split) * cfg->width;
    }
    LUTB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need * sizeof(float)), LUTB_ERR_WORKSPACE,
                 "workspace of %zu bytes needed", need * sizeof(float));
    LUTB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, LUTB_ERR_ALIGN, "workspace must be 16-byte aligned");
    return by_types(cfg, [&](auto xt, auto ft) -> int {
        {
            KernelScope scope(K_JOIN_BACKWARD, s);
            if (row_kernels(cfg)) {
                if (int rc = join_rows<decltype(xt), decltype(ft)>(true, vec, a, shape, split.blocks, s)) return rc;
            } else {
                join_backward_kernel<decltype(xt), decltype(ft)><<<split.blocks, kRowThreads, 0, s>>>(a);
                LUTB_LAUNCH_CHECK();
            }
        }
        const int64_t out_rows = l.count + (gate_summed && !a.gate_direct ? split.chunks / split.per_group : 0);
        if (out_rows) return launch_sums<decltype(ft)>(l, out_rows, cfg->width, s);
        return (int)LUTB_OK;
    });
}
