// Row kernels of the residual joins: a row's elements stay in registers from the first sum to the last store.
//
// A thread has eight elements of a row.  A team of threads has a row: a part of a warp up to 256 elements, a block up to 2048, a cluster of up
// to eight blocks up to 16384; sums over a row go through shuffles, shared memory and the cluster's shared memory accordingly, one
// exchange for each norm and direction (a norm's mean and squares are combined from the warps' own by the pairwise formula of Chan, Golub
// and LeVeque, 1979, so that no square is taken about a mean that is far off).  What a team does depends on the width alone, so that a row's
// result does not depend on the rows beside it.
//
// Rows in 16-byte aligned arrays of a multiple of eight elements (VEC): a thread's elements are neighbours, it fetches those of the next
// rows with 16-byte asynchronous copies into slots of shared memory of its own (no barrier), and one generator block decides its mask.
// Other rows: a thread's elements are a team apart, so that a warp's loads are neighbours, and the mask's bytes go through shared memory.
#pragma once

#include <atomic>

#include "residual_join.cuh"

namespace lutb {

constexpr int kRowElems = 8, kRowMaxThreads = 256, kRowMaxCluster = 8;
constexpr int64_t kRowMaxWidth = (int64_t)kRowElems * kRowMaxThreads * kRowMaxCluster;

struct RowShape {
    int team, teams, threads;   // threads of a row in a block, rows a block has at a time, threads of a block
    int cluster, slice;         // blocks of a row, columns of a block
};
inline RowShape row_shape(int64_t width) {
    RowShape s{};
    s.cluster = 1;
    while (width > (int64_t)s.cluster * kRowElems * kRowMaxThreads) s.cluster *= 2;
    const int t = (int)(((width + kRowElems - 1) / kRowElems + s.cluster - 1) / s.cluster);
    s.slice = t * kRowElems;
    if (t <= 32) {
        s.team = 1;
        while (s.team < t) s.team *= 2;
        s.threads = kRowMaxThreads;
        s.teams = s.threads / s.team;
    } else {
        s.team = s.threads = (t + 31) / 32 * 32;
        s.teams = 1;
    }
    return s;
}

// ------------------------------------------------------------------------------------------------ two floats an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)), "l"(reinterpret_cast<unsigned long long &>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float total(const float2 *v) {
    const float2 s = add2(add2(v[0], v[1]), add2(v[2], v[3]));
    return s.x + s.y;
}

// ------------------------------------------------------------------------------------------------ eight elements
__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 pair_of(uint32_t w, __half) { return __half22float2(reinterpret_cast<const __half2 &>(w)); }
__device__ __forceinline__ uint32_t word_of(float2 v, __nv_bfloat16) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
    return reinterpret_cast<const uint32_t &>(b);
}
__device__ __forceinline__ uint32_t word_of(float2 v, __half) {
    const __half2 b = __floats2half2_rn(v.x, v.y);
    return reinterpret_cast<const uint32_t &>(b);
}
template <class T>
constexpr int kParts = sizeof(T) * kRowElems / 16;   // 16-byte parts of eight elements

template <class T>
__device__ __forceinline__ void unpack8(const uint4 *part, float2 *v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int p = 0; p < 2; p++) {
            v[2 * p] = make_float2(__uint_as_float(part[p].x), __uint_as_float(part[p].y));
            v[2 * p + 1] = make_float2(__uint_as_float(part[p].z), __uint_as_float(part[p].w));
        }
    } else {
        v[0] = pair_of(part[0].x, T());
        v[1] = pair_of(part[0].y, T());
        v[2] = pair_of(part[0].z, T());
        v[3] = pair_of(part[0].w, T());
    }
}
template <class T>
__device__ __forceinline__ void store8(T *p, const float2 *v) {
    uint4 *q = reinterpret_cast<uint4 *>(p);
    if constexpr (sizeof(T) == 4) {
        q[0] = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
        q[1] = make_uint4(__float_as_uint(v[2].x), __float_as_uint(v[2].y), __float_as_uint(v[3].x), __float_as_uint(v[3].y));
    } else {
        q[0] = make_uint4(word_of(v[0], T()), word_of(v[1], T()), word_of(v[2], T()), word_of(v[3], T()));
    }
}
__device__ __forceinline__ void copy16(uint32_t to, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }

// ------------------------------------------------------------------------------------------------ a thread's place
struct RowPlace {
    int tid, t, team, teams, which;   // thread in the block, in its team; threads of a team, teams, this one
    int cluster, rank;
    int64_t width, first, limit;      // columns of the block: first .. limit - 1
    float warp_count;                 // elements of the warp
    uint32_t valid;                   // which of the eight elements exist
    uint32_t parity;
    float4 (*slots)[kRowMaxCluster * kRowMaxThreads / 32];

    template <bool VEC>
    __device__ __forceinline__ int64_t column(int k) const { return VEC ? first + t * 8 + k : first + t + (int64_t)k * team; }
};

template <bool VEC>
__device__ __forceinline__ RowPlace row_place(const JoinArgs &a, const RowShape &s, float4 (*slots)[kRowMaxCluster * kRowMaxThreads / 32]) {
    RowPlace p;
    p.tid = threadIdx.x;
    p.team = s.team;
    p.teams = s.teams;
    p.which = p.tid / s.team;
    p.t = p.tid - p.which * s.team;
    p.cluster = s.cluster;
    p.rank = s.cluster > 1 ? (int)(blockIdx.x % s.cluster) : 0;
    p.width = a.width;
    p.first = (int64_t)p.rank * s.slice;
    p.limit = min(p.first + s.slice, a.width);
    p.valid = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) p.valid |= (p.column<VEC>(k) < p.limit ? 1u : 0u) << k;
    p.warp_count = (float)__reduce_add_sync(0xffffffffu, __popc(p.valid));
    p.parity = 0;
    p.slots = slots;
    return p;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float team_sum(float v, int team) {   // teams of a warp or a part of one
    for (int o = team >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// A warp's values to every block of the row; they can be read after the sync, until the next but one.
__device__ __forceinline__ void publish(const RowPlace &p, float4 v) {
    const int lane = p.tid & 31, warps = p.team >> 5;
    if (p.cluster == 1) {
        if (lane == 0) p.slots[p.parity][p.tid >> 5] = v;
    } else if (lane < p.cluster) {
        uint32_t at = (uint32_t)__cvta_generic_to_shared(&p.slots[p.parity][p.rank * warps + (p.tid >> 5)]);
        asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(lane));
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
    }
}
__device__ __forceinline__ void meet(const RowPlace &p) {
    if (p.cluster == 1)
        __syncthreads();
    else
        cluster_sync();
}
// Sums of two values over the row; `between` runs while the others arrive.
template <class Fn>
__device__ __forceinline__ float2 row_sums(RowPlace &p, float a, float b, bool second, Fn between) {
    if (p.team <= 32) {
        a = team_sum(a, p.team);
        if (second) b = team_sum(b, p.team);
        between();
        return make_float2(a, b);
    }
    a = warp_sum(a);
    if (second) b = warp_sum(b);
    publish(p, make_float4(a, b, 0.0f, 0.0f));
    between();
    meet(p);
    float2 s = make_float2(0.0f, 0.0f);
    const int n = p.cluster * (p.team >> 5);
    for (int k = 0; k < n; k++) s = add2(s, *reinterpret_cast<const float2 *>(&p.slots[p.parity][k]));
    p.parity ^= 1;
    return s;
}
// Mean (0 for an RMS norm) and reciprocal deviation of the row's values; values of no element are 0.
template <bool VEC>
__device__ __forceinline__ float2 row_stats(RowPlace &p, const float2 *v, bool layer, float eps) {
    const float width = (float)p.width;
    auto squares = [&](float mean) {
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float2 d = add2(v[k], both(-mean));
            if (!VEC) {
                d.x = (p.valid >> (2 * k) & 1) ? d.x : 0.0f;
                d.y = (p.valid >> (2 * k) & 2) ? d.y : 0.0f;
            }
            s = fma2(d, d, s);
        }
        return p.valid ? s.x + s.y : 0.0f;
    };
    if (p.team <= 32) {
        const float mean = layer ? team_sum(total(v), p.team) / width : 0.0f;
        return make_float2(mean, rsqrtf(team_sum(squares(mean), p.team) / width + eps));
    }
    float mean = 0.0f;
    if (layer) {
        const float s = warp_sum(p.valid ? total(v) : 0.0f);
        mean = p.warp_count > 0.0f ? s / p.warp_count : 0.0f;
    }
    publish(p, make_float4(mean, warp_sum(squares(mean)), p.warp_count, 0.0f));
    meet(p);
    const int n = p.cluster * (p.team >> 5);
    float s = 0.0f;
    mean = 0.0f;
    if (layer) {
        for (int k = 0; k < n; k++) mean += p.slots[p.parity][k].x * p.slots[p.parity][k].z;
        mean /= width;
    }
    for (int k = 0; k < n; k++) {
        const float4 w = p.slots[p.parity][k];
        const float d = w.x - mean;
        s += layer ? w.y + w.z * d * d : w.y;
    }
    p.parity ^= 1;
    return make_float2(mean, rsqrtf(s / width + eps));
}

// Eight of a parameter's values; `none` where there is no such parameter, 0 for columns beyond the row.
template <class F, bool VEC>
__device__ __forceinline__ void param8(const RowPlace &p, const void *from, bool f32, int64_t at, float none, float scale, float2 *v) {
    float e[8];
    if (VEC && from != nullptr && p.valid) {
        const int64_t c = at + p.column<VEC>(0);
        if (f32) {
            const uint4 part[2] = {reinterpret_cast<const uint4 *>(static_cast<const float *>(from) + c)[0],
                                   reinterpret_cast<const uint4 *>(static_cast<const float *>(from) + c)[1]};
            unpack8<float>(part, v);
        } else {
            uint4 part[kParts<F>];
#pragma unroll
            for (int q = 0; q < kParts<F>; q++) part[q] = reinterpret_cast<const uint4 *>(static_cast<const F *>(from) + c)[q];
            unpack8<F>(part, v);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) e[k] = (p.valid >> k & 1) ? join_param<F>(from, f32, at + p.column<VEC>(k), none) : 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = mul2(v[k], both(scale));
}

// The rows of a block in turn: chunk by chunk, `teams` rows at a time.
struct RowCursor {
    int64_t chunk, base, end;
    __device__ __forceinline__ void enter(const JoinArgs &a) {
        if (chunk >= a.chunks) return;
        const int64_t group = chunk / a.per_group;
        base = group * a.group_rows + (chunk - group * a.per_group) * a.chunk_rows;
        end = min(base + a.chunk_rows, min((group + 1) * a.group_rows, a.rows));
    }
    __device__ __forceinline__ bool more(const JoinArgs &a) const { return chunk < a.chunks; }
    __device__ __forceinline__ void next(const JoinArgs &a, int teams, int64_t stride) {
        base += teams;
        if (base >= end) {
            chunk += stride;
            enter(a);
        }
    }
};

// The next rows' elements, in this thread's slots of shared memory (VEC), or nothing.
template <int STAGES>
struct RowRing {
    uint4 *at;         // [stage][part][thread]
    int parts, threads, tid;
    uint32_t fill = 0, take = 0;
    __device__ __forceinline__ void fetch(int part, const void *from, int n) const {
        for (int q = 0; q < n; q++)
            copy16((uint32_t)__cvta_generic_to_shared(at + ((int)fill * parts + part + q) * threads + tid), static_cast<const uint4 *>(from) + q);
    }
    __device__ __forceinline__ void filled() {
        asm volatile("cp.async.commit_group;" ::: "memory");
        fill = fill + 1 == STAGES ? 0 : fill + 1;
    }
    __device__ __forceinline__ void ready() const { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }
    __device__ __forceinline__ void taken() { take = take + 1 == STAGES ? 0 : take + 1; }
    template <class T>
    __device__ __forceinline__ void get(int part, float2 *v) const {
        uint4 w[kParts<T>];
#pragma unroll
        for (int q = 0; q < kParts<T>; q++) w[q] = at[((int)take * parts + part + q) * threads + tid];
        unpack8<T>(w, v);
    }
};

template <class T, bool VEC>
__device__ __forceinline__ void load_apart(const RowPlace &p, const T *row, bool on, float2 *v) {
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; k++) e[k] = on && (p.valid >> k & 1) ? to_f32(row[p.column<VEC>(k)]) : 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
}
template <class T, bool VEC>
__device__ __forceinline__ void store_row(const RowPlace &p, T *row, const float2 *v) {
    if constexpr (VEC) {
        if (p.valid) store8(row + p.column<VEC>(0), v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (p.valid >> k & 1) row[p.column<VEC>(k)] = from_f32<T>(k & 1 ? v[k >> 1].y : v[k >> 1].x);
    }
}
__device__ __forceinline__ void zero8(float2 *v) {
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = make_float2(0.0f, 0.0f);
}

// The mask of a thread's eight elements, as bits.  Rows that are not VEC: the team's generator blocks as bytes in shared memory, two sets
// in turn, so that one barrier a row is enough.
template <bool VEC>
__device__ __forceinline__ uint32_t row_mask(const RowPlace &p, const JoinArgs &a, const DropKey &key, int64_t row, uint8_t *bytes, uint32_t turn) {
    const int64_t at = row * a.width + p.first;
    if (VEC) return keep_bits((uint64_t)(at + p.t * 8) >> 3, key, a.drop);
    uint8_t *own = bytes + ((int)turn * p.teams + p.which) * (p.team + 1);
    const int off = (int)(at & 7);
    own[p.t] = (uint8_t)keep_bits(((uint64_t)at >> 3) + p.t, key, a.drop);
    if (p.t == 0) own[p.team] = (uint8_t)keep_bits(((uint64_t)at >> 3) + p.team, key, a.drop);
    if (p.team <= 32)
        __syncwarp();
    else
        __syncthreads();
    uint32_t kept = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int e = off + p.t + k * p.team;
        kept |= (uint32_t)(own[e >> 3] >> (e & 7) & 1) << k;
    }
    return kept;
}
__device__ __forceinline__ void drop8(float2 *v, uint32_t kept, float scale) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k].x = (kept >> (2 * k) & 1) ? v[k].x * scale : 0.0f;
        v[k].y = (kept >> (2 * k) & 2) ? v[k].y * scale : 0.0f;
    }
}
constexpr size_t kMaskBytes = 2 * 2 * kRowMaxThreads;   // two sets, a byte a thread and one a team

// ------------------------------------------------------------------------------------------------ forward
// BRANCH: 0 no branch (the norm alone), 1 a branch, 2 a branch with a norm of its own.  NEXT: the norm before the next block.
template <class X, class F>
constexpr int kForwardParts = kParts<X> + kParts<F>;   // x, f; two more for a gate of each element
constexpr int kForwardStages = 3;

template <class X, class F, int BRANCH, bool NEXT, bool VEC>
__global__ void __launch_bounds__(kRowMaxThreads, 2) join_rows_forward_kernel(const JoinArgs a, const RowShape shape) {
    extern __shared__ uint4 dynamic[];
    __shared__ float4 slots[2][kRowMaxCluster * kRowMaxThreads / 32];
    __shared__ uint8_t masks[VEC ? 1 : kMaskBytes];
    RowPlace p = row_place<VEC>(a, shape, slots);
    const DropKey key = BRANCH && a.drop.on ? drop_key(a.random, a.site) : DropKey{};
    float2 aw[4], ab[4], gate[4], bw[4], bb[4];
    if (BRANCH == 2) {
        param8<F, VEC>(p, a.aw, a.params_f32, 0, 1.0f, 1.0f, aw);
        param8<F, VEC>(p, a.ab, a.params_f32, 0, 0.0f, 1.0f, ab);
    }
    if (NEXT) {
        param8<F, VEC>(p, a.bw, a.params_f32, 0, 1.0f, 1.0f, bw);
        param8<F, VEC>(p, a.bb, a.params_f32, 0, 0.0f, 1.0f, bb);
    }
    const bool gate_each = BRANCH && a.gate_rows == 1;
    int64_t gate_end = 0;   // first row of another gate row
    if (BRANCH && a.gate_rows == 0) param8<F, VEC>(p, nullptr, true, 0, 1.0f, a.branch, gate);

    RowRing<kForwardStages> ring{dynamic, kForwardParts<X, F> + (gate_each ? 2 : 0), (int)blockDim.x, p.tid};
    const int64_t stride = gridDim.x / shape.cluster;
    RowCursor load{(int64_t)(blockIdx.x / shape.cluster), 0, 0}, here = load;
    load.enter(a);
    here.enter(a);
    auto fetch = [&]() {
        if (VEC) {
            if (load.more(a)) {
                const int64_t row = load.base + p.which, at = row * a.width + p.column<VEC>(0);
                if (row < load.end && p.valid) {
                    ring.fetch(0, static_cast<const X *>(a.x) + at, kParts<X>);
                    if (BRANCH) ring.fetch(kParts<X>, static_cast<const F *>(a.f) + at, kParts<F>);
                    if (gate_each) {
                        if (a.gate_f32)
                            ring.fetch(kParts<X> + kParts<F>, static_cast<const float *>(a.gate) + at, 2);
                        else
                            ring.fetch(kParts<X> + kParts<F>, static_cast<const F *>(a.gate) + at, kParts<F>);
                    }
                }
                load.next(a, p.teams, stride);
            }
            ring.filled();
        }
    };
#pragma unroll
    for (int s = 0; s < kForwardStages - 1; s++) fetch();
    if (p.cluster > 1) cluster_sync();   // the row's blocks are there
    uint32_t turn = 0;
    for (; here.more(a); here.next(a, p.teams, stride)) {
        const int64_t row = here.base + p.which, at = row * a.width;
        const bool on = row < here.end;
        if (BRANCH && a.gate_rows > 1 && on && row >= gate_end) {
            const int64_t gate_row = row / a.gate_rows;
            gate_end = (gate_row + 1) * a.gate_rows;
            param8<F, VEC>(p, a.gate, a.gate_f32, gate_row * a.width, 1.0f, a.branch, gate);
        }
        uint32_t kept = 0xffu;
        if (BRANCH && a.drop.on) kept = row_mask<VEC>(p, a, key, row, masks, turn);
        turn ^= 1;
        float2 h[4], v[4];
        if (VEC) {
            ring.ready();
            ring.template get<X>(0, h);
            if (BRANCH) ring.template get<F>(kParts<X>, v);
            if (gate_each) {
                if (a.gate_f32)
                    ring.template get<float>(kParts<X> + kParts<F>, gate);
                else
                    ring.template get<F>(kParts<X> + kParts<F>, gate);
            }
            ring.taken();
            if (!on || !p.valid) {
                zero8(h);
                if (BRANCH) zero8(v);
                if (gate_each) zero8(gate);
            }
        } else {
            load_apart<X, VEC>(p, static_cast<const X *>(a.x) + at, on, h);
            if (BRANCH) load_apart<F, VEC>(p, static_cast<const F *>(a.f) + at, on, v);
            if (gate_each) {
                if (a.gate_f32)
                    load_apart<float, VEC>(p, static_cast<const float *>(a.gate) + at, on, gate);
                else
                    load_apart<F, VEC>(p, static_cast<const F *>(a.gate) + at, on, gate);
            }
        }
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (BRANCH) {
            if (gate_each)
#pragma unroll
                for (int k = 0; k < 4; k++) gate[k] = mul2(gate[k], both(a.branch));
            if (a.drop.on) drop8(v, kept, a.drop.scale);
            if (BRANCH == 2) {
                const float2 s = row_stats<VEC>(p, v, a.after == LUTB_NORM_LAYER, a.eps);
                st.x = s.x;
                st.y = s.y;
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = fma2(mul2(add2(v[k], both(-s.x)), both(s.y)), aw[k], ab[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) h[k] = fma2(gate[k], v[k], mul2(h[k], both(a.skip)));
        }
        fetch();
        if (BRANCH && on) store_row<X, VEC>(p, static_cast<X *>(a.h) + at, h);
        if (NEXT) {
            const float2 s = row_stats<VEC>(p, h, a.before == LUTB_NORM_LAYER, a.eps);
            st.z = s.x;
            st.w = s.y;
#pragma unroll
            for (int k = 0; k < 4; k++) h[k] = fma2(mul2(add2(h[k], both(-s.x)), both(s.y)), bw[k], bb[k]);
            if (on) store_row<F, VEC>(p, static_cast<F *>(a.y) + at, h);
        }
        if (a.stats && on && p.t == 0 && p.rank == 0) a.stats[row] = st;
    }
}

// ------------------------------------------------------------------------------------------------ backward
template <class X, class F>
constexpr int kBackwardParts = 2 * kParts<X> + 2 * kParts<F>;   // x, dh, f, dy; two more for a gate of each element
template <class X, class F>
constexpr int kBackwardStages = sizeof(X) + sizeof(F) == 8 ? 2 : 3;
constexpr int kBackwardParams = 4;   // aw, ab, bw, gate

// See join_backward_kernel for the formulas.  A thread's sums over its rows stay in registers to the end (of the chunk, for a gate row).
template <class X, class F, int BRANCH, bool NEXT, bool VEC>
__global__ void __launch_bounds__(kRowMaxThreads, 2) join_rows_backward_kernel(const JoinArgs a, const RowShape shape) {
    extern __shared__ uint4 dynamic[];
    __shared__ float4 slots[2][kRowMaxCluster * kRowMaxThreads / 32];
    __shared__ uint8_t masks[VEC ? 1 : kMaskBytes];
    __shared__ float2 joined[4 * kRowMaxThreads];   // the teams' sums of a block
    RowPlace p = row_place<VEC>(a, shape, slots);
    const int threads = blockDim.x;
    const DropKey key = BRANCH && a.drop.on ? drop_key(a.random, a.site) : DropKey{};
    // parameters in slots of this thread's own: [parameter][half][thread]
    float4 *const params = reinterpret_cast<float4 *>(dynamic) + p.tid;
    auto keep_param = [&](int which, const void *from, bool f32, int64_t at, float none, float scale) {
        float2 v[4];
        param8<F, VEC>(p, from, f32, at, none, scale, v);
        params[(2 * which) * threads] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        params[(2 * which + 1) * threads] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    };
    auto param = [&](int which, float2 *v) {
        const float4 lo = params[(2 * which) * threads], hi = params[(2 * which + 1) * threads];
        v[0] = make_float2(lo.x, lo.y);
        v[1] = make_float2(lo.z, lo.w);
        v[2] = make_float2(hi.x, hi.y);
        v[3] = make_float2(hi.z, hi.w);
    };
    if (BRANCH == 2) {
        keep_param(0, a.aw, a.params_f32, 0, 1.0f, 1.0f);
        keep_param(1, a.ab, a.params_f32, 0, 0.0f, 1.0f);
    }
    if (NEXT) keep_param(2, a.bw, a.params_f32, 0, 1.0f, 1.0f);
    const bool gate_each = BRANCH && a.gate_rows == 1, gate_summed = BRANCH && a.dgate && a.gate_rows > 1;
    int64_t gate_end = 0;   // first row of another gate row
    if (BRANCH && a.gate_rows == 0) keep_param(3, nullptr, true, 0, 1.0f, a.branch);

    RowRing<kBackwardStages<X, F>> ring{dynamic + 2 * kBackwardParams * threads, kBackwardParts<X, F> + (gate_each ? 2 : 0), threads, p.tid};
    constexpr int kDh = kParts<X>, kF = 2 * kParts<X>, kDy = kF + kParts<F>, kGate = kDy + kParts<F>;
    const int64_t stride = gridDim.x / shape.cluster, own = blockIdx.x / shape.cluster;
    RowCursor load{own, 0, 0}, here = load;
    load.enter(a);
    here.enter(a);
    const X *const x_in = static_cast<const X *>(a.x), *const dh_in = static_cast<const X *>(a.dh);
    const F *const f_in = static_cast<const F *>(a.f), *const dy_in = static_cast<const F *>(a.dy);
    auto fetch = [&]() {
        if (VEC) {
            if (load.more(a)) {
                const int64_t row = load.base + p.which, at = row * a.width + p.column<VEC>(0);
                if (row < load.end && p.valid) {
                    if (NEXT) ring.fetch(0, x_in + at, kParts<X>);
                    if (dh_in) ring.fetch(kDh, dh_in + at, kParts<X>);
                    if (BRANCH) ring.fetch(kF, f_in + at, kParts<F>);
                    if (NEXT) ring.fetch(kDy, dy_in + at, kParts<F>);
                    if (gate_each) {
                        if (a.gate_f32)
                            ring.fetch(kGate, static_cast<const float *>(a.gate) + at, 2);
                        else
                            ring.fetch(kGate, static_cast<const F *>(a.gate) + at, kParts<F>);
                    }
                }
                load.next(a, p.teams, stride);
            }
            ring.filled();
        }
    };
    constexpr int kSums = 5;   // daw, dab, dbw, dbb, gate
    float2 sums[kSums][4];
#pragma unroll
    for (int s = 0; s < kSums; s++) zero8(sums[s]);
    // this thread's sum of eight columns, joined over the block's teams, handed on column by column
    auto hand_out = [&](const float2 *v, auto put) {
        if (p.teams == 1) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (p.valid >> k & 1) put(p.column<VEC>(k), k & 1 ? v[k >> 1].y : v[k >> 1].x);
            return;
        }
        float *all = reinterpret_cast<float *>(joined);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; k++) all[(VEC ? p.t * 8 + k : p.t + k * p.team) + p.which * p.team * 8] = k & 1 ? v[k >> 1].y : v[k >> 1].x;
        __syncthreads();
        for (int c = p.tid; c < (int)a.width; c += threads) {
            float s = 0.0f;
            for (int w = 0; w < p.teams; w++) s += all[w * p.team * 8 + c];
            put((int64_t)c, s);
        }
    };
#pragma unroll
    for (int s = 0; s < kBackwardStages<X, F> - 1; s++) fetch();
    if (p.cluster > 1) cluster_sync();
    uint32_t turn = 0;
    const float width = (float)a.width;
    while (here.more(a)) {
        const int64_t row = here.base + p.which, at = row * a.width, chunk = here.chunk;
        const bool on = row < here.end;
        const float4 st = on ? a.stats[row] : make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (BRANCH && a.gate_rows > 1 && on && row >= gate_end) {
            const int64_t gate_row = row / a.gate_rows;
            gate_end = (gate_row + 1) * a.gate_rows;
            keep_param(3, a.gate, a.gate_f32, gate_row * a.width, 1.0f, a.branch);
        }
        uint32_t kept = 0xffu;
        if (BRANCH && a.drop.on) kept = row_mask<VEC>(p, a, key, row, masks, turn);
        turn ^= 1;
        float2 d[4], t[4], z[4], g[4];   // dh, the branch, the stream, dy
        if (VEC) {
            ring.ready();
            if (NEXT) ring.template get<X>(0, z);
            if (dh_in) ring.template get<X>(kDh, d);
            if (BRANCH) ring.template get<F>(kF, t);
            if (NEXT) ring.template get<F>(kDy, g);
        } else {
            if (NEXT) load_apart<X, VEC>(p, x_in + at, on, z);
            if (dh_in) load_apart<X, VEC>(p, dh_in + at, on, d);
            if (BRANCH) load_apart<F, VEC>(p, f_in + at, on, t);
            if (NEXT) load_apart<F, VEC>(p, dy_in + at, on, g);
        }
        if (dh_in == nullptr || (VEC && (!on || !p.valid))) zero8(d);
        if (VEC && (!on || !p.valid)) {
            if (NEXT) zero8(z);
            if (BRANCH) zero8(t);
            if (NEXT) zero8(g);
        }
        float2 gate[4], w[4];
        if (BRANCH) {
            if (!gate_each)
                param(3, gate);
            else {
                if (VEC) {
                    if (a.gate_f32)
                        ring.template get<float>(kGate, gate);
                    else
                        ring.template get<F>(kGate, gate);
                    if (!on || !p.valid) zero8(gate);
                } else if (a.gate_f32) {
                    load_apart<float, VEC>(p, static_cast<const float *>(a.gate) + at, on, gate);
                } else {
                    load_apart<F, VEC>(p, static_cast<const F *>(a.gate) + at, on, gate);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) gate[k] = mul2(gate[k], both(a.branch));
            }
        }
        if (VEC) {
            ring.taken();
            fetch();
        }
        float2 n[4];   // the branch after its norm; t becomes its normalised values
        if (BRANCH) {
            if (a.drop.on) drop8(t, kept, a.drop.scale);
            if (BRANCH == 2) {
                float2 shift[4];
                param(0, w);
                param(1, shift);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    t[k] = mul2(add2(t[k], both(-st.x)), both(st.y));
                    n[k] = fma2(t[k], w[k], shift[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) n[k] = t[k];
            }
        }
        if (NEXT) {
            float2 u[4], s1 = make_float2(0.0f, 0.0f), bw[4];
            param(2, bw);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (BRANCH) z[k] = fma2(gate[k], n[k], mul2(z[k], both(a.skip)));
                z[k] = mul2(add2(z[k], both(-st.z)), both(st.w));
                u[k] = mul2(g[k], bw[k]);
                s1 = fma2(u[k], z[k], s1);
            }
            const bool layer = a.before == LUTB_NORM_LAYER;
            const float2 c = row_sums(p, s1.x + s1.y, layer ? total(u) : 0.0f, layer, [&]() {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (on) {
                        sums[2][k] = fma2(g[k], z[k], sums[2][k]);
                        sums[3][k] = add2(sums[3][k], g[k]);
                    }
                }
            });
            const float c1 = -c.x / width, c2 = layer ? -c.y / width : 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) d[k] = fma2(both(st.w), fma2(z[k], both(c1), add2(u[k], both(c2))), d[k]);
        }
        if (a.dx && on) {
            float2 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = BRANCH ? mul2(d[k], both(a.skip)) : d[k];
            store_row<X, VEC>(p, static_cast<X *>(a.dx) + at, o);
        }
        if (BRANCH) {
            if (gate_each && a.dgate && on) {
                float2 o[4];
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = mul2(mul2(d[k], both(a.branch)), n[k]);
                if (a.gate_f32)
                    store_row<float, VEC>(p, static_cast<float *>(a.dgate) + at, o);
                else
                    store_row<F, VEC>(p, static_cast<F *>(a.dgate) + at, o);
            }
            if (gate_summed && on) {
#pragma unroll
                for (int k = 0; k < 4; k++) sums[4][k] = fma2(d[k], n[k], sums[4][k]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) d[k] = mul2(d[k], gate[k]);
            if (BRANCH == 2) {
                float2 v[4], s1 = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[k] = mul2(d[k], w[k]);
                    if (!VEC) {
                        v[k].x = (p.valid >> (2 * k) & 1) ? v[k].x : 0.0f;
                        v[k].y = (p.valid >> (2 * k) & 2) ? v[k].y : 0.0f;
                    }
                    s1 = fma2(v[k], t[k], s1);
                }
                const bool layer = a.after == LUTB_NORM_LAYER, here_too = VEC ? p.valid != 0 : true;
                const float2 c = row_sums(p, here_too ? s1.x + s1.y : 0.0f, layer && here_too ? total(v) : 0.0f, layer, [&]() {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (on) {
                            sums[0][k] = fma2(d[k], t[k], sums[0][k]);
                            sums[1][k] = add2(sums[1][k], d[k]);
                        }
                    }
                });
                const float c1 = -c.x / width, c2 = layer ? -c.y / width : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) d[k] = mul2(both(st.y), fma2(t[k], both(c1), add2(v[k], both(c2))));
            }
            if (a.df && on) {
                if (a.drop.on) drop8(d, kept, a.drop.scale);
                store_row<F, VEC>(p, static_cast<F *>(a.df) + at, d);
            }
        }
        here.next(a, p.teams, stride);
        if (gate_summed && here.chunk != chunk) {   // (the same for the whole block)
            const int64_t out = (a.gate_direct ? chunk / a.per_group : chunk) * a.width;
            hand_out(sums[4], [&](int64_t c, float v) {
                v *= a.branch;
                if (!a.gate_direct)
                    a.gate_sums[out + c] = v;
                else if (a.gate_f32)
                    static_cast<float *>(a.dgate)[out + c] = v;
                else
                    static_cast<F *>(a.dgate)[out + c] = from_f32<F>(v);
            });
            zero8(sums[4]);
        }
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
        if ((s < 2 ? BRANCH == 2 : NEXT) && a.sums[s]) {
            float *to = a.sums[s] + own * a.width;
            hand_out(sums[s], [&](int64_t c, float v) { to[c] = v; });
        }
    }
}

// ------------------------------------------------------------------------------------------------ launches
int launch_rows(const void *kernel, std::atomic<uint32_t> &opted, const JoinArgs &a, const RowShape &s, int clusters, size_t smem, cudaStream_t stream);

template <class X, class F, bool VEC>
int launch_join_rows(bool backward, const JoinArgs &a, const RowShape &s, int clusters, cudaStream_t stream) {
    static std::atomic<uint32_t> opted[2][6];
    const int kind = (a.f == nullptr ? 0 : a.after == LUTB_NORM_NONE ? 1 : 2) * 2 + (backward ? a.dy != nullptr : a.y != nullptr);
    const void *kernel = nullptr;
#define LUTB_KIND(B, N)                                                                                      \
    case 2 * B + N:                                                                                          \
        kernel = backward ? reinterpret_cast<const void *>(&join_rows_backward_kernel<X, F, B, N != 0, VEC>) \
                          : reinterpret_cast<const void *>(&join_rows_forward_kernel<X, F, B, N != 0, VEC>); \
        break;
    switch (kind) {
        LUTB_KIND(0, 1)
        LUTB_KIND(1, 0)
        LUTB_KIND(1, 1)
        LUTB_KIND(2, 0)
        LUTB_KIND(2, 1)
    }
#undef LUTB_KIND
    LUTB_REQUIRE(kernel != nullptr, LUTB_ERR_MODE, "nothing to compute");
    const int gate = a.f != nullptr && a.gate_rows == 1 ? 2 : 0;
    size_t parts = backward ? 2 * kBackwardParams : 0;
    if (VEC) parts += backward ? (kBackwardParts<X, F> + gate) * kBackwardStages<X, F> : (kForwardParts<X, F> + gate) * kForwardStages;
    return launch_rows(kernel, opted[backward][kind], a, s, clusters, parts * 16 * s.threads, stream);
}

// defined for each pair of types in a file of its own
#define LUTB_JOIN_ROWS(X, F)                                                                                                              \
    template <>                                                                                                                           \
    int join_rows<X, F>(bool backward, bool vec, const JoinArgs &a, const RowShape &s, int clusters, cudaStream_t stream) {                \
        return vec ? launch_join_rows<X, F, true>(backward, a, s, clusters, stream) : launch_join_rows<X, F, false>(backward, a, s, clusters, stream); \
    }
template <class X, class F>
int join_rows(bool backward, bool vec, const JoinArgs &a, const RowShape &s, int clusters, cudaStream_t stream);

}  // namespace lutb
