// Row kernels of the residual joins: a row's elements stay in registers from the first sum to the last store.
//
// A thread has groups of eight elements of a row.  A team of threads has a row: a warp or a part of one up to 1024 elements (backward 256), a block up
// to 8192 (4096), beyond a cluster of two (or four) blocks; sums over a row go through shuffles, shared memory and the cluster's shared
// memory accordingly, one exchange for each norm and direction (a norm's mean and squares are combined from the warps' own by the pairwise
// formula of Chan, Golub and LeVeque, 1979, so that no square is taken about a mean that is far off).  What a team does depends on the
// width and the arrays' alignment alone, so that a row's result does not depend on the rows beside it.
//
// The next rows are fetched into shared memory with 16-byte asynchronous copies.  Rows of a multiple of eight elements in aligned arrays (VEC): a
// group is eight neighbours, a warp fetches what its threads will read (no barrier of the block), and one generator block decides a group's
// mask.  Other rows: the team fetches the aligned 16-byte pieces that its row touches, a thread's elements are a team apart, so that a
// warp reads and stores neighbours, and the mask's bytes go through shared memory too.
//
// Bound: the memory at 4-byte types (32768 x 1024 fp32 with both norms, gate and dropout: forward 93 us, 5.8 TB/s, backward 145 us, 5.6 TB/s),
// latency at 2-byte ones, whose instructions are nearly as many for half the bytes (bf16: 68 us, 3.9 TB/s, and 126 us, 3.2 TB/s: some 290
// for a warp's 256 elements forward and 560 backward, 110 of them the generator and its mask; the 16 warps an SM that registers allow issue
// 2.1 to 2.3 a cycle of the four that an SM can, waiting for loads, shared memory and results of fixed latency).
#pragma once

#include <atomic>

#include "mbarrier.cuh"
#include "residual_join.cuh"

namespace lutb {

constexpr int kRowElems = 8;
constexpr int kBlockThreads = 256, kWideThreads = 512;   // of a team; a warp's teams share a block of 128 forward, 256 backward
constexpr int kForwardCluster = 2, kBackwardCluster = 4;
constexpr int64_t kRowMaxWidth = 16384;   // such clusters of 512 threads, of two groups forward and one backward, or 512 threads of four
constexpr int64_t kRowMaxRows = 1 << 30;  // (row numbers of 32 bits)

// BLOCK and WIDE: a block of up to 256 or 512 threads.  BLOCKS: WIDE or CLUSTER, told at run time (backward, rows that are not VEC).
enum RowTeam { TEAM_WARP = 0, TEAM_BLOCK = 1, TEAM_WIDE = 2, TEAM_CLUSTER = 3, TEAM_BLOCKS = 4 };

struct RowShape {
    int groups;                 // of a thread
    int team, teams, threads;   // threads of a row in a block, rows a block has at a time, threads of a block
    int cluster, slice;         // blocks of a row, columns of a block
    int kind;                   // RowTeam
    int pad;                    // bytes between the places of two stages of a warp
    int stages;                 // rows whose elements a thread has room for in shared memory: this one and those that are fetched
};
inline void shape_team(RowShape &s, int64_t width, int block) {
    const int64_t each = (int64_t)s.groups * kRowElems;
    const int t = (int)(((width + each - 1) / each + s.cluster - 1) / s.cluster);
    s.slice = (int)(t * each);
    if (t <= 32) {
        s.team = 1;
        while (s.team < t) s.team *= 2;
        s.threads = block;
        s.teams = s.threads / s.team;
        s.kind = TEAM_WARP;
    } else {
        s.team = s.threads = (t + 31) / 32 * 32;
        s.teams = 1;
        s.kind = s.cluster > 1 ? TEAM_CLUSTER : s.threads > kBlockThreads ? TEAM_WIDE : TEAM_BLOCK;
    }
}
// Forward.  VEC: up to 256 elements one group a thread, up to 1024 four, always within a warp, with the parameters read for each row (20 KB at most, which
// stay in L1); beyond, two groups with the parameters in registers and slots of shared memory: read again for each row they came from L2, 20 bytes an element
// against the rows' own 8 at 16 bits (12288 x 8192 bf16 with all of them: 313 us so, 267 held; over a cluster of two blocks of 256 threads
// instead of one block of 512: 412).  Rows that are not VEC have one group up to
// 2048, where a warp's loads cover more neighbours.
inline RowShape forward_shape(int64_t width, bool vec) {
    RowShape s{};
    s.cluster = 1;
    s.groups = vec ? (width <= 256 ? 1 : width <= 1024 ? 4 : 2) : width <= 2048 ? 1 : 4;
    if (vec)
        while (width > (int64_t)s.cluster * 2 * kRowElems * kWideThreads) s.cluster *= 2;
    shape_team(s, width, 128);
    return s;
}
// Backward: one group, whose five sums over the rows take forty registers, a block of up to 512 threads (16384 x 4096 bf16 268 us, two blocks of 256 as a
// cluster 325).  Stages of a block's or cluster's rows 16 bytes apart measured faster
// than end to end (32768 x 1024 fp32 145 against 165 us, 12288 x 8192 bf16 558 against 575), those of a warp's rows did not (65536 x 256: 78 against
// 75), nor did the forward pass's.
inline RowShape backward_shape(int64_t width) {
    RowShape s{};
    s.cluster = s.groups = 1;
    while (width > (int64_t)s.cluster * kRowElems * kWideThreads) s.cluster *= 2;
    shape_team(s, width, 256);
    s.pad = s.kind == TEAM_WARP ? 0 : 16;
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
__device__ __forceinline__ void zero8(float2 *v) {
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = make_float2(0.0f, 0.0f);
}
__device__ __forceinline__ void drop8(float2 *v, uint32_t kept, float scale) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = mul2(v[k], both(scale));
        v[k].x = (kept >> (2 * k) & 1) ? v[k].x : 0.0f;
        v[k].y = (kept >> (2 * k) & 2) ? v[k].y : 0.0f;
    }
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
    if constexpr (sizeof(T) == 4) {   // (one store of a whole 32-byte sector; two of 16 bytes would each take half of every sector)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y),
                     "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y)
                     : "memory");
    } else {
        *reinterpret_cast<uint4 *>(p) = make_uint4(word_of(v[0], T()), word_of(v[1], T()), word_of(v[2], T()), word_of(v[3], T()));
    }
}
__device__ __forceinline__ void copy16(uint32_t to, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }

__device__ __forceinline__ void drop8(float2 *v, const DropDigits &d, float scale) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = mul2(v[k], both(scale));
        v[k].x = (d.w[k] << 16) > d.above ? v[k].x : 0.0f;
        v[k].y = d.w[k] > d.above ? v[k].y : 0.0f;
    }
}
// ------------------------------------------------------------------------------------------------ a thread's place
// Values that warps exchange: of two numbers each, two sets in turn (a set is written again only after the barrier of the next one, which a
// thread reaches when it has read this one).
template <int WARPS, int CLUSTER>
struct RowSlots {
    static constexpr int kWarps = WARPS;
    float a[2][WARPS * CLUSTER], b[2][WARPS * CLUSTER];
    float count[WARPS * CLUSTER];   // elements of the warps
    uint64_t arrived[2];   // clusters: all blocks' values of a set have come
};

struct RowPlace {
    int t, team, teams, which;   // thread in its team; threads of a team, teams, this one
    int cluster, rank;
    int first, limit;            // the block's columns: first .. limit - 1
    uint32_t valid;              // which elements exist: a bit a group (VEC) or an element
    uint32_t turn;               // exchanges so far
    float width, inverse;        // of a row, in elements
    bool waits;                  // false after a wait that ran out
};

// Column k of group g.
template <bool VEC>
__device__ __forceinline__ int row_column(const RowPlace &p, int g, int k) {
    return VEC ? p.first + (g * p.team + p.t) * 8 + k : p.first + p.t + (g * 8 + k) * p.team;
}
template <bool VEC>
__device__ __forceinline__ bool row_valid(const RowPlace &p, int g, int k) { return p.valid >> (VEC ? g : g * 8 + k) & 1; }

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// (no memory is handed over: nothing is waited for but the blocks themselves)
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait;" ::: "memory"); }

template <bool VEC, int G, int TEAM, class Slots>
__device__ __forceinline__ RowPlace row_place(const JoinArgs &a, const RowShape &s, Slots &slots) {
    RowPlace p;
    const int tid = threadIdx.x;
    p.team = s.team;
    p.teams = TEAM == TEAM_WARP ? s.teams : 1;
    p.which = TEAM == TEAM_WARP ? tid / s.team : 0;
    p.t = tid - p.which * s.team;
    p.cluster = TEAM == TEAM_CLUSTER || TEAM == TEAM_BLOCKS ? s.cluster : 1;
    p.rank = p.cluster > 1 ? (int)(blockIdx.x % p.cluster) : 0;
    p.first = p.rank * s.slice;
    p.limit = (int)min((int64_t)p.first + s.slice, a.width);
    p.width = (float)a.width;
    p.inverse = 1.0f / p.width;
    p.turn = 0;
    p.waits = true;
    p.valid = 0;
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (VEC) {
            if (row_column<VEC>(p, g, 0) < p.limit) p.valid |= 1u << g;
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (row_column<VEC>(p, g, k) < p.limit) p.valid |= 1u << (g * 8 + k);
        }
    }
    if (TEAM != TEAM_WARP) {
        constexpr int kAll = sizeof(slots.a[0]) / sizeof(float), kWarps = Slots::kWarps;
        for (int k = tid; k < kAll; k += blockDim.x) slots.a[0][k] = slots.a[1][k] = slots.b[0][k] = slots.b[1][k] = 0.0f;
        constexpr int kCounts = sizeof(slots.count) / sizeof(float);
        for (int k = tid; k < kCounts; k += blockDim.x) {   // elements of the row's warps, other blocks' too (VEC: their groups' 256 columns)
            const int rank = k / kWarps, warp = k - rank * kWarps, end = (int)min((int64_t)(rank + 1) * s.slice, a.width);
            int n = 0;
            if (rank < p.cluster && warp < (s.team >> 5)) {
#pragma unroll
                for (int g = 0; g < (VEC ? G : 8 * G); g++) {
                    const int step = VEC ? 8 : 1, begin = rank * s.slice + (g * s.team + warp * 32) * step;
                    n += max(0, min(end - begin, 32 * step));
                }
            }
            slots.count[k] = (float)n;
        }
        __syncthreads();
        if (p.cluster > 1) {
            if (tid == 0) {
                mbar_init(smem_u32(&slots.arrived[0]), 1);
                mbar_init(smem_u32(&slots.arrived[1]), 1);
                fence_barrier_init();
            }
            cluster_sync();   // the row's blocks are there and ready
        } else {
            __syncthreads();
        }
    }
    return p;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float team_sum(float v, int team) {   // teams of a warp or a part of one
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, v, o);
        v += o < team ? other : 0.0f;
    }
    return v;
}
// Both sums over the warp: one exchange sends each half of the lanes its value, the others add one value a lane; all lanes have both in the end.
__device__ __forceinline__ void warp_sums(float &a, float &b) {
    const bool upper = threadIdx.x & 16;
    float v = upper ? b : a;
    v += __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const float other = __shfl_xor_sync(0xffffffffu, v, 16);
    a = upper ? other : v;
    b = upper ? v : other;
}
template <int TEAM>
__device__ __forceinline__ bool over_cluster(const RowPlace &p) { return TEAM == TEAM_CLUSTER || (TEAM == TEAM_BLOCKS && p.cluster > 1); }

static __device__ int g_join_wait_errors;   // bounded waits that ran out (lutb_device_wait_errors)

// Every warp's two values to every warp of the row.  A cluster's blocks store them into each other's slots asynchronously, with the arrival
// counted on the receiver's barrier: a cluster-wide barrier would also wait for this block's stores of results to global memory
// (measured: 5 us a row).  A wait that runs out is counted, and later ones are not begun.
template <int TEAM, class Slots>
__device__ __forceinline__ void publish(const RowPlace &p, Slots &slots, float a, float b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, set = p.turn & 1;
    if (!over_cluster<TEAM>(p)) {
        if (lane == 0) {
            slots.a[set][warp] = a;
            slots.b[set][warp] = b;
        }
        return;
    }
    const int warps = p.team >> 5;
    if (threadIdx.x == 0) mbar_arrive_expect_tx(smem_u32(&slots.arrived[set]), (uint32_t)(8 * warps * p.cluster));
    if (lane < p.cluster) {
        const int at = p.rank * Slots::kWarps + warp;
        uint32_t to_a = smem_u32(&slots.a[set][at]), to_b = smem_u32(&slots.b[set][at]), bar = smem_u32(&slots.arrived[set]);
        asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(to_a) : "r"(lane));
        asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(to_b) : "r"(lane));
        asm("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(bar) : "r"(lane));
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to_a), "r"(__float_as_uint(a)), "r"(bar) : "memory");
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to_b), "r"(__float_as_uint(b)), "r"(bar) : "memory");
    }
}
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
template <int TEAM, class Slots>
__device__ __forceinline__ void collect(RowPlace &p, Slots &slots) {
    if (!over_cluster<TEAM>(p)) {
        __syncthreads();
        return;
    }
    const uint32_t bar = smem_u32(&slots.arrived[p.turn & 1]), parity = p.turn >> 1 & 1;
    if (!p.waits || arrived(bar, parity)) return;
    const long long t0 = clock64();
    while (!arrived(bar, parity)) {
        if (clock64() - t0 > kWaitLimitCycles) {
            if (threadIdx.x == 0) atomicAdd(&g_join_wait_errors, 1);
            p.waits = false;
            return;
        }
    }
}
// Sums over each N neighbouring lanes, in all of them.
template <int N>
__device__ __forceinline__ float lane_sums(float v) {
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The sum of a set of slots, always in the same order.
template <int N>
__device__ __forceinline__ float slot_sum(const float *from) {
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < N; k += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(from + k);
        s = add2(s, add2(make_float2(v.x, v.y), make_float2(v.z, v.w)));
    }
    return s.x + s.y;
}
template <int TEAM, class Slots>
__device__ __forceinline__ float all_slots(const RowPlace &p, const float *from) {
    constexpr int kWarps = Slots::kWarps;
    if (!over_cluster<TEAM>(p)) return slot_sum<kWarps>(from);
    const int lane = threadIdx.x & 31, n = p.cluster * kWarps;   // 16, 32 or 64 slots, one or two a lane
    float v = lane < n ? from[lane] : 0.0f;
    if (n > 32) v += from[lane + 32];
    return warp_sum(v);
}
// Sums of two values over the row; `between` runs while the others arrive.
template <int TEAM, class Slots, class Fn>
__device__ __forceinline__ float2 row_sums(RowPlace &p, Slots &slots, float a, float b, bool second, Fn between) {
    if (TEAM == TEAM_WARP) {
        a = team_sum(a, p.team);
        if (second) b = team_sum(b, p.team);
        between();
        return make_float2(a, b);
    }
    if (second)
        warp_sums(a, b);
    else
        a = warp_sum(a);
    publish<TEAM>(p, slots, a, b);
    between();
    collect<TEAM>(p, slots);
    const float *const sa = slots.a[p.turn & 1], *const sb = slots.b[p.turn & 1];
    constexpr int kWarps = Slots::kWarps;
    const int lane = threadIdx.x & 31;
    p.turn++;
    if (over_cluster<TEAM>(p) && second) {   // the slots' values over the lanes, then as before
        const int n = p.cluster * kWarps;    // 16, 32 or 64 slots, one or two a lane
        a = lane < n ? sa[lane] : 0.0f;
        b = lane < n ? sb[lane] : 0.0f;
        if (n > 32) {
            a += sa[lane + 32];
            b += sb[lane + 32];
        }
        warp_sums(a, b);
        return make_float2(a, b);
    }
    if (!over_cluster<TEAM>(p) && second) {   // a slot a lane: the first values, then the second ones
        const float v = lane_sums<kWarps>((lane & kWarps ? sb : sa)[lane & (kWarps - 1)]);
        return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, kWarps));
    }
    return make_float2(all_slots<TEAM, Slots>(p, sa), second ? all_slots<TEAM, Slots>(p, sb) : 0.0f);
}
// Mean (0 for an RMS norm) and reciprocal deviation of the row's values.  Values of no element do not count (in rows that are not VEC
// they are 0).
template <bool VEC, int G, int TEAM, class Slots>
__device__ __forceinline__ float2 row_stats(RowPlace &p, Slots &slots, const float2 (*v)[4], bool layer, float eps) {
    auto sum = [&]() {
        float s = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float one = total(v[g]);
            s += !VEC || row_valid<VEC>(p, g, 0) ? one : 0.0f;
        }
        return s;
    };
    auto squares = [&](float mean) {
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < G; g++) {
            float2 q = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float2 d = add2(v[g][k], both(-mean));
                if (!VEC) {
                    d.x = row_valid<VEC>(p, g, 2 * k) ? d.x : 0.0f;
                    d.y = row_valid<VEC>(p, g, 2 * k + 1) ? d.y : 0.0f;
                }
                q = fma2(d, d, q);
            }
            if (VEC) {
                q.x = row_valid<VEC>(p, g, 0) ? q.x : 0.0f;
                q.y = row_valid<VEC>(p, g, 0) ? q.y : 0.0f;
            }
            s = add2(s, q);
        }
        return s.x + s.y;
    };
    if (TEAM == TEAM_WARP) {
        const float mean = layer ? team_sum(sum(), p.team) / p.width : 0.0f;
        return make_float2(mean, rsqrtf(team_sum(squares(mean), p.team) * p.inverse + eps));
    }
    const int set = p.turn & 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = Slots::kWarps;
    float mean = 0.0f, s;
    if (layer) {
        const float count = slots.count[p.rank * kWarps + warp];
        mean = count > 0.0f ? warp_sum(sum()) / count : 0.0f;
    }
    publish<TEAM>(p, slots, warp_sum(squares(mean)), mean);
    collect<TEAM>(p, slots);
    mean = 0.0f;
    if (over_cluster<TEAM>(p)) {   // the row's warps over the lanes, 16 or 32 of them
        static_assert(TEAM != TEAM_CLUSTER || sizeof(slots.a[0]) <= 32 * sizeof(float), "a slot a lane");
        const bool some = lane < p.cluster * kWarps;
        s = some ? slots.a[set][lane] : 0.0f;
        if (layer) {
            const float m = some ? slots.b[set][lane] : 0.0f, n = some ? slots.count[lane] : 0.0f;
            mean = warp_sum(m * n) / p.width;
            s = fmaf(n * (m - mean), m - mean, s);
        }
        s = warp_sum(s);
    } else if (layer) {   // a slot a lane (all threads going through them took three times the instructions)
        const int w = lane & (kWarps - 1);
        const float m = slots.b[set][w], n = slots.count[w];
        mean = lane_sums<kWarps>(m * n) / p.width;
        s = lane_sums<kWarps>(fmaf(n * (m - mean), m - mean, slots.a[set][w]));
    } else {
        s = slot_sum<kWarps>(slots.a[set]);
    }
    p.turn++;
    return make_float2(mean, rsqrtf(s * p.inverse + eps));
}

// Eight of a parameter's values.  VEC: a group beyond the row reads another one's; else values of no element are 0.
template <class F, bool VEC>
__device__ __forceinline__ void param8(const RowPlace &p, int g, const void *from, bool f32, int64_t at, float2 *v) {
    if constexpr (VEC) {
        const int64_t c = at + min(row_column<VEC>(p, g, 0), p.limit - 8);
        if (sizeof(F) == 4 || f32) {
            const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(from) + c);
            const uint4 part[2] = {__ldg(q), __ldg(q + 1)};
            unpack8<float>(part, v);
        } else {
            const uint4 part[1] = {__ldg(reinterpret_cast<const uint4 *>(static_cast<const F *>(from) + c))};
            unpack8<F>(part, v);
        }
    } else {
        float e[8];
        int64_t c = at + row_column<VEC>(p, g, 0);
#pragma unroll
        for (int k = 0; k < 8; k++, c += p.team) {
            e[k] = 0.0f;
            if (row_valid<VEC>(p, g, k)) e[k] = sizeof(F) == 4 || f32 ? static_cast<const float *>(from)[c] : to_f32(static_cast<const F *>(from)[c]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
    }
}
// v = v w + b, for what there is of them (one test for all groups).
template <class F, bool VEC, int G>
__device__ __forceinline__ void affine(const RowPlace &p, const void *weight, const void *bias, bool f32, float2 (*v)[4]) {
    auto each = [&](bool of_f32) {
        if (weight != nullptr) {
#pragma unroll
            for (int g = 0; g < G; g++) {
                float2 w[4];
                param8<F, VEC>(p, g, weight, of_f32, 0, w);
#pragma unroll
                for (int k = 0; k < 4; k++) v[g][k] = mul2(v[g][k], w[k]);
            }
        }
        if (bias != nullptr) {
#pragma unroll
            for (int g = 0; g < G; g++) {
                float2 b[4];
                param8<F, VEC>(p, g, bias, of_f32, 0, b);
#pragma unroll
                for (int k = 0; k < 4; k++) v[g][k] = add2(v[g][k], b[k]);
            }
        }
    };
    if (sizeof(F) == 4 || f32)
        each(true);
    else
        each(false);
}

// The rows of a block in turn: chunk by chunk, `teams` rows at a time.
struct RowCursor {
    int chunk, base, end;
    __device__ __forceinline__ void enter(const JoinArgs &a) {
        if (chunk >= (int)a.chunks) return;
        const int per = (int)a.per_group, group = chunk / per, rows = (int)a.group_rows;
        base = group * rows + (chunk - group * per) * (int)a.chunk_rows;
        end = min(base + (int)a.chunk_rows, (group + 1) * rows);
    }
    __device__ __forceinline__ bool more(const JoinArgs &a) const { return chunk < (int)a.chunks; }
    __device__ __forceinline__ void next(const JoinArgs &a, int teams, int stride) {
        base += teams;
        if (base >= end) {
            chunk += stride;
            enter(a);
        }
    }
};

template <int TEAM>
__device__ __forceinline__ void team_barrier() {
    if (TEAM == TEAM_WARP)
        __syncwarp();
    else
        __syncthreads();
}

// Bytes of the next rows' elements of one array in a stage.  Rows that are not VEC: a place of 32 bytes more than a row's for each team, for the aligned
// pieces at its two ends.
__host__ __device__ inline int ring_row_bytes(int slice, int size) { return (slice * size + 15) / 16 * 16 + 32; }
__host__ __device__ inline int ring_bytes(bool vec, const RowShape &s, int size) {
    return vec ? s.groups * kRowElems * size * s.threads : s.teams * ring_row_bytes(s.slice, size);
}

// The current row and those that are fetched.  With one stage a row is fetched when its turn comes, else one or two rows ahead.  The current row can be
// read to the end of its turn.
//
// VEC: a warp has a place of its own, [stage][array][group][piece], in which arrays and groups begin at constants (AT, in parts of 512 bytes).  A
// warp's (or a smaller team's) 16-byte pieces of a group go side by side over its threads; those of 4-byte elements are two a
// thread, swapped in every other four pairs, so that the threads' reads of their two pieces meet no bank twice.
template <bool VEC, int G, int TEAM>
struct RowRing {
    unsigned char *at;          // VEC: this warp's place, else the block's
    int stage_bytes, stages, fill, take;   // VEC: of this warp; fill and take count bytes
    int u, wide;                // VEC: thread among those that share pieces, how many they are
    int mine, swapped;          // VEC: this thread's own pieces (in bytes, for one part), and whether its two are swapped

    __device__ __forceinline__ RowRing(unsigned char *memory, const RowPlace &p, int bytes_of_block, int n) : at(memory), stages(n), fill(0), take(0) {
        stage_bytes = bytes_of_block;
        if (VEC) {
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            stage_bytes = bytes_of_block / (int)(blockDim.x >> 5);
            at = memory + warp * n * stage_bytes;
            wide = min(p.team, 32);
            u = lane & (wide - 1);
            mine = (lane - u) * 16;
            swapped = u >> 2 & 1;
        }
    }
    // What this thread fetches of a row of one array.  VEC: pieces that the row does not have are another one's.
    template <class T, int AT>
    __device__ __forceinline__ void fetch(const RowPlace &p, const RowShape &s, int part, const T *from, int64_t row, bool some, const JoinArgs &a) const {
        constexpr int kEach = 16 / sizeof(T);
        if constexpr (VEC) {
            const T *const begin = from + row * a.width;
            const uint32_t to = smem_u32(at) + fill + AT * 512 + mine * kParts<T>;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int q = 0; q < kParts<T>; q++) {
                    const int c = q * wide + u, column = p.first + (g * p.team + p.t - u) * 8 + c * kEach;
                    copy16(to + g * kParts<T> * 512 + (kParts<T> == 2 ? c ^ (c >> 3 & 1) : c) * 16, begin + min(column, p.limit - kEach));
                }
        } else {
            if (!some) return;
            const int64_t begin = row * a.width + p.first, total = a.rows * a.width * (int64_t)sizeof(T);
            const int ahead = (int)(reinterpret_cast<uintptr_t>(from + begin) & 15);   // of the row in its first piece
            const int pieces = (ahead + (p.limit - p.first) * (int)sizeof(T) + 15) / 16;
            const int64_t offset = begin * (int64_t)sizeof(T) - ahead;   // of that piece, from the array's begin
            const unsigned char *const bytes = reinterpret_cast<const unsigned char *>(from) + offset;
            unsigned char *const place = at + fill + part + p.which * ring_row_bytes(s.slice, sizeof(T));
            if (offset >= 0 && offset + pieces * 16 <= total) {
                const uint32_t to = smem_u32(place);
                for (int c = p.t; c < pieces; c += p.team) copy16(to + c * 16, bytes + c * 16);
            } else {   // pieces that the array does not fill: their elements one by one
                for (int c = p.t; c < pieces; c += p.team) {
                    const int64_t o = offset + c * 16;
                    for (int e = 0; e < 16; e += (int)sizeof(T))
                        if (o + e >= 0 && o + e < total) *reinterpret_cast<T *>(place + c * 16 + e) = *reinterpret_cast<const T *>(bytes + c * 16 + e);
                }
            }
        }
    }
    __device__ __forceinline__ void filled() {
        asm volatile("cp.async.commit_group;" ::: "memory");
        fill = fill + stage_bytes == stages * stage_bytes ? 0 : fill + stage_bytes;
    }
    // The current row's elements are there, for the team; what was read of the row before may be overwritten.
    __device__ __forceinline__ void ready() const {
        if (stages == 3)
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        else
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (VEC)
            __syncwarp();
        else
            team_barrier<TEAM>();
    }
    __device__ __forceinline__ void taken() { take = take + stage_bytes == stages * stage_bytes ? 0 : take + stage_bytes; }
    // Eight elements; where there are none: 0, in VEC rows those of another group or row.
    template <class T, int AT>
    __device__ __forceinline__ void get(const RowPlace &p, const RowShape &s, int g, int part, const T *from, int64_t begin, bool on, float2 *v) const {
        if constexpr (VEC) {
            const uint4 *const own = reinterpret_cast<const uint4 *>(at + take + mine * kParts<T> + u * (kParts<T> * 16)) + (AT + g * kParts<T>)*32;
            uint4 w[kParts<T>];
            if constexpr (kParts<T> == 2) {
                w[0] = own[swapped];
                w[1] = own[1 - swapped];
            } else {
                w[0] = own[0];
            }
            unpack8<T>(w, v);
        } else {
            const unsigned char *const stage = at + take + part;
            const int ahead = (int)(reinterpret_cast<uintptr_t>(from + begin + p.first) & 15) / (int)sizeof(T);
            const T *own = reinterpret_cast<const T *>(stage + p.which * ring_row_bytes(s.slice, sizeof(T))) + ahead + p.t + g * 8 * p.team;
            const uint32_t valid = on ? p.valid : 0u;
            float e[8];
#pragma unroll
            for (int k = 0; k < 8; k++, own += p.team) {
                e[k] = 0.0f;
                if (valid >> (g * 8 + k) & 1) e[k] = to_f32(*own);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
        }
    }
};

template <class T, bool VEC>
__device__ __forceinline__ void store_row(const RowPlace &p, int g, T *row, const float2 *v) {   // (only where there is a row)
    if constexpr (VEC) {
        if (row_valid<VEC>(p, g, 0)) store8(row + row_column<VEC>(p, g, 0), v);
    } else {
        T *to = row + row_column<VEC>(p, g, 0);
#pragma unroll
        for (int k = 0; k < 8; k++, to += p.team)
            if (row_valid<VEC>(p, g, k)) *to = from_f32<T>(k & 1 ? v[k >> 1].y : v[k >> 1].x);
    }
}

// The masks of a thread's groups.  Rows that are not VEC: the team's generator blocks as bytes in shared memory, written before the row's barrier and
// read after it, two sets in turn.
template <int G>
__device__ __forceinline__ void form_masks(const RowPlace &p, const JoinArgs &a, const DropKey &key, int64_t row, uint8_t *bytes, uint32_t set) {
    const uint64_t block = (uint64_t)(row * a.width + p.first) >> 3;
    uint8_t *own = bytes + ((int)set * p.teams + p.which) * (G * p.team + 1);
#pragma unroll
    for (int g = 0; g < G; g++) own[g * p.team + p.t] = (uint8_t)keep_bits(block + g * p.team + p.t, key, a.drop);
    if (p.t == 0) own[G * p.team] = (uint8_t)keep_bits(block + G * p.team, key, a.drop);
}
template <int G>
__device__ __forceinline__ uint32_t read_masks(const RowPlace &p, const JoinArgs &a, int64_t row, const uint8_t *bytes, uint32_t set) {
    const uint8_t *own = bytes + ((int)set * p.teams + p.which) * (G * p.team + 1);
    int e = (int)((row * a.width + p.first) & 7) + p.t;
    uint32_t kept = 0;
#pragma unroll
    for (int k = 0; k < 8 * G; k++, e += p.team) kept |= ((uint32_t)own[e >> 3] >> (e & 7) & 1u) << k;
    return kept;
}
template <int G, int THREADS>
constexpr size_t kMaskBytes = 2 * (G * THREADS + THREADS);   // two sets, a byte a group and one more a team

// The kernels' own arrays at most (5456, 656, 9216 and 3344 bytes), and what a block takes beside them: what launches count with.
constexpr size_t kForwardStatic = 10 * 1024, kForwardVecStatic = 2 * 1024, kBackwardStatic = 13 * 1024, kBackwardTeamStatic = 4 * 1024;

// ------------------------------------------------------------------------------------------------ forward
// BRANCH: 0 no branch (the norm alone), 1 a branch, 2 a branch with a norm of its own.  NEXT: the norm before the next block.
// The parameters that a forward kernel keeps in shared memory.
__host__ __device__ inline int held_bytes(bool vec, const RowShape &s) {
    return (vec ? s.kind != TEAM_WARP : s.groups == 1) ? 2 * s.groups * kRowElems * 4 * s.threads : 0;
}
template <int G, int TEAM>
constexpr int kThreadsOf = TEAM == TEAM_WARP ? 128 : TEAM == TEAM_BLOCK ? kBlockThreads : kWideThreads;

// Blocks an SM: 512 threads of 128 registers, but three warps a scheduler of 168 where a thread has four groups and a branch (32768 x 1024 bf16 73
// against 69 us; fp32 the same).
template <int BRANCH, int G, int TEAM>
constexpr int kForwardBlocks = BRANCH && G == 4 && TEAM == TEAM_WARP ? 3 : 512 / kThreadsOf<G, TEAM>;

template <class X, class F, int BRANCH, bool NEXT, bool VEC, int G, int TEAM>
__global__ void __launch_bounds__(kThreadsOf<G, TEAM>, kForwardBlocks<BRANCH, G, TEAM>) join_rows_forward_kernel(const JoinArgs a, const RowShape shape) {
    constexpr int kThreads = kThreadsOf<G, TEAM>;
    constexpr bool kHeld = VEC ? TEAM != TEAM_WARP : G == 1;   // the parameters are kept
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ __align__(16) RowSlots<TEAM == TEAM_WARP ? 4 : kThreads / 32, TEAM == TEAM_CLUSTER ? kForwardCluster : 1> slots;
    __shared__ uint8_t masks[VEC ? 1 : kMaskBytes<G, kThreads>];
    static_assert(sizeof(slots) + sizeof(masks) <= (VEC ? kForwardVecStatic : kForwardStatic));
    RowPlace p = row_place<VEC, G, TEAM>(a, shape, slots);
    const DropKey key = BRANCH && a.drop.on ? drop_key(a.random, a.site) : DropKey{};
    const bool gate_each = BRANCH && a.gate_rows == 1, gate_f32 = sizeof(F) == 4 || a.gate_f32;
    constexpr bool sure = TEAM == TEAM_BLOCK || TEAM == TEAM_WIDE || TEAM == TEAM_CLUSTER;   // (a row in every turn)
    const int part_f = ring_bytes(VEC, shape, sizeof(X)), part_gate = part_f + (BRANCH ? ring_bytes(VEC, shape, sizeof(F)) : 0);
    constexpr int kF = G * kParts<X>, kGate = kF + (BRANCH ? G * kParts<F> : 0);
    RowRing<VEC, G, TEAM> ring(dynamic + held_bytes(VEC, shape), p, part_gate + (gate_each ? ring_bytes(VEC, shape, gate_f32 ? 4 : sizeof(F)) : 0), shape.stages);
    const X *const x_in = static_cast<const X *>(a.x);
    const F *const f_in = static_cast<const F *>(a.f);
    const int stride = gridDim.x / p.cluster;
    RowCursor load{(int)blockIdx.x / p.cluster, 0, 0}, here;
    load.enter(a);
    here = load;
    auto fetch = [&]() {
        if (load.more(a)) {
            const bool some = sure || load.base + p.which < load.end;
            const int64_t row = some ? load.base + p.which : load.end - 1;
            ring.template fetch<X, 0>(p, shape, 0, x_in, row, some, a);
            if (BRANCH) ring.template fetch<F, kF>(p, shape, part_f, f_in, row, some, a);
            if (gate_each) {
                if (gate_f32)
                    ring.template fetch<float, kGate>(p, shape, part_gate, static_cast<const float *>(a.gate), row, some, a);
                else
                    ring.template fetch<F, kGate>(p, shape, part_gate, static_cast<const F *>(a.gate), row, some, a);
            }
            load.next(a, p.teams, stride);
        }
        ring.filled();
    };
    for (int s = 1; s < shape.stages; s++) fetch();
    uint32_t set = 0;
    // Held: the norm after the block with the gate and the branch's scale in it, in registers; the norm before the next block in slots of this
    // thread's own, [warp][weight, bias][group][half][lane] (all of them in registers spilled).
    constexpr int H = kHeld ? G : 1;
    float2 aw[H][4], ab[H][4];
    float4 *const slot = reinterpret_cast<float4 *>(dynamic) + (threadIdx.x >> 5) * (4 * H * 32) + (threadIdx.x & 31);
    auto hold = [&](const void *from, bool f32, int64_t at, float none, float2 (*v)[4]) {
#pragma unroll
        for (int g = 0; g < H; g++) {
            if (from != nullptr) {
                param8<F, VEC>(p, g, from, f32, at, v[g]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) v[g][k] = both(none);
            }
        }
    };
    auto hold_branch = [&](int64_t gate_at) {
        if (BRANCH == 2) {
            hold(a.aw, a.params_f32, 0, 1.0f, aw);
            hold(a.ab, a.params_f32, 0, 0.0f, ab);
        } else {
            hold(nullptr, true, 0, 1.0f, aw);
        }
#pragma unroll
        for (int g = 0; g < H; g++) {
            float2 gate[4] = {both(1.0f), both(1.0f), both(1.0f), both(1.0f)};
            if (a.gate != nullptr && !gate_each) param8<F, VEC>(p, g, a.gate, gate_f32, gate_at, gate);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                gate[k] = mul2(gate[k], both(a.branch));
                aw[g][k] = mul2(aw[g][k], gate[k]);
                if (BRANCH == 2) ab[g][k] = mul2(ab[g][k], gate[k]);
            }
        }
    };
    if (kHeld) {
        if (BRANCH) hold_branch(0);
        if (NEXT) {
            float2 v[H][4];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                hold(n ? a.bb : a.bw, a.params_f32, 0, n ? 0.0f : 1.0f, v);
#pragma unroll
                for (int g = 0; g < H; g++) {
                    slot[((n * H + g) * 2) * 32] = make_float4(v[g][0].x, v[g][0].y, v[g][1].x, v[g][1].y);
                    slot[((n * H + g) * 2 + 1) * 32] = make_float4(v[g][2].x, v[g][2].y, v[g][3].x, v[g][3].y);
                }
            }
        }
    }
    int64_t gate_at = 0;   // the gate row in use
    int gate_end = 0;      // the first row of another one
    for (; here.more(a); here.next(a, p.teams, stride)) {
        const int row = here.base + p.which;
        const int64_t at = row * a.width;
        const bool on = sure || row < here.end;
        if (BRANCH && a.gate_rows > 1 && on && row >= gate_end) {
            const int gate_row = row / (int)a.gate_rows;
            gate_end = (gate_row + 1) * (int)a.gate_rows;
            gate_at = gate_row * a.width;
            if (kHeld) hold_branch(gate_at);
        }
        const bool drop = BRANCH && a.drop.on;
        if (!VEC && drop) form_masks<G>(p, a, key, row, masks, set);
        if (shape.stages == 1) {
            team_barrier<TEAM>();
            fetch();
        }
        ring.ready();
        uint32_t kept = 0;
        if (!VEC && drop) kept = read_masks<G>(p, a, row, masks, set);
        set ^= 1;
        if (shape.stages > 1) fetch();
        float2 v[G][4];
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (BRANCH) {
#pragma unroll
            for (int g = 0; g < G; g++) ring.template get<F, kF>(p, shape, g, part_f, f_in, at, on, v[g]);
            if (drop) {
                const uint64_t block = (uint64_t)(at + p.first) >> 3;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    if (VEC)
                        drop8(v[g], drop_digits(block + g * p.team + p.t, key, a.drop), a.drop.scale);
                    else
                        drop8(v[g], kept >> (8 * g), a.drop.scale);
                }
            }
        }
        if (BRANCH == 2) {
            const float2 s = row_stats<VEC, G, TEAM>(p, slots, v, a.after == LUTB_NORM_LAYER, a.eps);
            st.x = s.x;
            st.y = s.y;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < 4; k++) v[g][k] = mul2(add2(v[g][k], both(-s.x)), both(s.y));
            if (!kHeld) affine<F, VEC, G>(p, a.aw, a.ab, a.params_f32, v);
        }
        if (kHeld && BRANCH) {
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < 4; k++) v[g][k] = BRANCH == 2 ? fma2(v[g][k], aw[g % H][k], ab[g % H][k]) : mul2(v[g][k], aw[g % H][k]);
        }
        if (BRANCH) {
            auto gated = [&](auto get) {
#pragma unroll
                for (int g = 0; g < G; g++) {
                    float2 gate[4];
                    get(g, gate);
#pragma unroll
                    for (int k = 0; k < 4; k++) v[g][k] = mul2(v[g][k], gate[k]);
                }
            };
            if (gate_each) {
                if (gate_f32)
                    gated([&](int g, float2 *e) { ring.template get<float, kGate>(p, shape, g, part_gate, static_cast<const float *>(a.gate), at, on, e); });
                else
                    gated([&](int g, float2 *e) { ring.template get<F, kGate>(p, shape, g, part_gate, static_cast<const F *>(a.gate), at, on, e); });
            } else if (!kHeld && a.gate != nullptr) {
                if (gate_f32)
                    gated([&](int g, float2 *e) { param8<F, VEC>(p, g, a.gate, true, gate_at, e); });
                else
                    gated([&](int g, float2 *e) { param8<F, VEC>(p, g, a.gate, false, gate_at, e); });
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            float2 x[4];
            ring.template get<X, 0>(p, shape, g, 0, x_in, at, on, x);
#pragma unroll
            for (int k = 0; k < 4; k++)
                v[g][k] = !BRANCH ? x[k] : kHeld ? fma2(x[k], both(a.skip), v[g][k]) : fma2(v[g][k], both(a.branch), mul2(x[k], both(a.skip)));
            if (!VEC && BRANCH) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[g][k].x = row_valid<VEC>(p, g, 2 * k) ? v[g][k].x : 0.0f;
                    v[g][k].y = row_valid<VEC>(p, g, 2 * k + 1) ? v[g][k].y : 0.0f;
                }
            }
            if (BRANCH && on) store_row<X, VEC>(p, g, static_cast<X *>(a.h) + at, v[g]);
        }
        if (NEXT) {
            const float2 s = row_stats<VEC, G, TEAM>(p, slots, v, a.before == LUTB_NORM_LAYER, a.eps);
            st.z = s.x;
            st.w = s.y;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < 4; k++) v[g][k] = mul2(add2(v[g][k], both(-s.x)), both(s.y));
            if (kHeld) {
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const float4 w = slot[((g % H) * 2 + half) * 32], b = slot[((H + g % H) * 2 + half) * 32];
                        v[g][2 * half] = fma2(v[g][2 * half], make_float2(w.x, w.y), make_float2(b.x, b.y));
                        v[g][2 * half + 1] = fma2(v[g][2 * half + 1], make_float2(w.z, w.w), make_float2(b.z, b.w));
                    }
            }
            if (!kHeld) affine<F, VEC, G>(p, a.bw, a.bb, a.params_f32, v);
            if (on)
#pragma unroll
                for (int g = 0; g < G; g++) store_row<F, VEC>(p, g, static_cast<F *>(a.y) + at, v[g]);
        }
        if (a.stats && on && p.t == 0 && p.rank == 0) a.stats[row] = st;
        ring.taken();
    }
    if (over_cluster<TEAM>(p)) cluster_meet();   // (no block is gone while another may store into it)
}

// ------------------------------------------------------------------------------------------------ backward
constexpr int kBackwardParams = 4;   // aw, ab, bw, gate

// See join_backward_kernel for the formulas.  A thread's sums over its rows stay in registers to the end (of the chunk, for a gate row); what a step
// needs of the row is read from shared memory at that step, so that three sets of eight values are live at most beside the forty sums.
template <int TEAM>
constexpr int kBackwardThreads = TEAM == TEAM_WARP || TEAM == TEAM_BLOCK ? kBlockThreads : kWideThreads;

template <class X, class F, int BRANCH, bool NEXT, bool VEC, int TEAM>
__global__ void __launch_bounds__(kBackwardThreads<TEAM>, 512 / kBackwardThreads<TEAM>) join_rows_backward_kernel(const JoinArgs a, const RowShape shape) {
    constexpr int kThreads = kBackwardThreads<TEAM>;
    constexpr bool kTeams = TEAM == TEAM_WARP, kClusters = TEAM == TEAM_CLUSTER || TEAM == TEAM_BLOCKS;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ __align__(16) RowSlots<kThreads / 32, kClusters ? kBackwardCluster : 1> slots;
    __shared__ uint8_t masks[VEC ? 1 : kMaskBytes<1, kThreads>];
    __shared__ float2 joined[kTeams ? 4 * kBlockThreads : 1];   // the teams' sums of a block
    static_assert(sizeof(slots) + sizeof(masks) + sizeof(joined) <= (TEAM == TEAM_WARP ? kBackwardStatic : kBackwardTeamStatic));
    RowPlace p = row_place<VEC, 1, TEAM>(a, shape, slots);
    const int threads = blockDim.x, tid = threadIdx.x;
    const DropKey key = BRANCH && a.drop.on ? drop_key(a.random, a.site) : DropKey{};
    // parameters in slots of this thread's own: [warp][parameter][half][lane]
    float4 *const params = reinterpret_cast<float4 *>(dynamic) + (tid >> 5) * (2 * kBackwardParams * 32) + (tid & 31);
    auto keep = [&](int which, const float2 *v) {
        params[(2 * which) * 32] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        params[(2 * which + 1) * 32] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    };
    auto keep_param = [&](int which, const void *from, bool f32, int64_t at, float none, float scale) {
        float2 v[4];
        if (from != nullptr) {
            param8<F, VEC>(p, 0, from, f32, at, v);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = both(none);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = mul2(v[k], both(scale));
        keep(which, v);
    };
    auto param = [&](int which, float2 *v) {
        const float4 lo = params[(2 * which) * 32], hi = params[(2 * which + 1) * 32];
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
    const bool gate_each = BRANCH && a.gate_rows == 1, gate_summed = BRANCH && a.dgate && a.gate_rows > 1, gate_f32 = sizeof(F) == 4 || a.gate_f32;
    const bool with_f = BRANCH == 2 || (BRANCH && (NEXT || a.dgate));   // whether anything asks for the branch's values
    int gate_end = 0;   // first row of another gate row
    if (BRANCH && a.gate_rows == 0) keep_param(3, nullptr, true, 0, 1.0f, a.branch);

    const X *const x_in = static_cast<const X *>(a.x), *const dh_in = static_cast<const X *>(a.dh);
    const F *const f_in = static_cast<const F *>(a.f), *const dy_in = static_cast<const F *>(a.dy);
    const int bytes_x = ring_bytes(VEC, shape, sizeof(X)), bytes_f = ring_bytes(VEC, shape, sizeof(F));
    const int part_dh = NEXT ? bytes_x : 0, part_f = part_dh + bytes_x, part_dy = part_f + (BRANCH ? bytes_f : 0), part_gate = part_dy + (NEXT ? bytes_f : 0);
    constexpr bool sure = !kTeams;   // (a row in every turn)
    constexpr int kDh = NEXT ? kParts<X> : 0, kF = kDh + kParts<X>, kDy = kF + (BRANCH ? kParts<F> : 0), kGate = kDy + (NEXT ? kParts<F> : 0);
    RowRing<VEC, 1, TEAM> ring(dynamic + 2 * kBackwardParams * 16 * threads, p, part_gate + (gate_each ? ring_bytes(VEC, shape, gate_f32 ? 4 : sizeof(F)) : 0) + shape.pad * (threads / 32),
                               shape.stages);
    const int stride = gridDim.x / p.cluster, own = blockIdx.x / p.cluster;
    RowCursor load{own, 0, 0}, here;
    load.enter(a);
    here = load;
    auto fetch = [&]() {
        if (load.more(a)) {
            const bool some = sure || load.base + p.which < load.end;
            const int64_t row = some ? load.base + p.which : load.end - 1;
            if (with_f) ring.template fetch<F, kF>(p, shape, part_f, f_in, row, some, a);
            if (NEXT) {
                ring.template fetch<X, 0>(p, shape, 0, x_in, row, some, a);
                ring.template fetch<F, kDy>(p, shape, part_dy, dy_in, row, some, a);
            }
            if (dh_in) ring.template fetch<X, kDh>(p, shape, part_dh, dh_in, row, some, a);
            if (gate_each) {
                if (gate_f32)
                    ring.template fetch<float, kGate>(p, shape, part_gate, static_cast<const float *>(a.gate), row, some, a);
                else
                    ring.template fetch<F, kGate>(p, shape, part_gate, static_cast<const F *>(a.gate), row, some, a);
            }
            load.next(a, p.teams, stride);
        }
        ring.filled();
    };
    constexpr int kSums = 5;   // daw, dab, dbw, dbb, gate
    float2 sums[kSums][4];
#pragma unroll
    for (int s = 0; s < kSums; s++) zero8(sums[s]);
    // this thread's sum of eight columns, joined over the block's teams, handed on column by column
    auto hand_out = [&](const float2 *v, auto put) {
        if (!kTeams) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (row_valid<VEC>(p, 0, k)) put(row_column<VEC>(p, 0, k), k & 1 ? v[k >> 1].y : v[k >> 1].x);
            return;
        }
        float *all = reinterpret_cast<float *>(joined);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; k++) all[(VEC ? p.t * 8 + k : p.t + k * p.team) + p.which * p.team * 8] = k & 1 ? v[k >> 1].y : v[k >> 1].x;
        __syncthreads();
        for (int c = tid; c < (int)a.width; c += threads) {
            float s = 0.0f;
            for (int w = 0; w < p.teams; w++) s += all[w * p.team * 8 + c];
            put(c, s);
        }
    };
    for (int s = 1; s < shape.stages; s++) fetch();
    uint32_t set = 0;
    while (here.more(a)) {
        const int row = here.base + p.which, chunk = here.chunk;
        const int64_t at = row * a.width;
        const bool on = sure || row < here.end;
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (BRANCH == 2 || NEXT) st = a.stats[on ? row : here.end - 1];
        if (BRANCH && a.gate_rows > 1 && on && row >= gate_end) {
            const int gate_row = row / (int)a.gate_rows;
            gate_end = (gate_row + 1) * (int)a.gate_rows;
            keep_param(3, a.gate, gate_f32, gate_row * a.width, 1.0f, a.branch);
        }
        auto gate_of = [&](float2 *v) {   // times the branch's scale
            if (!gate_each) {
                param(3, v);
                return;
            }
            if (gate_f32)
                ring.template get<float, kGate>(p, shape, 0, part_gate, static_cast<const float *>(a.gate), at, on, v);
            else
                ring.template get<F, kGate>(p, shape, 0, part_gate, static_cast<const F *>(a.gate), at, on, v);
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = mul2(v[k], both(a.branch));
        };
        uint32_t kept = 0xffu;
        if (BRANCH && a.drop.on) {
            if (VEC)
                kept = keep_bits(((uint64_t)(at + p.first) >> 3) + p.t, key, a.drop);
            else
                form_masks<1>(p, a, key, row, masks, set);
        }
        if (shape.stages == 1) {
            team_barrier<TEAM>();
            fetch();
        }
        ring.ready();
        if (!VEC && BRANCH && a.drop.on) kept = read_masks<1>(p, a, row, masks, set);
        set ^= 1;
        if (shape.stages > 1) fetch();
        float2 t[4];   // the branch, from its norm on normalised
        if (with_f) {
            ring.template get<F, kF>(p, shape, 0, part_f, f_in, at, on, t);
            if (a.drop.on) drop8(t, kept, a.drop.scale);
            if (BRANCH == 2)
#pragma unroll
                for (int k = 0; k < 4; k++) t[k] = mul2(add2(t[k], both(-st.x)), both(st.y));   // (r t - r mean would cost rows far from zero a bit)
        }
        auto branch_out = [&](float2 *n) {   // the branch after its norm
            if (BRANCH == 2) {
                float2 w[4], b[4];
                param(0, w);
                param(1, b);
#pragma unroll
                for (int k = 0; k < 4; k++) n[k] = fma2(t[k], w[k], b[k]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) n[k] = t[k];
            }
        };
        float2 d[4];   // the gradient on its way
        if (NEXT) {
            float2 z[4], u[4], s1 = make_float2(0.0f, 0.0f);   // the stream normalised, dy bw
            ring.template get<X, 0>(p, shape, 0, 0, x_in, at, on, z);
            if (BRANCH) {
                float2 n[4], gate[4];
                branch_out(n);
                gate_of(gate);
#pragma unroll
                for (int k = 0; k < 4; k++) z[k] = fma2(gate[k], n[k], mul2(z[k], both(a.skip)));
            }
            float2 g[4];
            ring.template get<F, kDy>(p, shape, 0, part_dy, dy_in, at, on, g);
            param(2, u);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                z[k] = mul2(add2(z[k], both(-st.z)), both(st.w));
                u[k] = mul2(g[k], u[k]);
                s1 = fma2(u[k], z[k], s1);
            }
            const bool layer = a.before == LUTB_NORM_LAYER, some = !VEC || p.valid;
            const float2 c = row_sums<TEAM>(p, slots, some ? s1.x + s1.y : 0.0f, layer && some ? total(u) : 0.0f, layer, [&]() {
                if (!on) return;
#pragma unroll
                for (int k = 0; k < 4; k++) sums[2][k] = fma2(g[k], z[k], sums[2][k]);
                if (a.sums[3])
#pragma unroll
                    for (int k = 0; k < 4; k++) sums[3][k] = add2(sums[3][k], g[k]);
            });
            const float c1 = -c.x * p.inverse, c2 = layer ? -c.y * p.inverse : 0.0f;
            if (dh_in)
                ring.template get<X, kDh>(p, shape, 0, part_dh, dh_in, at, on, d);
            else
                zero8(d);
#pragma unroll
            for (int k = 0; k < 4; k++) z[k] = fma2(z[k], both(c1), u[k]);
            if (layer)
#pragma unroll
                for (int k = 0; k < 4; k++) z[k] = add2(z[k], both(c2));
#pragma unroll
            for (int k = 0; k < 4; k++) d[k] = fma2(both(st.w), z[k], d[k]);
        } else {
            ring.template get<X, kDh>(p, shape, 0, part_dh, dh_in, at, on, d);
        }
        if (a.dx && on) {
            float2 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = BRANCH ? mul2(d[k], both(a.skip)) : d[k];
            store_row<X, VEC>(p, 0, static_cast<X *>(a.dx) + at, o);
        }
        if (BRANCH) {
            if (a.dgate && on) {
                float2 n[4];
                branch_out(n);
                if (gate_summed) {
#pragma unroll
                    for (int k = 0; k < 4; k++) sums[4][k] = fma2(d[k], n[k], sums[4][k]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) n[k] = mul2(mul2(d[k], both(a.branch)), n[k]);
                    if (gate_f32)
                        store_row<float, VEC>(p, 0, static_cast<float *>(a.dgate) + at, n);
                    else
                        store_row<F, VEC>(p, 0, static_cast<F *>(a.dgate) + at, n);
                }
            }
            {
                float2 gate[4];
                gate_of(gate);
#pragma unroll
                for (int k = 0; k < 4; k++) d[k] = mul2(d[k], gate[k]);
            }
            if (BRANCH == 2) {
                float2 s1 = make_float2(0.0f, 0.0f), w[4];
                param(0, w);
                if (on) {
#pragma unroll
                    for (int k = 0; k < 4; k++) sums[0][k] = fma2(d[k], t[k], sums[0][k]);
                    if (a.sums[1])
#pragma unroll
                        for (int k = 0; k < 4; k++) sums[1][k] = add2(sums[1][k], d[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    d[k] = mul2(d[k], w[k]);
                    if (!VEC) {
                        d[k].x = row_valid<VEC>(p, 0, 2 * k) ? d[k].x : 0.0f;
                        d[k].y = row_valid<VEC>(p, 0, 2 * k + 1) ? d[k].y : 0.0f;
                    }
                    s1 = fma2(d[k], t[k], s1);
                }
                const bool layer = a.after == LUTB_NORM_LAYER, some = !VEC || p.valid;
                const float2 c = row_sums<TEAM>(p, slots, some ? s1.x + s1.y : 0.0f, layer && some ? total(d) : 0.0f, layer, []() {});
                const float c1 = -c.x * p.inverse, c2 = layer ? -c.y * p.inverse : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) d[k] = fma2(t[k], both(c1), d[k]);
                if (layer)
#pragma unroll
                    for (int k = 0; k < 4; k++) d[k] = add2(d[k], both(c2));
#pragma unroll
                for (int k = 0; k < 4; k++) d[k] = mul2(d[k], both(st.y));
            }
            if (a.df && on) {
                if (a.drop.on) drop8(d, kept, a.drop.scale);
                store_row<F, VEC>(p, 0, static_cast<F *>(a.df) + at, d);
            }
        }
        ring.taken();
        here.next(a, p.teams, stride);
        if (gate_summed && here.chunk != chunk) {   // (the same for the whole block)
            const int64_t out = (a.gate_direct ? chunk / a.per_group : chunk) * a.width;
            hand_out(sums[4], [&](int c, float v) {
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
            hand_out(sums[s], [&](int c, float v) { to[c] = v; });
        }
    }
    if (over_cluster<TEAM>(p)) cluster_meet();   // (no block is gone while another may store into it)
}

// ------------------------------------------------------------------------------------------------ launches
int resident_clusters(const void *kernel, const RowShape &s, size_t smem);
int launch_rows(const void *kernel, std::atomic<uint32_t> &opted, const JoinArgs &a, const RowShape &s, int clusters, size_t smem, cudaStream_t stream);

// Shared memory of a block besides the kernel's own arrays, for any join of these types, or for a norm alone.
template <class X, class F>
size_t join_rows_smem(bool backward, bool vec, const RowShape &s, bool alone, bool gate_each) {
    const size_t x = ring_bytes(vec, s, sizeof(X)), f = ring_bytes(vec, s, sizeof(F)), gate = gate_each ? ring_bytes(vec, s, 4) : 0;
    const size_t arrays = alone ? (backward ? 2 * x + f : x) : (backward ? 2 : 1) * (x + f) + gate;   // (a place for dh is kept in any case)
    return (backward ? 2 * kBackwardParams * 16 * s.threads : held_bytes(vec, s)) + s.stages * (arrays + s.pad * (s.threads / 32));
}
// Clusters of a kernel that are resident at a time, as the driver counts them; 0 where it cannot be asked.
template <class X, class F>
int join_rows_clusters(bool backward, const RowShape &s, size_t smem);
template <class X, class F, int BRANCH, bool NEXT>
const void *join_rows_kernel(bool backward, bool vec, const RowShape &s) {
#define LUTB_FORWARD(VEC, G, TEAM) reinterpret_cast<const void *>(&join_rows_forward_kernel<X, F, BRANCH, NEXT, VEC, G, TEAM>)
#define LUTB_BACKWARD(VEC, TEAM) reinterpret_cast<const void *>(&join_rows_backward_kernel<X, F, BRANCH, NEXT, VEC, TEAM>)
    if (backward) {
        if (!vec) return s.kind == TEAM_WARP ? LUTB_BACKWARD(false, TEAM_WARP) : s.kind == TEAM_BLOCK ? LUTB_BACKWARD(false, TEAM_BLOCK) : LUTB_BACKWARD(false, TEAM_BLOCKS);
        return s.kind == TEAM_WARP    ? LUTB_BACKWARD(true, TEAM_WARP)
               : s.kind == TEAM_BLOCK ? LUTB_BACKWARD(true, TEAM_BLOCK)
               : s.kind == TEAM_WIDE  ? LUTB_BACKWARD(true, TEAM_WIDE)
                                      : LUTB_BACKWARD(true, TEAM_CLUSTER);
    }
    if (!vec) return s.groups > 1 ? LUTB_FORWARD(false, 4, TEAM_WIDE) : s.kind == TEAM_WARP ? LUTB_FORWARD(false, 1, TEAM_WARP) : LUTB_FORWARD(false, 1, TEAM_BLOCK);
    if (s.kind == TEAM_WARP) return s.groups == 1 ? LUTB_FORWARD(true, 1, TEAM_WARP) : LUTB_FORWARD(true, 4, TEAM_WARP);
    return s.kind == TEAM_BLOCK ? LUTB_FORWARD(true, 2, TEAM_BLOCK) : s.kind == TEAM_WIDE ? LUTB_FORWARD(true, 2, TEAM_WIDE) : LUTB_FORWARD(true, 2, TEAM_CLUSTER);
#undef LUTB_FORWARD
#undef LUTB_BACKWARD
}
template <class X, class F>
int launch_join_rows(bool backward, bool vec, const JoinArgs &a, const RowShape &s, int clusters, cudaStream_t stream) {
    static std::atomic<uint32_t> opted[2][2][6][8];
    const int kind = (a.alone ? 0 : a.after == LUTB_NORM_NONE ? 1 : 2) * 2 + (backward ? a.dy != nullptr : a.y != nullptr);
    const void *kernel = kind == 1   ? join_rows_kernel<X, F, 0, true>(backward, vec, s)
                         : kind == 2 ? join_rows_kernel<X, F, 1, false>(backward, vec, s)
                         : kind == 3 ? join_rows_kernel<X, F, 1, true>(backward, vec, s)
                         : kind == 4 ? join_rows_kernel<X, F, 2, false>(backward, vec, s)
                         : kind == 5 ? join_rows_kernel<X, F, 2, true>(backward, vec, s)
                                     : nullptr;
    LUTB_REQUIRE(kernel != nullptr, LUTB_ERR_MODE, "nothing to compute");
    const size_t smem = join_rows_smem<X, F>(backward, vec, s, a.alone != 0, a.gate_rows == 1);
    return launch_rows(kernel, opted[backward][vec][kind][backward ? s.kind : 2 * s.kind + (s.groups > 1)], a, s, clusters, smem, stream);
}

// for each pair of types in a file of its own
template <class X, class F>
int join_rows(bool backward, bool vec, const JoinArgs &a, const RowShape &s, int clusters, cudaStream_t stream);
template <class X, class F>
int join_rows_wait_errors(int *count);
#define LUTB_JOIN_ROWS(X, F)                                                                                                        \
    template <>                                                                                                                     \
    int join_rows<X, F>(bool backward, bool vec, const JoinArgs &a, const RowShape &s, int clusters, cudaStream_t stream) {        \
        return launch_join_rows<X, F>(backward, vec, a, s, clusters, stream);                                                      \
    }                                                                                                                               \
    template <>                                                                                                                     \
    int join_rows_clusters<X, F>(bool backward, const RowShape &s, size_t smem) {                                                   \
        return resident_clusters(join_rows_kernel<X, F, 2, true>(backward, true, s), s, smem);                                      \
    }                                                                                                                               \
    template <>                                                                                                                     \
    int join_rows_wait_errors<X, F>(int *count) {                                                                                   \
        LUTB_CUDA(cudaMemcpyFromSymbol(count, g_join_wait_errors, sizeof(int)));                                                    \
        return LUTB_OK;                                                                                                             \
    }

}  // namespace lutb
