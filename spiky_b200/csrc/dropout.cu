// Dropout whose mask is a function of (seed, offset, element) and is never stored: the backward pass forms it again.
#include <math.h>

#include "residual_rows.cuh"

namespace lutb {

DropRule drop_rule(double p) {
    DropRule r{};
    const uint64_t below = (uint64_t)floor(p * 4294967296.0 + 0.5);
    const uint32_t high = (uint32_t)(below >> 16), low = (uint32_t)(below & 0xffff);
    r.on = below != 0;
    r.ties = low != 0;
    r.tie = low ? high | high << 16 : 0;
    r.low = low;
    r.above = (uint32_t)(((uint64_t)(low ? high + 1 : high) << 16) - 1);
    r.scale = below >= (1ull << 32) ? 0.0f : (float)(4294967296.0 / (double)((1ull << 32) - below));
    return r;
}

// A thread takes the eight elements of a generator block; VEC, whole blocks in aligned arrays: two such blocks of 4-byte elements side by side, four of
// 2-byte ones, whose rounds are independent and share the keys; the others element by element.  Bound: 4-byte types by the memory (67 M
// values 83 us, 6.4 TB/s, with a block of threads for each 4096 of them; 92 us when a grid of eight blocks an SM went through them), 2-byte types
// by the integer unit beside it, some 75 of its operations for eight elements (51 us, 5.3 TB/s; on another, slower-clocked GPU four side
// by side 57, two 61, one 67).  Tried and slower: the next 32 bytes a thread loaded ahead (67 us), the rounds' keys in registers (54).
constexpr int64_t kDropMost = 2048ll * INT32_MAX;   // (a grid has 2^31 - 1 blocks, of 2048 elements at least)

template <class T>
constexpr int kDropSide = sizeof(T) == 4 ? 2 : 4;

// The elements of block b one by one, up to the last.
template <class T>
__device__ __forceinline__ void drop_apart(int64_t b, int64_t n, const T *x, T *y, uint32_t kept, float scale) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int64_t i = 8 * b + j;
        if (i < n) y[i] = from_f32<T>((kept >> j & 1) ? to_f32(x[i]) * scale : 0.0f);
    }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(256, 4) dropout_kernel(int64_t n, const T *x, T *y, const int64_t *random, uint64_t site, const DropRule rule) {
    const DropKey key = drop_key(random, site);
    if constexpr (VEC) {
        constexpr int kSide = kDropSide<T>;
        const int64_t first = blockIdx.x * (256ll * kSide) + threadIdx.x;
        uint4 in[kSide][kParts<T>];
#pragma unroll
        for (int k = 0; k < kSide; k++) {
            const int64_t b = first + 256 * k;
            if (8 * b + 8 <= n) {
#pragma unroll
                for (int q = 0; q < kParts<T>; q++) in[k][q] = reinterpret_cast<const uint4 *>(x + 8 * b)[q];
            }
        }
        DropDigits digits[kSide];
#pragma unroll
        for (int k = 0; k < kSide; k++) digits[k] = drop_digits((uint64_t)(first + 256 * k), key, rule);
#pragma unroll
        for (int k = 0; k < kSide; k++) {
            const int64_t b = first + 256 * k;
            if (8 * b + 8 <= n) {
                float2 v[4];
                unpack8<T>(in[k], v);
                drop8(v, digits[k], rule.scale);
                store8(y + 8 * b, v);
            } else if (8 * b < n) {
                drop_apart(b, n, x, y, bits_of(digits[k]), rule.scale);
            }
        }
    } else {
        const int64_t b = blockIdx.x * 256ll + threadIdx.x;
        if (8 * b < n) drop_apart(b, n, x, y, keep_bits((uint64_t)b, key, rule), rule.scale);
    }
}

__global__ void dropout_advance_kernel(int64_t *state, int64_t count, int64_t *used) {
    const int64_t seed = state[0], at = state[1];
    used[0] = seed;
    used[1] = at;
    state[1] = (int64_t)((uint64_t)at + (uint64_t)count);
}

template <class T>
static int launch_dropout(int64_t n, const void *x, void *y, const int64_t *random, uint64_t site, const DropRule &rule, cudaStream_t stream) {
    const T *from = static_cast<const T *>(x);
    T *to = static_cast<T *>(y);
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 32 == 0;
    const int64_t each = 2048 * (vec ? kDropSide<T> : 1), blocks = (n + each - 1) / each;
    KernelScope scope(K_DROPOUT, stream);
    if (vec)
        dropout_kernel<T, true><<<(unsigned)blocks, 256, 0, stream>>>(n, from, to, random, site, rule);
    else
        dropout_kernel<T, false><<<(unsigned)blocks, 256, 0, stream>>>(n, from, to, random, site, rule);
    LUTB_LAUNCH_CHECK();
    return LUTB_OK;
}

}  // namespace lutb

extern "C" int lutb_dropout(int type, int64_t n, double p, const int64_t *random, int64_t site, const void *x, void *y, void *stream) {
    using namespace lutb;
    LUTB_REQUIRE(type == LUTB_F32 || type == LUTB_BF16 || type == LUTB_F16, LUTB_ERR_MODE, "unknown element type %d", type);
    LUTB_REQUIRE(n >= 0 && n <= kDropMost, LUTB_ERR_SHAPE, "number of elements must be between 0 and %lld", (long long)kDropMost);
    LUTB_REQUIRE(p >= 0.0 && p <= 1.0, LUTB_ERR_SHAPE, "dropout probability must be between 0 and 1");
    LUTB_REQUIRE(site >= 0, LUTB_ERR_SHAPE, "site < 0");
    if (n == 0) return LUTB_OK;
    LUTB_REQUIRE(x != nullptr && y != nullptr && random != nullptr, LUTB_ERR_NULL, "x, y and random are required");
    const int size = type == LUTB_F32 ? 4 : 2;
    LUTB_REQUIRE((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % size == 0 && reinterpret_cast<uintptr_t>(random) % 8 == 0,
                 LUTB_ERR_ALIGN, "x and y must be aligned to their elements, random to 8 bytes");
    const DropRule rule = drop_rule(p);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!rule.on) {
        if (x != y) LUTB_CUDA(cudaMemcpyAsync(y, x, (size_t)n * size, cudaMemcpyDeviceToDevice, s));
        return LUTB_OK;
    }
    if (type == LUTB_F32) return launch_dropout<float>(n, x, y, random, (uint64_t)site, rule, s);
    if (type == LUTB_BF16) return launch_dropout<__nv_bfloat16>(n, x, y, random, (uint64_t)site, rule, s);
    return launch_dropout<__half>(n, x, y, random, (uint64_t)site, rule, s);
}

extern "C" int lutb_dropout_advance(int64_t *state, int64_t count, int64_t *used, void *stream) {
    using namespace lutb;
    LUTB_REQUIRE(state != nullptr && used != nullptr, LUTB_ERR_NULL, "state and used are required");
    LUTB_REQUIRE(count >= 0, LUTB_ERR_SHAPE, "count < 0");
    LUTB_REQUIRE((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(used)) % 8 == 0, LUTB_ERR_ALIGN, "state and used must be 8-byte aligned");
    KernelScope scope(K_DROPOUT, static_cast<cudaStream_t>(stream));
    dropout_advance_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(state, count, used);
    LUTB_LAUNCH_CHECK();
    return LUTB_OK;
}
