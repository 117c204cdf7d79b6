// Shared parts of the residual-stream kernels: element types, the counter-based generator of the dropout masks, sums over a row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lutb_common.cuh"

namespace lutb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// What a launch needs to know of a dropout: element i is dropped iff the 32-bit number of its two 16-bit digits is below T =
// round(p 2^32).  The second digit decides only where the first equals T's upper half.
struct DropRule {
    uint32_t above;   // digit << 16 > above: kept by the first digit alone
    uint32_t tie;     // first digit that leaves it to the second one (in both halves of the word); ties: whether there are any
    uint32_t low;     // second digit of a kept element: >= low
    uint32_t ties;
    float scale;      // 2^32 / (2^32 - T); 0 where everything is dropped
    uint32_t on;
};
DropRule drop_rule(double p);

struct DropKey {
    uint32_t seed0, seed1, at0, at1;
};
__device__ __forceinline__ DropKey drop_key(const int64_t *random, uint64_t site) {
    const uint64_t seed = (uint64_t)random[0], at = (uint64_t)random[1] + site;
    return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)at, (uint32_t)(at >> 32)};
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): counter (block, block's upper half | second << 31, offset), key the seed.
__device__ __forceinline__ uint4 philox_block(uint64_t block, uint32_t second, const DropKey &key) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32) | second << 31, c2 = key.at0, c3 = key.at1, k0 = key.seed0, k1 = key.seed1;
#pragma unroll
    for (int round = 0; round < 10; round++) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// The digits of the elements 8 * block .. 8 * block + 7: element 2k stays when word k << 16 is above `above`, element 2k + 1 when word k is.  One block of
// 128 bits decides eight elements but for one in 8192 of these groups, where a digit ties and a second block is formed: 32-bit
// probabilities at the cost of 16-bit ones.
struct DropDigits {
    uint32_t w[4], above;
};
__device__ __forceinline__ DropDigits drop_digits(uint64_t block, const DropKey &key, const DropRule &rule) {
    const uint4 v = philox_block(block, 0, key);
    DropDigits d{{v.x, v.y, v.z, v.w}, rule.above};
    // the smaller halves of the words' differences from T's upper digit: 0 where a digit ties
    const uint32_t near = __vimin3_u16x2(d.w[0] ^ rule.tie, d.w[1] ^ rule.tie, __vminu2(d.w[2] ^ rule.tie, d.w[3] ^ rule.tie));
    if ((near < 0x10000u || (near & 0xffffu) == 0u) && rule.ties) {
        const uint4 s = philox_block(block, 1, key);
        const uint32_t q[4] = {s.x, s.y, s.z, s.w}, tie = rule.tie & 0xffffu;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t lo = d.w[k] & 0xffffu, hi = d.w[k] >> 16;
            const bool keep_lo = lo == tie ? (q[k] & 0xffffu) >= rule.low : (lo << 16) > rule.above;
            const bool keep_hi = hi == tie ? (q[k] >> 16) >= rule.low : d.w[k] > rule.above;
            d.w[k] = (keep_lo ? 0xffffu : 0u) | (keep_hi ? 0xffff0000u : 0u);
        }
        d.above = 0x7fffffffu;
    }
    return d;
}
// Which of the eight stay, as bits.
__device__ __forceinline__ uint32_t bits_of(const DropDigits &d) {
    uint32_t kept = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) kept |= ((d.w[k] << 16) > d.above ? 1u : 0u) << (2 * k) | (d.w[k] > d.above ? 2u : 0u) << (2 * k);
    return kept;
}
__device__ __forceinline__ uint32_t keep_bits(uint64_t block, const DropKey &key, const DropRule &rule) { return bits_of(drop_digits(block, key, rule)); }

}  // namespace lutb
