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

// Which of the elements 8 * block .. 8 * block + 7 stay, as bits.  One block of 128 bits decides eight elements but for one in 8192 of these
// groups, where a digit ties and a second block is formed: 32-bit probabilities at the cost of 16-bit ones.
__device__ __forceinline__ uint32_t keep_bits(uint64_t block, const DropKey &key, const DropRule &rule) {
    const uint4 v = philox_block(block, 0, key);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t kept = 0, tied = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        kept |= ((w[k] << 16) > rule.above ? 1u : 0u) << (2 * k) | (w[k] > rule.above ? 2u : 0u) << (2 * k);
        const uint32_t d = w[k] ^ rule.tie;   // a half of zero where the digits agree
        tied |= (d - 0x00010001u) & ~d & 0x80008000u;
    }
    if (tied && rule.ties) {
        const uint4 s = philox_block(block, 1, key);
        const uint32_t q[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if ((w[k] & 0xffffu) == (rule.tie & 0xffffu) && (q[k] & 0xffffu) >= rule.low) kept |= 1u << (2 * k);
            if ((w[k] >> 16) == (rule.tie & 0xffffu) && (q[k] >> 16) >= rule.low) kept |= 2u << (2 * k);
        }
    }
    return kept;
}

}  // namespace lutb
