// Device helpers of the 8-bit kernels.
#pragma once
#include "common.hpp"

// ((float)acc * sa) * sb [+ bias], every step rounded (no fused multiply-add): the product and the top-k form the same bits
__device__ __forceinline__ float scaled_sum(int acc, float sa, float sb)
{
#pragma clang fp contract(off)
    const float v = (float)acc * sa;
    return v * sb;
}
__device__ __forceinline__ float add_rounded(float v, float bias)
{
#pragma clang fp contract(off)
    return v + bias;
}

// the bytes of a 16-byte chunk that starts at column k which lie below column K
__device__ __forceinline__ uint4 keep_below(uint4 v, int64_t k, int64_t K)
{
    const int64_t left = K - k;
    if (left >= 16) return v;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t b = left - 4 * i;
        w[i] = b >= 4 ? w[i] : (b <= 0 ? 0u : w[i] & ((1u << (8 * b)) - 1u));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
