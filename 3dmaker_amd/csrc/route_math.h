// Scores and their order in routing (route.hip, expert_layer.hip).
#pragma once

#include "lanes.h"

namespace graft {

// Larger float, larger integer; 0 is below every number (an unavailable expert).
__device__ __forceinline__ uint32_t key_of(float c)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, c);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ float of_key(uint32_t k)
{
    return __builtin_bit_cast(float, k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// e^x for x <= 0 to about an ulp: 2^t with the rounding error of t = x log2(e)
// put back (t's error alone would be |x| ulps).  The instruction gives no subnormal
// numbers, so below 2^-126 it works 2^64 higher: experts far behind the first one
// still differ, down to 2^-149; below that they are 0, and equal.
__device__ __forceinline__ float exp_neg(float x)
{
    x = fmaxf(x, -120.0f);
    const float t = x * 1.44269504f;
    const float r = fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;
    const bool low = t < -126.0f;
    const float e = __builtin_amdgcn_exp2f(low ? t + 64.0f : t);
    return fmaf(e, r * 0.693147181f, e) * (low ? 0x1p-64f : 1.0f);
}

}  // namespace graft
