// Reductions over aligned groups of W lanes (W a power of two up to 64) whose
// result every lane of the group holds: row DPP up to 16 lanes, the lane swaps
// between rows of 16 and halves of 32 above.  Partners combine the same two
// values in either order, so all lanes of a group get the same bits.
#pragma once

#include "common.h"

namespace graft {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_mov(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

// f(own, partner) over the group, one step per power of two.
template <int W, class F>
__device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, F f)
{
    static_assert(W >= 1 && W <= 64 && (W & (W - 1)) == 0, "a power of two up to the wave");
    if constexpr (W >= 2) v = f(v, dpp_mov<0xB1>(v));    // quad_perm [1,0,3,2]
    if constexpr (W >= 4) v = f(v, dpp_mov<0x4E>(v));    // quad_perm [2,3,0,1]
    if constexpr (W >= 8) v = f(v, dpp_mov<0x141>(v));   // row_half_mirror: the other quad of 8
    if constexpr (W >= 16) v = f(v, dpp_mov<0x140>(v));  // row_mirror: the other 8 of 16
    if constexpr (W >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(r[0], r[1]);
    }
    if constexpr (W >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(r[0], r[1]);
    }
    return v;
}

template <int W>
__device__ __forceinline__ float lanes_sum(float v)
{
    return __builtin_bit_cast(float, lanes_reduce<W>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}

template <int W>
__device__ __forceinline__ float lanes_max(float v)
{
    return __builtin_bit_cast(float, lanes_reduce<W>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
    }));
}

template <int W>
__device__ __forceinline__ uint32_t lanes_umax(uint32_t v)
{
    return lanes_reduce<W>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// Inclusive sum over the wave: row shifts, then the rows' last values onward.
__device__ __forceinline__ int lanes_scan(int v)
{
    v += (int)dpp_mov<0x111>((uint32_t)v);  // row_shr:1, zero at the row's start
    v += (int)dpp_mov<0x112>((uint32_t)v);
    v += (int)dpp_mov<0x114>((uint32_t)v);
    v += (int)dpp_mov<0x118>((uint32_t)v);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
    return v;
}

}  // namespace graft
