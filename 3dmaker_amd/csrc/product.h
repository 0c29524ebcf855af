// What the products (fp8_product.hip, fp4_product.hip, expert_layer.hip) share: their
// arguments, the rows of grouped products, operands widened, the stores of results.
#pragma once

#include "experts.h"
#include "lanes.h"

#include <utility>

namespace graft {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));

struct ProductArgs {
    const uint8_t *a, *as, *b, *bs;
    const int* offsets;
    void* out;
    int m, n, experts, grouping;
    int pitch, spitch;         // of A and B
    int scale_shift;           // rows of B a scale, as a shift: 7 or 0
    long long b_size, bs_size; // of one expert's B and scales
    long long out_stride;
    bool relu, vec;
    int tiles_m, tiles_n;
};

// Eight e4m3 values times 2^(scale - 127) as bf16: exact, as e4m3 has 4 bits, where
// the smallest and largest are in bf16's range (2^-9 and 448 times 2^-110 to 2^119).
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 widen(int lo, int hi, float scale)
{
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A scale from its byte, 0..254.
__device__ __forceinline__ float scale_of(int byte) { return __builtin_bit_cast(float, byte << 23); }

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>)
template <class F, int... I>
__device__ __forceinline__ void each_of(F& f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f)
{
    each_of(f, std::make_integer_sequence<int, N>{});
}

// The workgroup meets when its waves' memory counters have come down to COUNTS
// (an s_waitcnt operand); no memory access moves across.
constexpr int kAllDone = 0x0070, kLdsDone = 0xc07f, kCopiesDone = 0x0f70;
template <int COUNTS>
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(COUNTS);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Row tile `t` of tm rows among all experts' segments: its expert and rows, or
// none.  Every wave finds it by itself.
__device__ __forceinline__ void find_rows(const ProductArgs& a, int t, int tm, int& expert, int& row0, int& row1)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    row0 = row1 = expert = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane;
        int lo = 0, hi = 0;
        if (e < a.experts) {
            lo = min(max(a.offsets[e], 0), a.m);
            hi = min(max(a.offsets[e + 1], lo), a.m);
        }
        const int tiles = (hi - lo + tm - 1) / tm;
        const int up = lanes_scan(tiles);
        const uint64_t found = __ballot(before + up > t);
        if (found) {
            const int l = __ffsll((unsigned long long)found) - 1;
            const int first = before + __shfl(up - tiles, l);
            expert = __builtin_amdgcn_readfirstlane(e0 + l);
            row0 = __builtin_amdgcn_readfirstlane(__shfl(lo, l) + (t - first) * tm);
            row1 = __builtin_amdgcn_readfirstlane(__shfl(hi, l));
            return;
        }
        before += __shfl(up, 63);
    }
}

// Where a segment's row tiles begin: starts[e] for e in 0..experts, from the
// offsets, by the first wave; the last one is their number.
template <int TM>
__device__ __forceinline__ void row_tiles(const ProductArgs& a, int* starts)
{
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < 64) {
        int before = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int e = e0 + lane;
            int n = 0;
            if (e < a.experts) {
                const int lo = min(max(a.offsets[e], 0), a.m), hi = min(max(a.offsets[e + 1], lo), a.m);
                n = (hi - lo + TM - 1) / TM;
            }
            const int up = lanes_scan(n);
            if (e < a.experts) starts[e] = before + up - n;
            before += __shfl(up, 63);
        }
        if (lane == 0) starts[a.experts] = before;
    }
    __syncthreads();
}

// The expert whose row tiles hold tile t < starts[experts].
__device__ __forceinline__ int expert_of_tile(const int* starts, int experts, int t)
{
    const int lane = threadIdx.x & 63;
    for (int e0 = 0;; e0 += 64) {
        const uint64_t found = __ballot(e0 + lane < experts && starts[e0 + lane + 1] > t);
        if (found) return e0 + __ffsll((unsigned long long)found) - 1;
    }
}

template <class T>
__device__ __forceinline__ T finish(float v, bool relu)
{
    return (T)(relu && v < 0.0f ? 0.0f : v);  // NaN stays
}

// N consecutive results from column n on.
template <class T, int N>
__device__ __forceinline__ void store_row(const ProductArgs& a, T* row, int n, const float (&v)[N])
{
    constexpr int P = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
    if (a.vec && n + N <= a.n) {
#pragma unroll
        for (int i = 0; i < N; i += P) {
            Vec<T, P> o;
#pragma unroll
            for (int j = 0; j < P; j++) o[j] = finish<T>(v[i + j], a.relu);
            *reinterpret_cast<Vec<T, P>*>(row + n + i) = o;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (n + i < a.n) row[n + i] = finish<T>(v[i], a.relu);
    }
}

}  // namespace graft
