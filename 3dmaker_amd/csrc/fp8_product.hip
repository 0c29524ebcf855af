// Products of 8-bit matrices with a power-of-two scale for each block of 128,
// for gfx950:
//   out[m, n] = sum_kb 2^(sa[m, kb] + sb[n, kb] - 254) sum_{k in kb} a[m, k] b[n, k]
// Two matrix instructions carry it.  v_mfma_scale_f32_16x16x128_f8f6f4 takes 128
// of k, one block, and both scales; its accumulators are fp32, but it adds eight
// products at a time and cuts them below 2^-13 of the largest (measured: a 15
// beside 65536 counts as 8), which leaves sums of normal values 1.5e-5 off (of
// their 2-norm).  That is a sixteenth of an fp16 output's own rounding, so 16-bit
// outputs take it.  fp32 outputs (weight gradients) take
// v_mfma_f32_16x16x32_bf16 on operands widened with their scales, which is exact:
// products and sums in fp32 (4e-8), at half the rate.
//
// The first MFMA operand is B's rows, the second A's, so that a lane ends with
// four consecutive n of one row m.  Its two operands are read with the same
// order of k within the block, whatever it is.
#include "experts.h"

#include <algorithm>

namespace graft {

namespace {

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
    int out_type;
    bool relu, vec;
    int tiles_m, tiles_n;
};

__device__ __forceinline__ f4 mfma_scaled(i8v a, int sa, i8v b, int sb, f4 c)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// Eight e4m3 values times 2^(scale - 127) as bf16 (exact: e4m3 has 4 bits).
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 widen(int lo, int hi, float scale)
{
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float scale_of(int byte) { return __builtin_bit_cast(float, byte << 23); }

// 16 bytes a lane from global memory to consecutive LDS addresses of the wave.
__device__ __forceinline__ void load_lds16(const uint8_t* from, uint8_t* to)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// A segment's rows and the expert they belong to: tile `t` of all experts' row
// tiles of `tm` rows, or no rows.  Every wave finds it by itself.
__device__ __forceinline__ void find_rows(const ProductArgs& a, int t, int tm, int& expert, int& row0, int& row1)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    row0 = row1 = 0;
    expert = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane;
        int lo = 0, hi = 0;
        if (e < a.experts) {
            lo = min(max(a.offsets[e], 0), a.m);
            hi = min(max(a.offsets[e + 1], lo), a.m);
        }
        const int tiles = (hi - lo + tm - 1) / tm;
        int up = tiles;
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(up, d);
            up += lane >= d ? o : 0;
        }
        const uint64_t found = __ballot(before + up > t);
        if (found) {
            const int l = __ffsll((unsigned long long)found) - 1;
            const int first = before + __shfl(up - tiles, l);
            expert = e0 + l;
            row0 = __shfl(lo, l) + (t - first) * tm;
            row1 = __shfl(hi, l);
            return;
        }
        before += __shfl(up, 63);
    }
}

__device__ __forceinline__ void store4(const ProductArgs& a, long long at, int n, f4 v)
{
    if (a.relu) {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // NaN stays
    }
    const int left = a.n - n;
    auto put = [&](auto zero) {
        using T = decltype(zero);
        T* p = (T*)a.out + at + n;
        if (a.vec && left >= 4) {
            *reinterpret_cast<Vec<T, 4>*>(p) = Vec<T, 4>{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < left) p[j] = (T)v[j];
        }
    };
    if (a.out_type == DATA_F32) put(float{});
    else if (a.out_type == DATA_F16) put((_Float16)0);
    else put((__bf16)0.0f);
}

// Tiles of TM x TN, WM x WN waves.  Both operands of a block of k go through
// two LDS stages, rows of 128 bytes whose 16-byte pieces are permuted by the
// row's low bits (the permutation is in the global addresses: the copy to LDS
// is linear), so that 8 rows' pieces of one column lie in different banks.
template <int TM, int TN, int WM, int WN, bool WIDE>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(ProductArgs a)
{
    constexpr int kWaves = WM * WN, MT = TM / WM / 16, NT = TN / WN / 16;
    constexpr int kStage = (TM + TN) * 128, kLoads = (TM + TN) / 8 / kWaves;
    static_assert((TM + TN) % (8 * kWaves) == 0 && TM % 8 == 0, "whole wave loads");
    __shared__ __attribute__((aligned(128))) uint8_t lds[2 * kStage];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int tm, tn, expert = 0, row0, row1, kb0 = 0, kb1 = a.pitch / 128;
    if (a.grouping == PRODUCT_SUM) {
        const int per = a.tiles_m * a.tiles_n;
        expert = blockIdx.x / per;
        tm = blockIdx.x % per / a.tiles_n;
        tn = blockIdx.x % a.tiles_n;
        kb0 = min(max(a.offsets[expert] / 128, 0), kb1);
        kb1 = min(max(a.offsets[expert + 1] / 128, kb0), kb1);
        row0 = tm * TM;
        row1 = a.m;
    } else {
        tm = blockIdx.x / a.tiles_n;
        tn = blockIdx.x % a.tiles_n;
        if (a.grouping == PRODUCT_ROWS) {
            find_rows(a, tm, TM, expert, row0, row1);
            if (row0 >= row1) return;
        } else {
            row0 = tm * TM;
            row1 = a.m;
        }
    }
    const int n0 = tn * TN;
    const long long be = a.grouping == PRODUCT_ROWS ? expert : 0;
    const uint8_t* A = a.a + (long long)row0 * a.pitch;
    const uint8_t* B = a.b + be * a.b_size + (long long)n0 * a.pitch;
    const uint8_t* SA = a.as + (long long)row0 * a.spitch;
    const uint8_t* SB = a.bs + be * a.bs_size + (long long)(n0 >> a.scale_shift) * a.spitch;

    // The wave's pieces of a stage: 8 rows by 128 bytes each.
    uint32_t from[kLoads];
    bool of_a[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const int r = (i * kWaves + wave) * 8 + (lane >> 3);
        const int piece = (lane & 7) ^ (r & 7);
        of_a[i] = (i * kWaves + wave) * 8 < TM;
        const int row = of_a[i] ? min(r, row1 - row0 - 1) : min(r - TM, a.n - n0 - 1);
        from[i] = (uint32_t)row * a.pitch + piece * 16;
    }
    auto fetch = [&](int kb, int stage) {
#pragma unroll
        for (int i = 0; i < kLoads; i++)
            load_lds16((of_a[i] ? A : B) + (long long)kb * 128 + from[i], lds + stage * kStage + (i * kWaves + wave) * 1024);
    };

    const int wm = wave / WN, wn = wave % WN, col = lane & 15, quad = lane >> 4;
    uint32_t sa_at[MT], sb_at[NT];
#pragma unroll
    for (int i = 0; i < MT; i++) sa_at[i] = min(wm * (TM / WM) + i * 16 + col, row1 - row0 - 1) * a.spitch;
#pragma unroll
    for (int i = 0; i < NT; i++)
        sb_at[i] = (uint32_t)((min(n0 + wn * (TN / WN) + i * 16 + col, a.n - 1) >> a.scale_shift) - (n0 >> a.scale_shift)) *
                   a.spitch;

    f4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f4zero();

    if (kb0 < kb1) fetch(kb0, 0);
    __syncthreads();
    for (int kb = kb0; kb < kb1; kb++) {
        const int stage = (kb - kb0) & 1;
        if (kb + 1 < kb1) fetch(kb + 1, stage ^ 1);
        int sa[MT], sb[NT];
#pragma unroll
        for (int i = 0; i < MT; i++) sa[i] = SA[sa_at[i] + kb];
#pragma unroll
        for (int i = 0; i < NT; i++) sb[i] = SB[sb_at[i] + kb];
        const uint8_t* base = lds + stage * kStage;
        auto fragment = [&](int r) {  // row r of the stage, pieces quad and quad + 4
            const uint8_t* p = base + r * 128;
            const i4v lo = *reinterpret_cast<const i4v*>(p + ((quad ^ (r & 7)) * 16));
            const i4v hi = *reinterpret_cast<const i4v*>(p + (((quad + 4) ^ (r & 7)) * 16));
            return i8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
        if constexpr (WIDE) {
            bf16x8 fa[MT][4];
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const i8v f = fragment(wm * (TM / WM) + j * 16 + col);
#pragma unroll
                for (int q = 0; q < 4; q++) fa[j][q] = widen(f[2 * q], f[2 * q + 1], scale_of(sa[j]));
            }
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const i8v f = fragment(TM + wn * (TN / WN) + i * 16 + col);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const bf16x8 fb = widen(f[2 * q], f[2 * q + 1], scale_of(sb[i]));
#pragma unroll
                    for (int j = 0; j < MT; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fa[j][q], acc[i][j], 0, 0, 0);
                }
            }
        } else {
            i8v fa[MT];
#pragma unroll
            for (int j = 0; j < MT; j++) fa[j] = fragment(wm * (TM / WM) + j * 16 + col);
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const i8v fb = fragment(TM + wn * (TN / WN) + i * 16 + col);
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = mfma_scaled(fb, sb[i], fa[j], sa[j], acc[i][j]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const int r = wm * (TM / WM) + j * 16 + col;
        if (row0 + r >= row1) continue;
        const long long at = ((a.grouping == PRODUCT_SUM ? (long long)expert * a.m : 0) + row0 + r) * a.out_stride;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int n = n0 + wn * (TN / WN) + i * 16 + quad * 4;
            if (n < a.n) store4(a, at, n, acc[i][j]);
        }
    }
}

template <int TM, int TN, int WM, int WN, bool WIDE>
void product_launch(ProductArgs& a, hipStream_t s)
{
    a.tiles_n = (a.n + TN - 1) / TN;
    a.tiles_m = (a.m + TM - 1) / TM;
    long long grid = (long long)a.tiles_m * a.tiles_n;
    if (a.grouping == PRODUCT_ROWS) grid = ((long long)a.m / TM + a.experts) * a.tiles_n;
    if (a.grouping == PRODUCT_SUM) grid *= a.experts;
    require(grid <= 0x7fffffffll, "too many tiles for one call");
    product_kernel<TM, TN, WM, WN, WIDE><<<(unsigned)grid, WM * WN * 64, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

}  // namespace

void fp8_product(const Fp8ProductOption& o, const uint8_t* a, const uint8_t* a_scales, const uint8_t* b,
                 const uint8_t* b_scales, const int* offsets, void* out, hipStream_t s)
{
    require(o.m >= 0 && o.m <= kMaxRows, "m must be 0..2^30");
    require(o.n >= 1 && o.n <= 1 << 22 && o.k >= (o.grouping == PRODUCT_SUM ? 0 : 1) && o.k <= 1 << 22,
            "n must be 1..2^22 and k 1..2^22 (SUM: from 0 on)");
    require(o.grouping == PRODUCT_DENSE || o.grouping == PRODUCT_ROWS || o.grouping == PRODUCT_SUM, "unknown grouping");
    require(o.numExperts >= 1 && o.numExperts <= 1024 && (o.grouping != PRODUCT_DENSE || o.numExperts == 1),
            "numExperts must be 1..1024, and 1 for a dense product");
    require(o.scaleRowsB == 1 || o.scaleRowsB == 128, "scaleRowsB must be 1 or 128");
    require(o.activation == 0 || o.activation == 1, "unknown activation");
    require_type(o.outType);
    require(o.outStride >= o.n, "outStride must be at least n");
    require((o.grouping == PRODUCT_DENSE) == !offsets, "offsets go with grouped products");
    if (o.m == 0) return;
    require(out && ((a && a_scales && b && b_scales) || o.k == 0), "null argument");
    require(aligned16(a) && aligned16(b) && ((uintptr_t)a_scales & 3) == 0 && ((uintptr_t)b_scales & 3) == 0,
            "8-bit matrices must be 16-byte aligned and scales 4-byte aligned");
    ProductArgs p{};
    p.a = a;
    p.as = a_scales;
    p.b = b;
    p.bs = b_scales;
    p.offsets = offsets;
    p.out = out;
    p.m = o.m;
    p.n = o.n;
    p.experts = o.numExperts;
    p.grouping = o.grouping;
    p.pitch = fp8_pitch(o.k);
    p.spitch = fp8_scale_pitch(o.k);
    p.scale_shift = o.scaleRowsB == 128 ? 7 : 0;
    p.b_size = (long long)o.n * p.pitch;
    p.bs_size = (long long)((o.n + o.scaleRowsB - 1) / o.scaleRowsB) * p.spitch;
    p.out_stride = o.outStride;
    p.out_type = o.outType;
    p.relu = o.activation == 1;
    p.vec = (uintptr_t)out % (4 * data_bytes(o.outType)) == 0 && o.outStride % 4 == 0;
    // Up to two blocks of k the output's bytes bound the product, and widening
    // costs nothing.
    if (o.outType == DATA_F32 || p.pitch <= 256) product_launch<128, 128, 2, 2, true>(p, s);
    else product_launch<128, 128, 2, 2, false>(p, s);
}

}  // namespace graft
