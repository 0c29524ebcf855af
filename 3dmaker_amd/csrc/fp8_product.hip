// Products of 8-bit matrices with a power-of-two scale for each block of 128,
// for gfx950:
//   out[m, n] = sum_kb 2^(sa[m, kb] + sb[n, kb] - 254) sum_{k in kb} a[m, k] b[n, k]
// Two matrix instructions carry it.  v_mfma_scale_f32_16x16x128_f8f6f4 takes 128
// of k, one block, and both scales; its accumulators are fp32, but it adds eight
// products at a time and cuts each towards zero to a multiple of 2^-13 of the
// largest one's power of two (measured: a 15 beside 65536 counts as 8; between the
// eights and with the accumulator nothing is cut).  Sums of normal values come out
// 1.5e-5 off (2-norm; non-negative ones 3e-6), of values spread over all of e4m3
// 7e-5, below an fp16 output's own rounding of 1.4e-4; but the error goes by the
// largest product of an eight, not by the sum.  So 16-bit outputs take it unless
// the caller asks for exact sums.  Those, fp32 outputs and weight gradients take
// v_mfma_f32_16x16x32_bf16 on operands widened with their scales, which is exact:
// products and sums in fp32 (4e-8), at half the rate (8191 x 5120 x 4096 bf16: 307
// us and 195, 65,536 rows by eight experts of 2048 x 1024 280 and 189).
//
// The first MFMA operand is B's rows, the second A's, so that a lane ends with
// four consecutive n of one row m.  Its two operands are read with the same
// order of k within the block, whatever it is.
#include "experts.h"
#include "lanes.h"

#include <algorithm>
#include <type_traits>
#include <utility>

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

// Experts in the order of their columns, most first (equal ones in their own
// order), up to 128 of them; more balance themselves.
__device__ __forceinline__ void by_length(const ProductArgs& a, int* order)
{
    int* length = order + a.experts;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        order[e] = e;
        if (a.experts <= 128) length[e] = a.offsets[e + 1] - a.offsets[e];
    }
    __syncthreads();
    if (a.experts <= 128) {
        const int e = threadIdx.x;
        if (e < a.experts) {
            int rank = 0;
            for (int o = 0; o < a.experts; o++) rank += length[o] > length[e] || (length[o] == length[e] && o < e);
            order[rank] = e;
        }
        __syncthreads();
    }
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

// Large products: TM x TN tiles by four waves, persistent workgroups.
//
// A block of k of both operands lies in one of two LDS stages, rows of 128
// bytes whose 16-byte pieces are permuted by a key of the row, so that the 16
// rows of a fragment are read from all banks; the copy to LDS is linear, so the
// permutation is in its global addresses.  It is a buffer load, which gives rows
// behind the tile's last as zeros.
//
// A wave's tile is worked through in quadrants of its two halves of A's and of
// B's fragments.  The next quadrant's half is read from LDS, and the block after
// the next copied to it, between this one's matrix instructions: a copy or read
// that is issued in a burst holds the wave's matrix instructions up (8192 x
// 5120 x 4096 in tiles of 256: 207 us with bursts, 197 spread; of 128: 176 and 168).  The order is held by the empty
// asm on the accumulators and the scheduling barriers.  The one barrier of a
// block stands behind its last LDS read, half a block before its last matrix
// instruction.
//
// B's row of fragment i and lane column c is (i / 2) 32 + (c / 4) 8 + (i % 2) 4 +
// c % 4: a lane ends with eight consecutive columns of two fragments, one 16-byte
// store of 16-bit results.
//
// The scales of 32 blocks lie in LDS in the order in which a lane takes them:
// one read gives four fragments' bytes, which the matrix instruction selects.
//
// Tile sizes: a block costs a CU (TM + TN) 128 bytes of copies at 64 a clock and
// (TM WN + TN WM) 128 of LDS reads at 128 a clock besides writes, for TM TN / 512
// clocks of matrix work.  256 x 256 has most room (2.5 PFLOP/s at 8192^3) but one
// workgroup a CU; two of 128 x 128 fit (2.2 PFLOP/s) and lose less to a last round
// of tiles.  131,128 rows of 256 experts of 1024 x 2048: 405 us, 1.36 PFLOP/s.
template <class T, int TM, int TN, bool WIDE>
__global__ __launch_bounds__(256, TM * TN > 128 * 128 ? 1 : 2) void product_kernel(ProductArgs a)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host pass needs the kernel's name alone
    using std::integral_constant;
    constexpr int WM = 2, WN = 2, kWaves = 4, MT = TM / WM / 16, NT = TN / WN / 16, MH = MT / 2, NH = NT / 2;
    constexpr int kStage = (TM + TN) * 128, kLoads = (TM + TN) / 8 / kWaves, kScaleRow = TM + TN;
    static_assert(TM % (8 * kWaves) == 0 && MT % 4 == 0 && NT % 4 == 0, "whole fragments and copies");
    // One array: with two, the compiler waits for all copies before each LDS read.
    __shared__ __attribute__((aligned(128))) uint8_t lds[2 * kStage + 32 * kScaleRow + 1028 * 4];
    int* const starts = reinterpret_cast<int*>(lds + 2 * kStage + 32 * kScaleRow);
    uint8_t* const scale_lds = lds + 2 * kStage;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave / WN, wn = wave % WN, col = lane & 15, quad = lane >> 4;

    int total = a.tiles_m * a.tiles_n;
    if (a.grouping == PRODUCT_SUM) total *= a.experts;
    int row_tile_count = a.tiles_m;
    // The segments: up to 64 of them lane by lane (rows, and the row tiles up to
    // their end), more through LDS and memory.
    int seg_lo = 0, seg_hi = 0, seg_end = 0;
    if (a.grouping == PRODUCT_ROWS) {
        if (a.experts <= 64) {
            if (lane < a.experts) {
                seg_lo = min(max(a.offsets[lane], 0), a.m);
                seg_hi = min(max(a.offsets[lane + 1], seg_lo), a.m);
            }
            seg_end = lanes_scan((seg_hi - seg_lo + TM - 1) / TM);
            row_tile_count = __builtin_amdgcn_readlane(seg_end, 63);
        } else {
            row_tiles<TM>(a, starts);
            row_tile_count = __builtin_amdgcn_readfirstlane(starts[a.experts]);
        }
        total = row_tile_count * a.tiles_n;
    }
    // Workgroups go round the XCDs.  Each XCD works through a range of tiles of its
    // own; but where experts' k differ (SUM), a range of one expert's would leave
    // the XCDs of small ones idle (experts of 1,700 to 11,000 columns: 200 us): there
    // the workgroups take the tiles of the experts of most k first, every second
    // round backwards, and an expert's tiles are dealt to all XCDs in ranges.
    const int per = a.tiles_m * a.tiles_n;
    if (a.grouping == PRODUCT_SUM) by_length(a, starts);
    const int xcd = blockIdx.x & 7, x0 = xcd * (total / 8) + min(xcd, total % 8), xn = total / 8 + (xcd < total % 8);
    int round = 0;
    auto tile_of_round = [&]() -> int {  // -1: none left
        if (a.grouping == PRODUCT_SUM) {
            const int t = round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            if (t >= total) return -1;
            const int rank = t / per, q = t - rank * per;
            return starts[rank] * per + (per % 8 == 0 ? q % 8 * (per / 8) + q / 8 : q);
        }
        const int at = (blockIdx.x >> 3) + round * ((gridDim.x + 7 - xcd) / 8);
        return at < xn ? x0 + at : -1;
    };
    int tile = __builtin_amdgcn_readfirstlane(tile_of_round());
    if (tile < 0) return;

    int row0, row1, n0, kb0, kb1;
    long long out0;
    const uint8_t *SA, *SB;
    __amdgpu_buffer_rsrc_t ra, rb;
    auto place = [&](int t) {  // four row tiles by all columns at a time: what an XCD has in flight shares its L2
        int expert = 0;
        if (a.grouping == PRODUCT_SUM) {
            expert = t / per;
            t -= expert * per;
        }
        const int group = t / (4 * a.tiles_n), first = group * 4, rows = min(4, row_tile_count - first);
        const int in = t - first * a.tiles_n, tm = first + in % rows;
        n0 = in / rows * TN;
        kb0 = 0;
        kb1 = a.pitch / 128;
        row0 = tm * TM;
        row1 = a.m;
        const uint8_t* B = a.b;
        SB = a.bs;
        out0 = 0;
        if (a.grouping == PRODUCT_ROWS) {
            if (a.experts <= 64) {
                expert = __ffsll((unsigned long long)__ballot(seg_end > tm)) - 1;
                row1 = __builtin_amdgcn_readlane(seg_hi, expert);
                row0 = __builtin_amdgcn_readlane(seg_lo, expert);
                row0 += (tm - __builtin_amdgcn_readlane(seg_end, expert) + (row1 - row0 + TM - 1) / TM) * TM;
            } else {
                expert = __builtin_amdgcn_readfirstlane(expert_of_tile(starts, a.experts, tm));
                const int lo = min(max(a.offsets[expert], 0), a.m);
                row0 = __builtin_amdgcn_readfirstlane(lo + (tm - starts[expert]) * TM);
                row1 = __builtin_amdgcn_readfirstlane(min(max(a.offsets[expert + 1], lo), a.m));
            }
            B += expert * a.b_size;
            SB += expert * a.bs_size;
        } else if (a.grouping == PRODUCT_SUM) {
            kb0 = __builtin_amdgcn_readfirstlane(min(max(a.offsets[expert] / 128, 0), kb1));
            kb1 = __builtin_amdgcn_readfirstlane(min(max(a.offsets[expert + 1] / 128, kb0), kb1));
            out0 = (long long)expert * a.m * a.out_stride;
        }
        const int flags = 0x00020000;
        ra = __builtin_amdgcn_make_buffer_rsrc((void*)(a.a + (long long)row0 * a.pitch), 0, min(TM, row1 - row0) * a.pitch,
                                               flags);
        rb = __builtin_amdgcn_make_buffer_rsrc((void*)(B + (long long)n0 * a.pitch), 0, min(TN, a.n - n0) * a.pitch, flags);
        SA = a.as + (long long)row0 * a.spitch;
        SB += (long long)(n0 >> a.scale_shift) * a.spitch;
    };

    uint32_t from[kLoads];  // the lane's piece of each copy: 8 rows of 128 bytes a wave
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const bool of_a = i * kWaves * 8 < TM;
        const int r = (i * kWaves + wave) * 8 + (lane >> 3) - (of_a ? 0 : TM);
        const int key = of_a ? r & 7 : (r & 3) | (r >> 1 & 4);
        from[i] = (uint32_t)r * a.pitch + ((lane & 7) ^ key) * 16;
    }
    auto copy = [&](int kb, int stage, int i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(i * kWaves * 8 < TM ? ra : rb,
                                                 (__attribute__((address_space(3))) void*)(lds + stage * kStage +
                                                                                           (i * kWaves + wave) * 1024),
                                                 16, from[i], kb * 128, 0, 0);
    };
    auto copy_first = [&] {
#pragma unroll
        for (int i = 0; i < kLoads; i++) copy(kb0, 0, i);
#pragma unroll
        for (int i = 0; i < kLoads; i++) copy(min(kb0 + 1, kb1 - 1), 1, i);
    };
    // Scale bytes of blocks kb .. kb + 31 (kb a multiple of 4) to
    // [block][the fragments' bytes of a wave and lane column together].
    auto copy_scales = [&](int kb) {
        const int words = min(8, (kb1 - kb + 3) / 4);
        for (int r = threadIdx.x; r < TM + TN; r += 256) {
            const bool of_a = r < TM;
            const int row = of_a ? min(r, row1 - row0 - 1)
                                 : (min(n0 + r - TM, a.n - 1) >> a.scale_shift) - (n0 >> a.scale_shift);
            const uint8_t* p = (of_a ? SA : SB) + (uint32_t)row * a.spitch + kb;
            const int w = of_a ? r : r - TM, in = w % (of_a ? TM / WM : TN / WN);
            const int to = of_a ? w - in + (in & 15) * MT + (in >> 4)
                                : TM + w - in + ((in >> 3 & 3) * 4 + (in & 3)) * NT + (in >> 5) * 2 + (in >> 2 & 1);
            for (int d = 0; d < words; d++) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(p + d * 4);
#pragma unroll
                for (int q = 0; q < 4; q++) scale_lds[(d * 4 + q) * kScaleRow + to] = (uint8_t)(v >> (8 * q));
            }
        }
    };

    f4 acc[NT][MT];
    i8v a0[MH], a1[MH], b0[NH], b1[NH];
    bf16x8 wa[WIDE ? MH : 1][4], w0[WIDE ? NH : 1][4], w1[WIDE ? NH : 1][4];
    int sa[MT / 4], sb[NT / 4];
    auto scales = [&](int slot) {
        const uint8_t* p = scale_lds + (slot & 31) * kScaleRow;
#pragma unroll
        for (int i = 0; i < MT / 4; i++) sa[i] = *reinterpret_cast<const int*>(p + wm * (TM / WM) + col * MT + i * 4);
#pragma unroll
        for (int i = 0; i < NT / 4; i++) sb[i] = *reinterpret_cast<const int*>(p + TM + wn * (TN / WN) + col * NT + i * 4);
    };
    // Half h (pieces quad or quad + 4) of fragment i.
    const int a_at = (wm * (TM / WM) + col) * 128, b_at = (TM + wn * (TN / WN) + (col >> 2) * 8 + (col & 3)) * 128;
    const int a_key = col & 7, b_key = col & 7;  // of rows 16 i + col; of B's rows (row & 3) | (row >> 1 & 4)
    auto read_half = [&](i8v& f, int address, int h, int key) {
        const i4v v = *reinterpret_cast<const i4v*>(lds + address + (((quad + 4 * h) ^ key) * 16));
#pragma unroll
        for (int j = 0; j < 4; j++) f[4 * h + j] = v[j];
    };
    auto read_a = [&](i8v& f, int stage, int i, int h) { read_half(f, stage * kStage + a_at + i * 2048, h, a_key); };
    auto read_b = [&](i8v& f, int stage, int i, int h) {
        read_half(f, stage * kStage + b_at + (i >> 1) * 4096 + (i & 1) * 512, h, b_key);
    };
    auto widen_all = [&](auto& w, auto& f, const int* s, int first) {
        each<sizeof(f) / sizeof(f[0])>([&](auto I) {
            constexpr int i = decltype(I)::value;
            const float scale = scale_of(s[(first + i) / 4] >> (8 * ((first + i) % 4)) & 0xff);
#pragma unroll
            for (int q = 0; q < 4; q++) w[i][q] = widen(f[i][2 * q], f[i][2 * q + 1], scale);
        });
    };
    // One quadrant; between(m) behind its m-th fragment pair.
    auto quadrant = [&](auto& x, auto& wx, auto MO, auto& y, auto& wy, auto NO, auto between) {
        constexpr int mo = decltype(MO)::value, no = decltype(NO)::value;
        each<NH>([&](auto I) {
            each<MH>([&](auto J) {
                constexpr int i = decltype(I)::value, j = decltype(J)::value;
                f4& c = acc[no + i][mo + j];
                if constexpr (WIDE) {
#pragma unroll
                    for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wy[i][q], wx[j][q], c, 0, 0, 0);
                } else {
                    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(y[i], x[j], c, 0, 0, (no + i) % 4, sb[(no + i) / 4],
                                                                         (mo + j) % 4, sa[(mo + j) / 4]);
                }
                asm volatile("" : "+v"(c));
                between(integral_constant<int, i * MH + j>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    };
    // f(0) .. f(N - 1) spread over a quadrant's MH * NH places.
    auto spread = [&](auto N, auto M, auto f) {
        constexpr int n = decltype(N)::value, m = decltype(M)::value, places = MH * NH;
        constexpr int lo = (m * n + places - 1) / places, hi = ((m + 1) * n + places - 1) / places;
        each<hi - lo>([&](auto Q) { f(lo + decltype(Q)::value); });
    };
    // Block kb in `stage`: A's first half and B's half X have been read; leaves the
    // next block's first half of A and half Y of B read, Y its X.
    auto block = [&](int kb, int stage, auto& bx, auto& wx, auto X, auto& by, auto& wy, auto Y) {
        constexpr int xo = decltype(X)::value, yo = decltype(Y)::value;
        const integral_constant<int, 0> lower{};
        const integral_constant<int, MH> upper{};
        const integral_constant<int, 2 * MH> a_reads{};
        const integral_constant<int, 2 * NH> b_reads{};
        const integral_constant<int, kLoads / 2> copies{};
        if constexpr (WIDE) {
            widen_all(wa, a0, sa, 0);
            widen_all(wx, bx, sb, xo);
        }
        quadrant(a0, wa, lower, bx, wx, X, [&](auto m) {
            spread(b_reads, m, [&](int q) { read_b(by[q / 2], stage, yo + q / 2, q % 2); });
        });
        if constexpr (WIDE) widen_all(wy, by, sb, yo);
        quadrant(a0, wa, lower, by, wy, Y, [&](auto m) {
            spread(a_reads, m, [&](int q) { read_a(a1[q / 2], stage, MH + q / 2, q % 2); });
        });
        if (kb != kb0) __builtin_amdgcn_s_waitcnt(kCopiesDone);  // the next block is here (the second was before the first)
        meet<kLdsDone>();                                        // this one is read
        const int after = min(kb + 2, kb1 - 1);  // behind the last block: copied again, and not read
        if constexpr (WIDE) widen_all(wa, a1, sa, MH);
        quadrant(a1, wa, upper, by, wy, Y, [&](auto m) {
            spread(a_reads, m, [&](int q) { read_a(a0[q / 2], stage ^ 1, q / 2, q % 2); });
            spread(copies, m, [&](int q) { copy(after, stage, q); });
        });
        quadrant(a1, wa, upper, bx, wx, X, [&](auto m) {
            spread(b_reads, m, [&](int q) { read_b(by[q / 2], stage ^ 1, yo + q / 2, q % 2); });
            spread(copies, m, [&](int q) { copy(after, stage, kLoads / 2 + q); });
        });
        const int slot = kb + 1 - (kb0 & ~3);
        if ((slot & 31) == 0 && kb + 1 < kb1) {
            meet<kLdsDone>();
            copy_scales(kb + 1);
            meet<kLdsDone>();
        }
        scales(slot);
    };

    // What a tile needs before its first block; done when this returns.
    auto begin = [&] {
        place(tile);
        if (kb0 < kb1) copy_first();
        copy_scales(kb0 & ~3);
        __builtin_amdgcn_s_waitcnt(kCopiesDone);
    };
    begin();
    for (;;) {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[i][j] = f4zero();
        const int r0 = row0, r1 = row1, c0 = n0;
        const long long o0 = out0;
        meet<kLdsDone>();
        if (kb0 < kb1) {
            scales(kb0 & 3);
#pragma unroll
            for (int i = 0; i < 2 * MH; i++) read_a(a0[i / 2], 0, i / 2, i % 2);
#pragma unroll
            for (int i = 0; i < 2 * NH; i++) read_b(b0[i / 2], 0, i / 2, i % 2);
            const integral_constant<int, 0> lower{};
            const integral_constant<int, NH> upper{};
            int kb = kb0;
            for (; kb + 1 < kb1; kb += 2) {
                block(kb, 0, b0, w0, lower, b1, w1, upper);
                block(kb + 1, 1, b1, w1, upper, b0, w0, lower);
            }
            if (kb < kb1) block(kb, 0, b0, w0, lower, b1, w1, upper);
        }
        round++;
        tile = __builtin_amdgcn_readfirstlane(tile_of_round());
        // Copies behind the last block end here at the latest.  The next tile's are
        // here before this one's results are stored, so that its first block need
        // not wait for the stores.
        meet<kAllDone>();
        if (tile >= 0) begin();
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int r = r0 + wm * (TM / WM) + j * 16 + col;
            if (r >= r1) continue;
            T* row = (T*)a.out + o0 + (long long)r * a.out_stride;
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                const f4 u = acc[i][j], w = acc[i + 1][j];
                const float v[8] = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
                const int n = c0 + wn * (TN / WN) + (i >> 1) * 32 + quad * 8;
                if (n < a.n) store_row<T, 8>(a, row, n, v);
            }
        }
        if (tile < 0) break;
    }
#endif
}

// Few rows of A, or few tiles with a long k: up to 16 MT rows by 16 rows of B a
// workgroup, its waves sharing out k, four blocks at a time, and their sums joined
// in LDS in wave order.  With few rows B's bytes bound it, so both operands go
// straight from memory to registers, all of a wave's four blocks under way at
// once, and are widened (one row by 4096 x 4096: 21 us through the tiles above,
// whose 32 workgroups wait for one block after the other; 5.7 us here).
constexpr int kFewWaves = 8;
template <class T, int MT>
__global__ __launch_bounds__(kFewWaves * 64) void product_few_kernel(ProductArgs a)
{
    __shared__ f4 sums[kFewWaves][MT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int waves = blockDim.x >> 6, col = lane & 15, quad = lane >> 4;
    const int tm = blockIdx.x / a.tiles_n, n0 = blockIdx.x % a.tiles_n * 16;
    int expert = 0, row0 = tm * 16 * MT, row1 = a.m;
    if (a.grouping == PRODUCT_ROWS) {
        find_rows(a, tm, 16 * MT, expert, row0, row1);
        if (row0 >= row1) return;
    }
    const int brow = min(n0 + col, a.n - 1);
    const uint8_t* B = a.b + expert * a.b_size + (long long)brow * a.pitch + quad * 16;
    const uint8_t* SB = a.bs + expert * a.bs_size + (long long)(brow >> a.scale_shift) * a.spitch;
    const uint8_t *A[MT], *SA[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const long long r = min(row0 + j * 16 + col, row1 - 1);
        A[j] = a.a + r * a.pitch + quad * 16;
        SA[j] = a.as + r * a.spitch;
    }
    f4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) acc[j] = f4zero();
    const int blocks = a.pitch / 128;
    for (int kb = wave * 4; kb < blocks; kb += waves * 4) {
        const uint32_t sb = *reinterpret_cast<const uint32_t*>(SB + kb);
        uint32_t sa[MT];
        i4v b[4][2], x[4][MT][2];
#pragma unroll
        for (int j = 0; j < MT; j++) sa[j] = *reinterpret_cast<const uint32_t*>(SA[j] + kb);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int at = min(kb + q, blocks - 1) * 128;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                b[q][h] = *reinterpret_cast<const i4v*>(B + at + h * 64);
#pragma unroll
                for (int j = 0; j < MT; j++) x[q][j][h] = *reinterpret_cast<const i4v*>(A[j] + at + h * 64);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (kb + q >= blocks) break;
            const float fb = scale_of(sb >> (8 * q) & 0xff);
            float fa[MT];
#pragma unroll
            for (int j = 0; j < MT; j++) fa[j] = scale_of(sa[j] >> (8 * q) & 0xff);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const bf16x8 wb = widen(b[q][h][2 * p], b[q][h][2 * p + 1], fb);
#pragma unroll
                    for (int j = 0; j < MT; j++)
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            wb, widen(x[q][j][h][2 * p], x[q][j][h][2 * p + 1], fa[j]), acc[j], 0, 0, 0);
                }
        }
    }
#pragma unroll
    for (int j = 0; j < MT; j++) sums[wave][j][lane] = acc[j];
    __syncthreads();
    for (int j = wave; j < MT; j += waves) {
        f4 v = sums[0][j][lane];
        for (int w = 1; w < waves; w++) v += sums[w][j][lane];
        const int r = row0 + j * 16 + col, n = n0 + quad * 4;
        const float o[4] = {v[0], v[1], v[2], v[3]};
        if (r < row1 && n < a.n) store_row<T, 4>(a, (T*)a.out + (long long)r * a.out_stride, n, o);
    }
}

template <class T, int MT>
void few_launch(ProductArgs& a, hipStream_t s)
{
    a.tiles_n = (a.n + 15) / 16;
    const long long row_tiles = a.grouping == PRODUCT_ROWS ? a.m / (16 * MT) + a.experts : (a.m + 16 * MT - 1) / (16 * MT);
    const int waves = std::min(kFewWaves, std::max(1, (a.pitch / 128 + 3) / 4));
    // fewer than 2^32 threads, which is what a grid can have
    require(row_tiles * a.tiles_n <= 0xffffffffll / (waves * 64), "too many tiles for one call");
    product_few_kernel<T, MT><<<(unsigned)(row_tiles * a.tiles_n), waves * 64, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

// 16-row tiles a workgroup where sharing out k is the faster way, 0 where the
// 128 x 128 tiles are: the time of a block of k on a CU, in units of 10 ns, times
// the rounds of workgroups over the CUs.  A few-rows workgroup's goes by the rows
// of A beside its 16 of B, a tile's by the form of its products (dense, k = 4096,
// sharing against tiles: 65 x 512 fp32 7 and 34 us, 128 x 2048 bf16 12.7 and
// 17.0, 300 x 2048 fp32 29.6 and 34.9; 64 x 65536 bf16 164 and 45, 1024 x 2048
// bf16 79 and 23).  Experts are taken to be of equal length, without the empty
// ones that a short plan is bound to have.
int few_tiles(const Fp8ProductOption& o, bool wide)
{
    const long long cus = num_cus(), experts = o.grouping == PRODUCT_DENSE ? 1 : std::min(o.numExperts, o.m);
    const long long rows = (o.m + experts - 1) / experts;
    const long long tiles = experts * ((rows + 127) / 128) * ((o.n + 127) / 128);
    double best = (double)((tiles + cus - 1) / cus) * (wide ? 95 : 45);
    int chosen = 0;
    for (int mt = 1; mt <= 4; mt *= 2) {
        const long long groups = experts * ((rows + 16 * mt - 1) / (16 * mt)) * ((o.n + 15) / 16);
        const double cost = std::max(1.0, (double)groups / cus) * (7 + 0.37 * std::min<long long>(rows, 16 * mt));
        if (cost < best) best = cost, chosen = mt;
    }
    return chosen;
}

template <class T, int TM, int TN, bool WIDE>
void product_launch(ProductArgs& a, hipStream_t s)
{
    a.tiles_n = (a.n + TN - 1) / TN;
    a.tiles_m = (a.m + TM - 1) / TM;
    long long tiles = (long long)a.tiles_m * a.tiles_n;
    if (a.grouping == PRODUCT_ROWS) tiles = ((long long)a.m / TM + a.experts) * a.tiles_n;
    if (a.grouping == PRODUCT_SUM) tiles *= a.experts;
    require(tiles <= 0x7fff0000ll, "too many tiles for one call");
    const long long slots = (long long)num_cus() * (TM * TN > 128 * 128 ? 1 : 2);
    product_kernel<T, TM, TN, WIDE><<<(unsigned)std::min(tiles, slots), 256, 0, s>>>(a);
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
    const int type = o.outType & ~PRODUCT_EXACT;
    require_type(type);
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
    p.relu = o.activation == 1;
    // stores of up to 16 bytes
    p.vec = aligned16(out) && o.outStride * data_bytes(type) % 16 == 0;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        // fp32 results, weight gradients of any type, what is asked for, and products
        // of up to two blocks of k, which their output's bytes bound: there widening
        // costs nothing.
        const bool wide = std::is_same_v<T, float> || o.grouping == PRODUCT_SUM || (o.outType & PRODUCT_EXACT) || p.pitch <= 256;
        if (o.grouping != PRODUCT_SUM) {
            const int few = few_tiles(o, wide);
            if (few == 1) return few_launch<T, 1>(p, s);
            if (few == 2) return few_launch<T, 2>(p, s);
            if (few == 4) return few_launch<T, 4>(p, s);
        }
        if (wide) return product_launch<T, 128, 128, true>(p, s);
        if constexpr (!std::is_same_v<T, float>) {
            // Rounds of tiles over the CUs, by what a round takes: 256 x 256 at 2.5
            // PFLOP/s, two 128 x 128 a CU at 2.2.  Of rows by expert every segment may end
            // inside a tile, which costs the large ones: they are counted with all such
            // ends, the small ones without (128 rows of one in 32 experts, 2048 x 1024:
            // 20 and 8 us).
            const long long cus = num_cus(), experts = o.numExperts;
            auto tiles = [&](int t) {
                const long long n = (o.n + t - 1) / t, m = (o.m + t - 1) / t;
                return (t == 256 && o.grouping == PRODUCT_ROWS ? o.m / t + experts : m) * n;
            };
            const long long large = (tiles(256) + cus - 1) / cus, small = (tiles(128) + 2 * cus - 1) / (2 * cus);
            if (large * 4 * 22 < small * 2 * 25) product_launch<T, 256, 256, false>(p, s);
            else product_launch<T, 128, 128, false>(p, s);
        }
    });
}

}  // namespace graft
