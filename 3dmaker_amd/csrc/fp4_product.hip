// Products of 4-bit matrices with a power-of-two scale for each block of 32, for
// gfx950:
//   out[m, n] = sum_kb 2^(sa[m, kb] + sb[n, kb] - 254) sum_{k in kb} a[m, k] b[n, k]
// v_mfma_scale_f32_16x16x128_f8f6f4 takes four blocks of each row with their scales
// and adds exactly as far as fp32 goes (measured: a 1 is kept beside 2^23 in the
// accumulator and 2^-18 beside 36 among the products, and large products that
// cancel leave what is small): 4-bit operands need no widening.
//
// The first MFMA operand is B's rows, the second A's, so that a lane ends with
// four consecutive n of one row m.
#include "product.h"

#include <algorithm>
#include <type_traits>

namespace graft {

namespace {

// A fragment's scale of the lane's block of 32, from the four of its row's 128.
__device__ __forceinline__ int lane_scale(uint32_t four) { return (int)(four >> (8 * ((threadIdx.x & 63) >> 4))); }

__device__ __forceinline__ f4 mfma_fp4(i4v b, int sb, i4v a, int sa, f4 c)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host pass does not know its type check
    const i8v x{b[0], b[1], b[2], b[3], 0, 0, 0, 0}, y{a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, sb, 0, sa);
#else
    return c;
#endif
}

// Few rows of A, or few tiles with a long k: up to 16 MT rows by 16 rows of B a
// workgroup, its waves sharing out k, four times 128 at a time, straight from memory
// to registers, and their sums joined in LDS in wave order.  With few rows B's bytes
// and one round trip bound it: one row by 4096 x 4096 5.2 us, 9 MB at 1.7 TB/s.
constexpr int kFewWaves = 8;
template <class T, int MT>
__global__ __launch_bounds__(kFewWaves * 64) void product4_few_kernel(ProductArgs a)
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
    const uint8_t* SB = a.bs + expert * a.bs_size + (long long)brow * a.spitch;
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
    const int blocks = a.pitch / 64;
    for (int kb = wave * 4; kb < blocks; kb += waves * 4) {
        uint32_t sb[4], sa[4][MT];
        i4v b[4], x[4][MT];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int at = min(kb + q, blocks - 1);
            b[q] = *reinterpret_cast<const i4v*>(B + at * 64);
            sb[q] = *reinterpret_cast<const uint32_t*>(SB + at * 4);
#pragma unroll
            for (int j = 0; j < MT; j++) {
                x[q][j] = *reinterpret_cast<const i4v*>(A[j] + at * 64);
                sa[q][j] = *reinterpret_cast<const uint32_t*>(SA[j] + at * 4);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (kb + q >= blocks) break;
#pragma unroll
            for (int j = 0; j < MT; j++) acc[j] = mfma_fp4(b[q], lane_scale(sb[q]), x[q][j], lane_scale(sa[q][j]), acc[j]);
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
    const int waves = std::min(kFewWaves, std::max(1, (a.pitch / 64 + 3) / 4));
    // fewer than 2^32 threads, which is what a grid can have
    require(row_tiles * a.tiles_n <= 0xffffffffll / (waves * 64), "too many tiles for one call");
    product4_few_kernel<T, MT><<<(unsigned)(row_tiles * a.tiles_n), waves * 64, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

// Large products: TM x TN tiles, persistent workgroups of WM x WN waves.
//
// 256 of k of both operands are a stage; the stages of all of a workgroup's tiles
// are one stream through two places in LDS.  A stage's rows of 128 bytes (whole
// lines, for the L2's requests) are eight 16-byte pieces, permuted by a key of the
// row, so that the 16 rows of a fragment are read from all banks; the copy to LDS
// is linear, so the permutation is in its global addresses.  It is a buffer load,
// which gives rows behind the tile's last, and the pieces behind the last block of
// k, as zeros.  The scales come the same way, 16 bytes of a row for two stages, a
// fragment's rows in the order of their lane columns.
//
// A stage is worked through in its two halves of 128 of k.  A fragment of A is read
// again, for the next half, as soon as it has been multiplied with all of B's; B's
// have two sets of registers.  The one barrier of a stage stands behind the first
// row of matrix instructions of its second half: there all waves have read the
// stage, whose place is free for the next but one, and the next one has been waited
// for, so that a copy has a whole stage's time.  The order is held by the empty asm
// on the accumulators and the scheduling barriers.
//
// B's row of fragment i and lane column c is (i / 2) 32 + (c / 4) 8 + (i % 2) 4 +
// c % 4: a lane ends with eight consecutive columns of two fragments, one 16-byte
// store of 16-bit results.
//
// 256 x 256 by eight waves: 8192 cubed 255 us, 4.3 PFLOP/s (5.0 of zeros: power), its
// matrix cores busy 55% of the time; four waves of 128 x 128 need more registers for
// two halves of A than there are, and spill (750 us).  128 x 128, two workgroups a CU,
// copies twice the bytes for the same work (342 us).  Rows of 64 bytes in four places
// made twice the L2 requests (326 us), copies in a burst behind the barrier instead of
// between the matrix instructions 261.
template <class T, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void product4_kernel(ProductArgs a)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host pass needs the kernel's name alone
    using std::integral_constant;
    constexpr int kWaves = WM * WN, MT = TM / WM / 16, NT = TN / WN / 16, GA = MT / 4;
    constexpr int kPlace = (TM + TN) * 128, kScales = (TM + TN) * 16, kCopies = (TM + TN) / 8 / kWaves;
    constexpr int kStores = MT * NT / (sizeof(T) == 4 ? 1 : 2);
    static_assert(MT % 4 == 0 && NT == 4 && kWaves % 2 == 0 && TM % (8 * kWaves) == 0 && TN % (8 * kWaves) == 0 &&
                  TM + TN == 64 * kWaves && TM % 64 == 0, "whole fragments and copies");
    // One array: with two, the compiler waits for all copies before each LDS read.
    __shared__ __attribute__((aligned(128))) uint8_t lds[2 * kPlace + 2 * kScales + 1028 * 4];
    uint8_t* const scale_lds = lds + 2 * kPlace;
    int* const starts = reinterpret_cast<int*>(scale_lds + 2 * kScales);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave / WN, wn = wave % WN, col = lane & 15, quad = lane >> 4;

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
    }
    // Workgroups go round the XCDs; each XCD works through a range of tiles of its own.
    const int total = row_tile_count * a.tiles_n;
    const int xcd = blockIdx.x & 7, x0 = xcd * (total / 8) + min(xcd, total % 8), xn = total / 8 + (xcd < total % 8);
    const int per_round = (gridDim.x + 7 - xcd) / 8, rank = blockIdx.x >> 3;
    if (rank >= xn) return;
    const int rounds = (xn - rank + per_round - 1) / per_round;

    struct Tile {
        int row0, row1, n0, expert;
    };
    auto tile_of = [&](int round) {  // four row tiles by all columns at a time: what an XCD has in flight shares its L2
        const int t = x0 + rank + round * per_round;
        const int group = t / (4 * a.tiles_n), first = group * 4, rows = min(4, row_tile_count - first);
        const int in = t - first * a.tiles_n, tm = first + in % rows;
        Tile r{tm * TM, a.m, in / rows * TN, 0};
        if (a.grouping == PRODUCT_ROWS) {
            if (a.experts <= 64) {
                r.expert = __ffsll((unsigned long long)__ballot(seg_end > tm)) - 1;
                r.row1 = __builtin_amdgcn_readlane(seg_hi, r.expert);
                r.row0 = __builtin_amdgcn_readlane(seg_lo, r.expert);
                r.row0 += (tm - __builtin_amdgcn_readlane(seg_end, r.expert) + (r.row1 - r.row0 + TM - 1) / TM) * TM;
            } else {
                r.expert = __builtin_amdgcn_readfirstlane(expert_of_tile(starts, a.experts, tm));
                const int lo = min(max(a.offsets[r.expert], 0), a.m);
                r.row0 = __builtin_amdgcn_readfirstlane(lo + (tm - starts[r.expert]) * TM);
                r.row1 = __builtin_amdgcn_readfirstlane(min(max(a.offsets[r.expert + 1], lo), a.m));
            }
        }
        return r;
    };

    // What is copied: a stage of a tile, ahead of what is worked on.
    const int blocks = a.pitch / 64, stages = (blocks + 1) / 2;
    int copy_round = 0, copy_stage = 0, copy_scales = 0;  // and the place of its scales
    __amdgpu_buffer_rsrc_t ra, rb, rs;
    const bool scales_of_a = wave * 64 < TM;  // the wave's 64 rows of scales
    auto aim = [&] {
        const Tile t = tile_of(copy_round);
        const int flags = 0x00020000, rows_a = min(TM, t.row1 - t.row0), rows_b = min(TN, a.n - t.n0);
        auto of = [&](const uint8_t* p, long long row, int pitch, int rows) {
            return __builtin_amdgcn_make_buffer_rsrc((void*)(p + row * pitch), 0, rows * pitch, flags);
        };
        ra = of(a.a, t.row0, a.pitch, rows_a);
        rb = of(a.b + t.expert * a.b_size, t.n0, a.pitch, rows_b);
        rs = scales_of_a ? of(a.as, t.row0, a.spitch, rows_a) : of(a.bs + t.expert * a.bs_size, t.n0, a.spitch, rows_b);
    };
    // A wave's copy is of 8 rows of 128 bytes.  Keys: A's rows row % 8, B's row % 4 + 4 (row / 8 % 2).
    const int copy_row = wave * 8 + (lane >> 3);
    const int piece_a = (lane & 7) ^ (lane >> 3), piece_b = (lane & 7) ^ ((lane >> 3 & 3) | (wave & 1) << 2);
    const uint32_t from_a = (uint32_t)copy_row * a.pitch + piece_a * 16, from_b = (uint32_t)copy_row * a.pitch + piece_b * 16;
    // Lane 16 i + c copies the scales of fragment i's row of lane column c.
    const int scale_col = lane & 15, scale_i = lane >> 4;
    const int scale_row = scales_of_a ? wave * 64 + scale_i * 16 + scale_col
                                      : wave * 64 - TM + (scale_i >> 1) * 32 + (scale_col >> 2) * 8 + (scale_i & 1) * 4 + (scale_col & 3);
    const uint32_t from_s = (uint32_t)scale_row * a.spitch;
    auto copy = [&](int place, int i) {  // A's and B's rows
        const bool of_a = i * kWaves * 8 < TM, none = 2 * copy_stage + 1 >= blocks && (of_a ? piece_a : piece_b) >= 4;
        const uint32_t at = (of_a ? from_a : from_b) + (uint32_t)(i * kWaves * 8 - (of_a ? 0 : TM)) * a.pitch + copy_stage * 128;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            of_a ? ra : rb, (__attribute__((address_space(3))) void*)(lds + place * kPlace + (i * kWaves + wave) * 1024), 16,
            none ? 0x80000000u : at, 0, 0, 0);
    };
    auto copy_scales_now = [&] {  // of this stage and the next
        if (copy_stage & 1) return;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void*)(scale_lds + copy_scales * kScales + wave * 1024), 16,
            from_s + copy_stage * 8, 0, 0, 0);
        copy_scales ^= 1;
    };
    auto advance = [&]() {  // false behind the last tile
        if (copy_stage + 1 < stages) copy_stage++;
        else if (copy_round + 1 < rounds) {
            copy_stage = 0;
            copy_round++;
            aim();
        } else return false;
        return true;
    };

    f4 acc[NT][MT];
    i4v fa[MT], b0[NT], b1[NT], raw[GA + 1];
    int sa0[GA], sa1[GA], sb0, sb1;
    // Half h of a row (pieces quad or quad + 4): 64 to and fro.
    const int at_a = (wm * (TM / WM) + col) * 128 + (quad ^ (col & 7)) * 16;
    const int at_b = (TM + wn * (TN / WN) + (col >> 2) * 8 + (col & 3)) * 128 + (quad ^ (col & 7)) * 16;
    auto read_a = [&](int place, int h, int i) {
        fa[i] = *reinterpret_cast<const i4v*>(lds + place * kPlace + (at_a ^ 64 * h) + i * 2048);
    };
    auto read_b = [&](i4v& f, int place, int h, int i) {
        f = *reinterpret_cast<const i4v*>(lds + place * kPlace + (at_b ^ 64 * h) + (i >> 1) * 4096 + (i & 1) * 512);
    };
    // Four bytes of four fragments' scales, of half `half` (0..3) of two stages; then
    // the lane's byte of each.
    const int group_a = wm * (TM / WM / 64), group_b = TM / 64 + wn * (TN / WN / 64);
    auto read_scales = [&](int place, int half, int g) {
        const uint8_t* p = scale_lds + place * kScales + (g < GA ? group_a + g : group_b) * 1024 + col * 16 + half * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) raw[g][i] = *reinterpret_cast<const int*>(p + i * 256);
    };
    const uint32_t low = (uint32_t)(quad | (4 + quad) << 8) | 0x0c0c0000u, high = (uint32_t)(quad << 16 | (4 + quad) << 24) | 0x0c0cu;
    auto scales = [&](int g, bool there) -> int {  // behind the last block values are zero, and must not become NaN
        const i4v v = raw[g];
        return there ? (int)(__builtin_amdgcn_perm(v[1], v[0], low) | __builtin_amdgcn_perm(v[3], v[2], high)) : 0x7f7f7f7f;
    };

    int place = 0, scale_place = 0;  // of the stage that is worked on
    int stage = 0;                   // of its tile
    bool stored = false, more = true;
    auto copy_stage_now = [&](int to) {
#pragma unroll
        for (int i = 0; i < kCopies; i++) copy(to, i);
        copy_scales_now();
    };
    // Half H of the stage: its fragments are in fa and bx, its scales in sax and sbx.
    auto half = [&](auto H, auto& bx, auto& sax, auto& sbx, auto& by, auto& say, auto& sby) {
        constexpr int h = decltype(H)::value;
        const int to = h ? place ^ 1 : place;  // what is read for the next half
        const int next = h ? (stage + 1 == stages ? 0 : stage + 1) : stage;
        if (h && (next & 1) == 0) scale_place ^= 1;
        each<MT>([&](auto I) {
            constexpr int i = decltype(I)::value;
            each<NT>([&](auto J) {
                constexpr int j = decltype(J)::value;
                f4& c = acc[j][i];
                const i8v p{bx[j][0], bx[j][1], bx[j][2], bx[j][3], 0, 0, 0, 0};
                const i8v q{fa[i][0], fa[i][1], fa[i][2], fa[i][3], 0, 0, 0, 0};
                c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, q, c, 4, 4, j, sbx, i % 4, sax[i / 4]);
                asm volatile("" : "+v"(c));
                constexpr int n = 2 * (i - 1) + (j & 1);  // of the next half's B
                constexpr int slots = (MT - 1) * NT, at = (i - 1) * NT + j;
                constexpr int m = (at * kCopies + slots - 1) / slots, m1 = ((at + 1) * kCopies + slots - 1) / slots;  // copies
                if constexpr (i > 0 && j < 2 && n < NT) read_b(by[n], to, 1 - h, n);
                if constexpr (h && i > 0 && m < m1) copy(place, m);
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (h && i == 0) {
                // The next stage's copies, behind which a tile's results may be under way.
                if (stored) __builtin_amdgcn_s_waitcnt((kStores & 15) | (kStores >> 4) << 14 | 0x0f70);
                else __builtin_amdgcn_s_waitcnt(kCopiesDone);
                meet<kLdsDone>();
                stored = false;
            }
            read_a(to, 1 - h, i);
            if constexpr (i == MT - 3 || (MT == 4 && i == 1)) {
#pragma unroll
                for (int g = 0; g <= GA; g++) read_scales(scale_place, (next & 1) * 2 + 1 - h, g);
            }
            if constexpr (i == MT - 1) {
                const bool there = 2 * next + 1 - h < blocks;
#pragma unroll
                for (int g = 0; g < GA; g++) say[g] = scales(g, there);
                sby = scales(GA, there);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        if (h) {
            if (more) {
                copy_scales_now();
                more = advance();
            }
            place ^= 1;
            stage = next;
        }
    };

    aim();
    copy_stage_now(0);
    more = advance();
    if (more) {
        copy_stage_now(1);
        more = advance();
    }
    __builtin_amdgcn_s_waitcnt(kCopiesDone);
    meet<kLdsDone>();
#pragma unroll
    for (int i = 0; i < MT; i++) read_a(0, 0, i);
#pragma unroll
    for (int i = 0; i < NT; i++) read_b(b0[i], 0, 0, i);
#pragma unroll
    for (int g = 0; g <= GA; g++) read_scales(0, 0, g);
#pragma unroll
    for (int g = 0; g < GA; g++) sa0[g] = scales(g, true);
    sb0 = scales(GA, true);
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[i][j] = f4zero();
    };
    auto store = [&](int round) {
        const Tile t = tile_of(round);
        const bool whole = a.vec && t.row0 + TM <= t.row1 && t.n0 + TN <= a.n;
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int r = t.row0 + wm * (TM / WM) + j * 16 + col;
            if (r >= t.row1) continue;
            T* row = (T*)a.out + (long long)r * a.out_stride;
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                const f4 u = acc[i][j], w = acc[i + 1][j];
                const float v[8] = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
                const int n = t.n0 + wn * (TN / WN) + (i >> 1) * 32 + quad * 8;
                if (n < a.n) store_row<T, 8>(a, row, n, v);
            }
        }
        stored = whole;  // others are not kStores
    };
    clear();
    for (int round = 0;;) {
        half(integral_constant<int, 0>{}, b0, sa0, sb0, b1, sa1, sb1);
        half(integral_constant<int, 1>{}, b1, sa1, sb1, b0, sa0, sb0);
        if (stage == 0) {
            store(round);
            if (++round == rounds) break;
            clear();
        }
    }
    __builtin_amdgcn_s_waitcnt(kAllDone);  // no copy to LDS outlives the workgroup
#endif
}

template <class T, int TM, int TN, int WM, int WN>
void product_launch(ProductArgs& a, hipStream_t s)
{
    a.tiles_n = (a.n + TN - 1) / TN;
    a.tiles_m = (a.m + TM - 1) / TM;
    const long long tiles =
        (a.grouping == PRODUCT_ROWS ? (long long)a.m / TM + a.experts : (long long)a.tiles_m) * a.tiles_n;
    require(tiles <= 0x7fff0000ll, "too many tiles for one call");
    const long long slots = (long long)num_cus() * (8 / (WM * WN));
    product4_kernel<T, TM, TN, WM, WN><<<(unsigned)std::min(tiles, slots), WM * WN * 64, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

// The form by what it takes for 128 of k, in units of 10 ns: rows of a workgroup
// that shares out k (16, 32, 64), or of a tile (128, 256).  Measured (dense, k =
// 4096, us sharing 16, 32 or 64 rows and in tiles of 128 and 256): 16 x 8192 9.6,
// 10.3, 11.7, 14.2, 25.7; 128 x 2048 17.0, 13.1, 11.6, 14.8, 27.3; 256 x 2048 31,
// 24, 21, 14.9, 28.4; 4096 x 2048 446, 336, 281, 25.6, 35.8; 4096 x 8192 1775, 1332,
// 1113, 93, 80.  Workgroups that share k take 5 and 6.1 for each 16 rows, as many at
// a time as there are CUs; a CU's tiles of 128 37, or 44 the only one; a round of
// tiles of 256 112, or 85 if there is one.  Of rows by expert, every segment may
// end inside a large tile: they are counted with all such ends, the others without
// (19,200 rows of 64 experts, 2048 x 1024: 44 us in tiles of 128, 52 of 256; 96,000
// 223 and 188).  Experts are taken to be of equal length, without the empty ones
// that a short plan is bound to have.
int form_of(const Fp4ProductOption& o)
{
    const long long cus = num_cus(), experts = o.grouping == PRODUCT_DENSE ? 1 : std::min(o.numExperts, o.m);
    const long long rows = (o.m + experts - 1) / experts;
    auto up = [](long long n, long long d) { return (n + d - 1) / d; };
    const long long small = experts * up(rows, 128) * up(o.n, 128);
    const long long large = (o.grouping == PRODUCT_DENSE ? up(o.m, 256) : o.m / 256 + o.numExperts) * up(o.n, 256);
    double best = small <= cus ? 44 : 37.0 * up(small, cus);
    int form = 128;
    const double in_large = large <= cus ? 85 : 112.0 * up(large, cus);
    if (in_large < best) best = in_large, form = 256;
    for (int mt = 1; mt <= 4; mt *= 2) {
        const long long groups = experts * up(rows, 16 * mt) * up(o.n, 16);
        const double cost = std::max(1.0, (double)groups / cus) * (5 + 6.1 * mt);
        if (cost < best) best = cost, form = 16 * mt;
    }
    return form;
}

}  // namespace

void fp4_product(const Fp4ProductOption& o, const uint8_t* a, const uint8_t* a_scales, const uint8_t* b,
                 const uint8_t* b_scales, const int* offsets, void* out, hipStream_t s)
{
    require(o.m >= 0 && o.m <= kMaxRows, "m must be 0..2^30");
    require(o.n >= 1 && o.n <= 1 << 22 && o.k >= 1 && o.k <= 1 << 22, "n and k must be 1..2^22");
    require(o.grouping == PRODUCT_DENSE || o.grouping == PRODUCT_ROWS, "unknown grouping");
    require(o.numExperts >= 1 && o.numExperts <= 1024 && (o.grouping != PRODUCT_DENSE || o.numExperts == 1),
            "numExperts must be 1..1024, and 1 for a dense product");
    require(o.activation == 0 || o.activation == 1, "unknown activation");
    require_type(o.outType);
    require(o.outStride >= o.n, "outStride must be at least n");
    require((o.grouping == PRODUCT_DENSE) == !offsets, "offsets go with grouped products");
    if (o.m == 0) return;
    require(out && a && a_scales && b && b_scales, "null argument");
    require(aligned16(a) && aligned16(b) && ((uintptr_t)a_scales & 3) == 0 && ((uintptr_t)b_scales & 3) == 0,
            "4-bit matrices must be 16-byte aligned and scales 4-byte aligned");
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
    p.pitch = fp4_pitch(o.k);
    p.spitch = fp4_scale_pitch(o.k);
    p.b_size = (long long)o.n * p.pitch;
    p.bs_size = (long long)o.n * p.spitch;
    p.out_stride = o.outStride;
    p.relu = o.activation == 1;
    // stores of up to 16 bytes
    p.vec = aligned16(out) && o.outStride * data_bytes(o.outType) % 16 == 0;
    with_type(o.outType, [&](auto zero) {
        using T = decltype(zero);
        switch (form_of(o)) {
            case 16: return few_launch<T, 1>(p, s);
            case 32: return few_launch<T, 2>(p, s);
            case 64: return few_launch<T, 4>(p, s);
            case 128: return product_launch<T, 128, 128, 2, 2>(p, s);
            default: return product_launch<T, 256, 256, 2, 4>(p, s);
        }
    });
}

}  // namespace graft
