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

// Up to 16 MT rows by 16 rows of B a workgroup, its waves sharing out k, four
// times 128 at a time, and their sums joined in LDS in wave order.
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
        if (o.m <= 16) few_launch<T, 1>(p, s);
        else few_launch<T, 4>(p, s);
    });
}

}  // namespace graft
