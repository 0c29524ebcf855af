// Quantising to e4m3 with a power-of-two scale for each block of 128, for
// gfx950 (layout: experts_abi.h).
//
//   s = the smallest power of two with max |x| <= 448 s,   q = e4m3(x / s)
//
// The scale comes from the bits of the block's largest magnitude (exponent - 8,
// one more where its mantissa is above that of 448 = 1.75 * 2^8) and x / s is a
// change of exponent: the one rounding is the conversion's.
#include "experts.h"
#include "lanes.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kQuantThreads = 256;

struct QuantArgs {
    const void* src;
    const int* order;
    const float* weights;
    const void* gate;
    uint8_t *q, *scales, *qt, *scalesT;
    int rows, cols, slots_per_row, src_rows;
    int pitch, spitch, pitch_t, spitch_t;
    long long stride, batch_stride, gate_stride;
    long long wg0;  // the launch's first workgroup (rows only)
    bool vec;  // source rows are whole 16-byte pieces of eight columns
};

// Bits of |v|: larger floats have larger ones.
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

constexpr uint32_t kInfinity = 0x7f800000u;

// Largest of a thread's values with infinities and NaN left out: only where a
// block's largest is one, which it seldom is.
template <int N, class F>
__device__ __forceinline__ uint32_t largest_finite(F&& value)
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t m = magnitude(value(i));
        top = m < kInfinity ? max(top, m) : top;
    }
    return top;
}

// Scale byte of a block from the bits of its largest finite magnitude.
__device__ __forceinline__ int scale_byte(uint32_t top)
{
    const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}

__device__ __forceinline__ float inverse_scale(int byte)
{
    return __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23);
}

// Infinities and NaN become NaN: the conversion has no infinity, and nothing
// finite is above 448 here.
__device__ __forceinline__ uint32_t fp8x4(const float* v, float inverse)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, w, true);
    return (uint32_t)w;
}

// Scale byte of the 128 values of 16 lanes, eight each.
__device__ __forceinline__ int row_byte(const float (&v)[8])
{
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, magnitude(v[j]));
    top = lanes_umax<16>(top);
    if (top >= kInfinity) {
        top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, magnitude(v[j]) < kInfinity ? magnitude(v[j]) : 0u);
        top = lanes_umax<16>(top);
    }
    return scale_byte(top);
}

// Where a quantised row comes from; weight 0 and no source where there is none.
struct Source {
    long long row;
    float weight;
    bool there;
};

__device__ __forceinline__ Source source_of(const QuantArgs& a, int row)
{
    Source s{row, 1.0f, row < a.rows};
    if (a.order) {
        const int slot = s.there ? a.order[row] : -1;
        s.row = slot / a.slots_per_row;
        s.there = slot >= 0 && s.row < a.src_rows;
        if (a.weights && s.there) s.weight = a.weights[slot];
    }
    if (!s.there) s.row = 0;
    return s;
}

// Columns col .. col + 7 of R quantised rows: all rows' loads are under way
// before the first is used (rows without a source load the first row, columns
// behind the last the first ones).
template <class T, int R>
__device__ __forceinline__ void load_rows(float (&v)[R][8], const QuantArgs& a, const T* src, const int (&row)[R],
                                          const int (&col)[R])
{
    Source s[R];
#pragma unroll
    for (int i = 0; i < R; i++) s[i] = source_of(a, row[i]);
    if (a.vec) {
        constexpr int N = 16 / sizeof(T), P = 8 / N;
        Vec<T, N> raw[R][P];
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int q = 0; q < P; q++)
                raw[i][q] = *reinterpret_cast<const Vec<T, N>*>(src + s[i].row * a.stride + (col[i] < a.cols ? col[i] : 0) + q * N);
#pragma unroll
        for (int i = 0; i < R; i++) {
            const bool there = s[i].there && col[i] < a.cols;
#pragma unroll
            for (int q = 0; q < P; q++) {
                const Vec<uint32_t, 4> bits = __builtin_bit_cast(Vec<uint32_t, 4>, raw[i][q]);
                const Vec<uint32_t, 4> kept{there ? bits[0] : 0u, there ? bits[1] : 0u, there ? bits[2] : 0u,
                                            there ? bits[3] : 0u};
                const Vec<T, N> w = __builtin_bit_cast(Vec<T, N>, kept);
#pragma unroll
                for (int j = 0; j < N; j++) v[i][q * N + j] = (float)w[j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 8; j++)
                v[i][j] = s[i].there && col[i] + j < a.cols ? (float)src[s[i].row * a.stride + col[i] + j] : 0.0f;
    }
    if (a.weights) {
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] *= s[i].weight;  // 1 where there is no source, and zeros
    }
    if (a.gate) {
        const T* gate = (const T*)a.gate;
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 8; j++)
                v[i][j] = s[i].there && col[i] + j < a.cols &&
                                  (float)gate[(long long)row[i] * a.gate_stride + col[i] + j] > 0.0f
                              ? v[i][j] : 0.0f;
    }
}

// Rows only: 16 lanes a (row, block), UNITS of them 16 apart.  Four at a time
// once there are enough for all CUs (65,536 x 1,024 bf16 gathered: 45 us, 4.5 TB/s
// of its 201 MB; 50 with one, whose loads wait for one another's row numbers).
template <class T, int UNITS>
__global__ __launch_bounds__(kQuantThreads) void quant_rows_kernel(QuantArgs a)
{
    const uint32_t blocks = a.pitch / 128;
    const unsigned long long first = (unsigned long long)(a.wg0 + blockIdx.x) * (16 * UNITS);
    const uint32_t row0 = (uint32_t)(first / blocks), in0 = (uint32_t)(first % blocks);
    const T* src = (const T*)a.src + (long long)blockIdx.y * a.batch_stride;
    float v[UNITS][8];
    int row[UNITS], col[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const uint32_t in = in0 + u * 16 + threadIdx.x / 16, down = in / blocks;
        row[u] = (int)(row0 + down);
        col[u] = (int)(in - down * blocks) * 128 + (threadIdx.x & 15) * 8;
    }
    load_rows(v, a, src, row, col);
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const int byte = row_byte(v[u]);
        if (row[u] >= a.rows) continue;
        const float inv = inverse_scale(byte);
        const long long r = (long long)blockIdx.y * a.rows + row[u];
        *reinterpret_cast<Vec<uint32_t, 2>*>(a.q + r * a.pitch + col[u]) =
            Vec<uint32_t, 2>{fp8x4(v[u], inv), fp8x4(v[u] + 4, inv)};
        if ((threadIdx.x & 15) == 0) a.scales[r * a.spitch + col[u] / 128] = (uint8_t)byte;
    }
}

// A tile of 128 x 128 in registers (thread: 8 rows by 8 columns), as rows,
// as columns or both.  The transposed bytes cross LDS in pieces of 8, piece ty of
// column c at ty ^ (c / 8): a wave's writes, one column of every eight, spread
// over the banks.  33,792 x 2,048 fp16 gathered and weighted, both ways: 64 us,
// 4.2 TB/s of its 272 MB; behind a gate 193 us, whose elements are loaded one by
// one.  Weights of eight experts, 2,048 x 1,024 fp32 in blocks, both ways: 18 us.
template <class T, bool BLOCKS>
__global__ __launch_bounds__(kQuantThreads) void quant_tile_kernel(QuantArgs a)
{
    __shared__ uint32_t tops[16][128];
    __shared__ uint32_t wave_top[4];
    __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int r0 = blockIdx.x * 128, c0 = blockIdx.y * 128;
    const T* src = (const T*)a.src + (long long)blockIdx.z * a.batch_stride;
    float v[8][8];
    int row_of[8], col_of[8];
#pragma unroll
    for (int i = 0; i < 8; i++) row_of[i] = r0 + ty * 8 + i, col_of[i] = c0 + tx * 8;
    load_rows(v, a, src, row_of, col_of);
    int block_byte = 0;
    if (BLOCKS) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) top = max(top, magnitude(v[i][j]));
        if (lanes_umax<64>(top) >= kInfinity) top = largest_finite<64>([&](int i) { return v[i / 8][i % 8]; });
        top = lanes_umax<64>(top);
        if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
        __syncthreads();
        block_byte = scale_byte(max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3])));
    }
    if (a.q) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            int byte = block_byte;
            if (!BLOCKS) byte = row_byte(v[i]);
            if (row_of[i] >= a.rows) continue;
            const float inv = inverse_scale(byte);
            const long long r = (long long)blockIdx.z * a.rows + row_of[i];
            *reinterpret_cast<Vec<uint32_t, 2>*>(a.q + r * a.pitch + c0 + tx * 8) =
                Vec<uint32_t, 2>{fp8x4(v[i], inv), fp8x4(v[i] + 4, inv)};
            if (!BLOCKS && tx == 0) a.scales[r * a.spitch + blockIdx.y] = (uint8_t)byte;
        }
        if (BLOCKS && threadIdx.x == 0)
            a.scales[((long long)blockIdx.z * gridDim.x + blockIdx.x) * a.spitch + blockIdx.y] = (uint8_t)block_byte;
    }
    if (!a.qt) return;
    if (!BLOCKS) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) top = max(top, magnitude(v[i][j]));
            if (top >= kInfinity) top = largest_finite<8>([&](int i) { return v[i][j]; });
            tops[ty][j * 16 + tx] = top;  // column tx * 8 + j
        }
        __syncthreads();
        if (threadIdx.x < 128) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) top = max(top, tops[i][threadIdx.x]);
            tops[0][threadIdx.x] = top;  // its column is this thread's alone
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int byte = BLOCKS ? block_byte : scale_byte(tops[0][j * 16 + tx]);
        const float inv = inverse_scale(byte);
        const float c[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
        *reinterpret_cast<Vec<uint32_t, 2>*>(&tile[(tx * 8 + j) * 128 + ((ty ^ tx) * 8)]) =
            Vec<uint32_t, 2>{fp8x4(c, inv), fp8x4(c + 4, inv)};
        const int col = c0 + tx * 8 + j;
        if (!BLOCKS && ty == 0 && col < a.cols)
            a.scalesT[((long long)blockIdx.z * a.cols + col) * a.spitch_t + blockIdx.x] = (uint8_t)byte;
    }
    if (BLOCKS && threadIdx.x == 0)
        a.scalesT[((long long)blockIdx.z * gridDim.y + blockIdx.y) * a.spitch_t + blockIdx.x] = (uint8_t)block_byte;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int unit = i * kQuantThreads + threadIdx.x, c = unit >> 3, piece = (unit & 7) * 2, key = c >> 3;
        if (c0 + c >= a.cols) continue;
        const Vec<uint32_t, 4> w = *reinterpret_cast<const Vec<uint32_t, 4>*>(&tile[c * 128 + (((piece ^ key) & ~1) * 8)]);
        const Vec<uint32_t, 4> swapped{w[2], w[3], w[0], w[1]};
        *reinterpret_cast<Vec<uint32_t, 4>*>(a.qt + ((long long)blockIdx.z * a.cols + c0 + c) * a.pitch_t + r0 + piece * 8) =
            key & 1 ? swapped : w;
    }
}

}  // namespace

void fp8_quantize(const Fp8QuantOption& o, const void* src, const int* order, const float* weights, const void* gate,
                  uint8_t* q, uint8_t* scales, uint8_t* qt, uint8_t* scalesT, hipStream_t s)
{
    require(o.rows >= 0 && o.rows <= kMaxRows && o.srcRows >= 0, "rows must be 0..2^30 and srcRows >= 0");
    require(o.cols >= 1 && o.cols <= 1 << 22, "cols must be 1..2^22");
    require(o.batch >= 1 && o.batch <= 65535, "batch must be 1..65535");
    require(o.blockRows == 1 || o.blockRows == 128, "blockRows must be 1 or 128");
    require_type(o.srcType);
    require(o.srcStride >= o.cols, "srcStride must be at least cols");
    require(o.batch == 1 || o.srcBatchStride >= 0, "srcBatchStride must be >= 0");
    require(!gate || o.gateStride >= o.cols, "gateStride must be at least cols");
    require(!order || (o.slotsPerRow >= 1 && o.batch == 1), "an order needs slotsPerRow >= 1 and a batch of 1");
    require(!weights || order, "weights need an order");
    require(!gate || o.batch == 1, "a gate needs a batch of 1");
    require(order || o.srcRows >= o.rows, "srcRows must be at least rows");
    require((q || qt) && !q == !scales && !qt == !scalesT, "q or qt, each with its scales");
    require(aligned16(q) && aligned16(qt), "q and qt must be 16-byte aligned");
    if (o.rows == 0) return;
    require(src, "null argument");
    QuantArgs a{};
    a.src = src;
    a.order = order;
    a.weights = weights;
    a.gate = gate;
    a.q = q;
    a.scales = scales;
    a.qt = qt;
    a.scalesT = scalesT;
    a.rows = o.rows;
    a.cols = o.cols;
    a.slots_per_row = o.slotsPerRow;
    a.src_rows = o.srcRows;
    a.pitch = fp8_pitch(o.cols);
    a.spitch = fp8_scale_pitch(o.cols);
    a.pitch_t = fp8_pitch(o.rows);
    a.spitch_t = fp8_scale_pitch(o.rows);
    a.stride = o.srcStride;
    a.batch_stride = o.srcBatchStride;
    a.gate_stride = o.gateStride;
    const int bytes = data_bytes(o.srcType);
    auto fits = [&](const void* p, long long stride) { return aligned16(p) && stride * bytes % 16 == 0; };
    a.vec = o.srcRows > 0 && o.cols % 8 == 0 && fits(src, o.srcStride) &&
            (o.batch == 1 || o.srcBatchStride * bytes % 16 == 0);
    const int cb = a.pitch / 128, rb = a.pitch_t / 128;
    with_type(o.srcType, [&](auto zero) {
        using T = decltype(zero);
        if (o.blockRows == 128) quant_tile_kernel<T, true><<<dim3(rb, cb, o.batch), kQuantThreads, 0, s>>>(a);
        else if (qt) quant_tile_kernel<T, false><<<dim3(rb, cb, o.batch), kQuantThreads, 0, s>>>(a);
        else {
            const long long units = (long long)o.rows * cb;
            const bool many = units * o.batch >= 64ll * 8 * num_cus();
            in_launches((units + (many ? 63 : 15)) / (many ? 64 : 16), kQuantThreads, [&](long long first, unsigned wgs) {
                a.wg0 = first;
                if (many) quant_rows_kernel<T, 4><<<dim3(wgs, o.batch), kQuantThreads, 0, s>>>(a);
                else quant_rows_kernel<T, 1><<<dim3(wgs, o.batch), kQuantThreads, 0, s>>>(a);
            });
        }
    });
    GRAFT_LAUNCH_CHECK();
}

}  // namespace graft
