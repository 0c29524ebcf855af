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
    bool vec;  // source (and gate) rows take 16-byte loads
};

__device__ __forceinline__ uint32_t magnitude(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;  // infinities and NaN do not set the scale
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

__device__ __forceinline__ float fp8_operand(float v, float inverse)
{
    return fabsf(v) < INFINITY ? v * inverse : __builtin_nanf("");
}

__device__ __forceinline__ uint32_t fp8x4(const float* v, float inverse)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_operand(v[0], inverse), fp8_operand(v[1], inverse), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_operand(v[2], inverse), fp8_operand(v[3], inverse), w, true);
    return (uint32_t)w;
}

// Eight consecutive values of a row, zero from `n` on.
template <class T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, int n, bool vec)
{
    if (vec && n >= 8) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            const Vec<T, N> w = *reinterpret_cast<const Vec<T, N>*>(p + i);
#pragma unroll
            for (int j = 0; j < N; j++) v[i + j] = (float)w[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? (float)p[i] : 0.0f;
    }
}

// Columns col .. col + 7 of quantised row `row`: gathered, weighted, gated.
template <class T>
__device__ __forceinline__ void load_row8(float (&v)[8], const QuantArgs& a, const T* src, int row, int col)
{
    const int n = a.cols - col;
    long long from = row;
    float w = 1.0f;
    bool there = row < a.rows && n > 0;
    if (there && a.order) {
        const int slot = a.order[row];
        from = slot / a.slots_per_row;
        there = slot >= 0 && from < a.src_rows;
        if (there && a.weights) w = a.weights[slot];
    }
    if (!there) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = 0.0f;
        return;
    }
    load8(v, src + from * a.stride + col, n, a.vec);
    if (a.weights) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= w;
    }
    if (a.gate) {
        float g[8];
        load8(g, (const T*)a.gate + (long long)row * a.gate_stride + col, n, a.vec);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = g[i] > 0.0f ? v[i] : 0.0f;
    }
}

// Rows only: 16 lanes a (row, block).
template <class T>
__global__ __launch_bounds__(kQuantThreads) void quant_rows_kernel(QuantArgs a)
{
    const int blocks = a.pitch / 128;
    const long long unit = (long long)blockIdx.x * (kQuantThreads / 16) + threadIdx.x / 16;
    const int row = (int)(unit / blocks), block = (int)(unit % blocks), col = block * 128 + (threadIdx.x & 15) * 8;
    const T* src = (const T*)a.src + (long long)blockIdx.y * a.batch_stride;
    float v[8];
    load_row8(v, a, src, row, col);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, magnitude(v[i]));
    const int byte = scale_byte(lanes_umax<16>(top));
    if (row >= a.rows) return;
    const float inv = inverse_scale(byte);
    const long long r = (long long)blockIdx.y * a.rows + row;
    *reinterpret_cast<Vec<uint32_t, 2>*>(a.q + r * a.pitch + col) = Vec<uint32_t, 2>{fp8x4(v, inv), fp8x4(v + 4, inv)};
    if ((threadIdx.x & 15) == 0) a.scales[r * a.spitch + block] = (uint8_t)byte;
}

// A tile of 128 x 128 in registers (thread: 8 rows by 8 columns), as rows,
// as columns or both.
template <class T, bool BLOCKS>
__global__ __launch_bounds__(kQuantThreads) void quant_tile_kernel(QuantArgs a)
{
    __shared__ uint32_t tops[16][128];
    __shared__ uint32_t wave_top[4];
    __shared__ __attribute__((aligned(16))) uint8_t tile[128][144];  // transposed bytes, rows 16-byte aligned
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int r0 = blockIdx.x * 128, c0 = blockIdx.y * 128;
    const T* src = (const T*)a.src + (long long)blockIdx.z * a.batch_stride;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; i++) load_row8(v[i], a, src, r0 + ty * 8 + i, c0 + tx * 8);
    int block_byte = 0;
    if (BLOCKS) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) top = max(top, magnitude(v[i][j]));
        top = lanes_umax<64>(top);
        if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
        __syncthreads();
        block_byte = scale_byte(max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3])));
    }
    if (a.q) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int row = r0 + ty * 8 + i;
            int byte = block_byte;
            if (!BLOCKS) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) top = max(top, magnitude(v[i][j]));
                byte = scale_byte(lanes_umax<16>(top));
            }
            if (row >= a.rows) continue;
            const float inv = inverse_scale(byte);
            const long long r = (long long)blockIdx.z * a.rows + row;
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
            tops[ty][tx * 8 + j] = top;
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
        const int byte = BLOCKS ? block_byte : scale_byte(tops[0][tx * 8 + j]);
        const float inv = inverse_scale(byte);
        const float c[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
        *reinterpret_cast<Vec<uint32_t, 2>*>(&tile[tx * 8 + j][ty * 8]) = Vec<uint32_t, 2>{fp8x4(c, inv), fp8x4(c + 4, inv)};
        const int col = c0 + tx * 8 + j;
        if (!BLOCKS && ty == 0 && col < a.cols)
            a.scalesT[((long long)blockIdx.z * a.cols + col) * a.spitch_t + blockIdx.x] = (uint8_t)byte;
    }
    if (BLOCKS && threadIdx.x == 0)
        a.scalesT[((long long)blockIdx.z * gridDim.y + blockIdx.y) * a.spitch_t + blockIdx.x] = (uint8_t)block_byte;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int unit = i * kQuantThreads + threadIdx.x, c = unit >> 3, at = (unit & 7) * 16;
        if (c0 + c < a.cols)
            *reinterpret_cast<Vec<uint32_t, 4>*>(a.qt + ((long long)blockIdx.z * a.cols + c0 + c) * a.pitch_t + r0 + at) =
                *reinterpret_cast<const Vec<uint32_t, 4>*>(&tile[c][at]);
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
    a.vec = fits(src, o.srcStride) && (o.batch == 1 || o.srcBatchStride * bytes % 16 == 0) &&
            (!gate || fits(gate, o.gateStride));
    const int cb = a.pitch / 128, rb = a.pitch_t / 128;
    with_type(o.srcType, [&](auto zero) {
        using T = decltype(zero);
        if (o.blockRows == 128) quant_tile_kernel<T, true><<<dim3(rb, cb, o.batch), kQuantThreads, 0, s>>>(a);
        else if (qt) quant_tile_kernel<T, false><<<dim3(rb, cb, o.batch), kQuantThreads, 0, s>>>(a);
        else {
            const long long units = (long long)o.rows * cb, wgs = (units + kQuantThreads / 16 - 1) / (kQuantThreads / 16);
            require(wgs <= 0x7fffffffll, "too many blocks for one call");
            quant_rows_kernel<T><<<dim3((unsigned)wgs, o.batch), kQuantThreads, 0, s>>>(a);
        }
    });
    GRAFT_LAUNCH_CHECK();
}

}  // namespace graft
