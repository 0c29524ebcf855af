// Quantising to e2m1 with a power-of-two scale for each block of 32, for gfx950
// (layout: experts_abi.h).
//
//   s = 2^(floor(log2 max |x|) - 2), or the next one where max |x| > 6 s,
//   q = e2m1(x / s)
//
// The scale comes from the bits of the block's largest magnitude (exponent - 2,
// under the covering rule one more where its mantissa is above that of 6 = 1.5 *
// 2^2), and x / s is a change of exponent: the one rounding is the conversion's,
// which takes 6 for what is beyond.
#include "experts.h"
#include "lanes.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kQuantThreads = 256;
constexpr uint32_t kInfinity = 0x7f800000u;

struct Quant4Args {
    const void* src;
    const int* order;
    uint8_t *q, *scales;
    int rows, cols, slots_per_row, src_rows;
    int pitch, spitch;
    long long stride, batch_stride;
    long long wg0;  // the launch's first workgroup
    bool vec, cover;
};

// Where columns col .. col + 7 of a quantised row come from; nullptr: they are zero.
template <class T>
__device__ __forceinline__ const T* source_of(const Quant4Args& a, const T* src, int row, int col)
{
    if (row >= a.rows || col >= a.cols) return nullptr;
    long long from = row;
    if (a.order) {
        const int slot = a.order[row];
        from = slot / a.slots_per_row;
        if (slot < 0 || from >= a.src_rows) return nullptr;
    }
    return src + from * a.stride + col;
}

template <class T>
__device__ __forceinline__ void load8(float (&v)[8], const Quant4Args& a, const T* p, int col)
{
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.0f;
    if (!p) return;
    if (a.vec) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            const Vec<T, N> w = *reinterpret_cast<const Vec<T, N>*>(p + i);
#pragma unroll
            for (int j = 0; j < N; j++) v[i + j] = (float)w[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (col + j < a.cols) v[j] = (float)p[j];
    }
}

// Four lanes a block of 32, eight columns each; kUnits such a thread, whose loads are
// under way together.  Bound by memory where rows come as they are (8,191 x 4,096 bf16:
// 21 us, 4.1 TB/s; 22.6 and 24.3 with two and four units), by the loads that wait for
// an order's where they are gathered (65,536 rows of 1,024 fp16: 43 us with four
// units, 3.9 TB/s; 45 with two, 49 with one).
constexpr int kGathered = 4;
template <class T, int kUnits>
__global__ __launch_bounds__(kQuantThreads) void quant4_kernel(Quant4Args a)
{
    const uint32_t pieces = a.pitch / 4;
    const unsigned long long unit = (unsigned long long)(a.wg0 + blockIdx.x) * (kQuantThreads * kUnits);
    const uint32_t row0 = (uint32_t)(unit / pieces), left = (uint32_t)(unit % pieces);  // the workgroup's first
    const T* const src = (const T*)a.src + (long long)blockIdx.y * a.batch_stride;
    int row[kUnits], col[kUnits];
    const T* p[kUnits];
    float v[kUnits][8];
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
        const uint32_t at = left + u * kQuantThreads + threadIdx.x;
        row[u] = (int)(row0 + at / pieces);
        col[u] = (int)(at % pieces) * 8;
        p[u] = source_of(a, src, row[u], col[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnits; u++) load8(v[u], a, p[u], col[u]);
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, __builtin_bit_cast(uint32_t, v[u][j]) & 0x7fffffffu);
        top = lanes_umax<4>(top);
        if (row[u] >= a.rows) return;  // and so are those behind it
        const int e = (int)(top >> 23) - 2 + (a.cover && (top & 0x7fffffu) > 0x400000u ? 1 : 0);
        const int byte = top >= kInfinity ? 255 : max(e, 1);
        uint32_t w = 0;
        if (byte != 255) {
            const float inv = __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u][0] * inv, v[u][1] * inv, 1.0f, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u][2] * inv, v[u][3] * inv, 1.0f, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u][4] * inv, v[u][5] * inv, 1.0f, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u][6] * inv, v[u][7] * inv, 1.0f, 3);
        }
        const long long r = (long long)blockIdx.y * a.rows + row[u];
        *reinterpret_cast<uint32_t*>(a.q + r * a.pitch + col[u] / 2) = w;
        if ((threadIdx.x & 3) == 0) a.scales[r * a.spitch + col[u] / 32] = (uint8_t)byte;
    }
}

}  // namespace

void fp4_quantize(const Fp4QuantOption& o, const void* src, const int* order, uint8_t* q, uint8_t* scales, hipStream_t s)
{
    require(o.rows >= 0 && o.rows <= kMaxRows && o.srcRows >= 0, "rows must be 0..2^30 and srcRows >= 0");
    require(o.cols >= 1 && o.cols <= 1 << 22, "cols must be 1..2^22");
    require(o.batch >= 1 && o.batch <= 65535, "batch must be 1..65535");
    require(o.scaleRule == FP4_SCALE_FLOOR || o.scaleRule == FP4_SCALE_COVER, "unknown scaleRule");
    require_type(o.srcType);
    require(o.srcStride >= o.cols, "srcStride must be at least cols");
    require(o.batch == 1 || o.srcBatchStride >= 0, "srcBatchStride must be >= 0");
    require(!order || (o.slotsPerRow >= 1 && o.batch == 1), "an order needs slotsPerRow >= 1 and a batch of 1");
    require(order || o.srcRows >= o.rows, "srcRows must be at least rows");
    if (o.rows == 0) return;
    require(q && scales && (src || (order && o.srcRows == 0)), "null argument");
    require(aligned16(q) && ((uintptr_t)scales & 3) == 0, "q must be 16-byte and scales 4-byte aligned");
    Quant4Args a{};
    a.src = src;
    a.order = order;
    a.q = q;
    a.scales = scales;
    a.rows = o.rows;
    a.cols = o.cols;
    a.slots_per_row = o.slotsPerRow;
    a.src_rows = o.srcRows;
    a.pitch = fp4_pitch(o.cols);
    a.spitch = fp4_scale_pitch(o.cols);
    a.stride = o.srcStride;
    a.batch_stride = o.srcBatchStride;
    a.cover = o.scaleRule == FP4_SCALE_COVER;
    const int bytes = data_bytes(o.srcType);
    a.vec = o.cols % 8 == 0 && aligned16(src) && o.srcStride * bytes % 16 == 0 &&
            (o.batch == 1 || o.srcBatchStride * bytes % 16 == 0);
    with_type(o.srcType, [&](auto zero) {
        const long long units = (long long)o.rows * (a.pitch / 4);
        const int each = kQuantThreads * (order ? kGathered : 1);
        in_launches((units + each - 1) / each, kQuantThreads, [&](long long first, unsigned wgs) {
            a.wg0 = first;
            if (order) quant4_kernel<decltype(zero), kGathered><<<dim3(wgs, o.batch), kQuantThreads, 0, s>>>(a);
            else quant4_kernel<decltype(zero), 1><<<dim3(wgs, o.batch), kQuantThreads, 0, s>>>(a);
        });
    });
}

}  // namespace graft
