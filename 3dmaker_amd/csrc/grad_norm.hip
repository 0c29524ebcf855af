// The norm over all elements of many tensors, and the tensors scaled to at most a
// given one, for gfx950:
//   n = sqrt(sum g^2) / scale  or  max |g| / scale;   g = g min(1, max / n)
// Bound by memory: one read for the norm, one read and one write for the clipping.
//
// The list of tensors goes to the kernels by value, kMostTensors to a launch, so
// that nothing has to be kept for it.  It is worked through as pieces of 16 KiB; a
// workgroup takes consecutive ones, so that it looks its first tensor up once.
// Squares of fp32 numbers are exact in 64 bits, and neither overflow nor vanish:
// the sum is off by 2^-53 an addition.  Sums of workgroups are joined in their
// order.
#include "grad_norm.h"

#include "lanes.h"

#include <algorithm>
#include <cmath>

namespace graft {

namespace {

constexpr int kGradThreads = 256, kGradWaves = kGradThreads / 64;
constexpr int kPieceBytes = 16384;
constexpr int kMostTensors = 128;  // kernel arguments of 4 KiB

struct GradTable {
    const void* data[kMostTensors];
    void* out[kMostTensors];
    long long n[kMostTensors];
    uint32_t end[kMostTensors];  // pieces up to the tensor's end
    uint8_t type[kMostTensors];
    int count;
};

struct GradArgs {
    double* sums;         // of the workgroups
    int num_sums;
    int kind;
    float scale, max_norm;
    bool zero;            // where the norm is not finite
    const float* norm_in; // given, or from the sums
    float* norm_out;      // nullable
};

// A tensor's elements as 16-byte pieces of memory: those of its first and last that
// are another's are left out.
template <class T>
struct Span {
    static constexpr int N = 16 / sizeof(T);
    const T* base;    // at a multiple of 16 bytes
    long long lo, hi; // the tensor's elements from there

    __device__ __forceinline__ Span(const void* p, long long n)
    {
        const int off = (int)((uintptr_t)p & 15) / (int)sizeof(T);
        base = (const T*)p - off;
        lo = off;
        hi = off + n;
    }
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// A thread's sum of squares, or its largest magnitude as bits (NaN above all).
struct Sum {
    double sq = 0.0;
    uint32_t top = 0;
    __device__ __forceinline__ void add(float v, int kind)
    {
        if (kind == GRAD_NORM_2) sq = fma((double)v, (double)v, sq);
        else top = max(top, magnitude(v));
    }
};

template <class T>
__device__ __forceinline__ void add_piece(Sum& s, const Span<T>& t, long long first, int kind)
{
    constexpr int N = Span<T>::N, kPer = kPieceBytes / 16 / kGradThreads;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const long long at = first + (i * kGradThreads + (int)threadIdx.x) * N;
        if (at >= t.lo && at + N <= t.hi) {
            const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(t.base + at);
#pragma unroll
            for (int j = 0; j < N; j++) s.add((float)v[j], kind);
        } else {
            for (int j = 0; j < N; j++)
                if (at + j >= t.lo && at + j < t.hi) s.add((float)t.base[at + j], kind);
        }
    }
}

// f(tensor, piece of it) over the workgroup's pieces.
template <class F>
__device__ __forceinline__ void for_pieces(const GradTable& t, F&& f)
{
    const uint32_t pieces = t.end[t.count - 1];
    const uint32_t p0 = (uint32_t)((uint64_t)pieces * blockIdx.x / gridDim.x);
    const uint32_t p1 = (uint32_t)((uint64_t)pieces * (blockIdx.x + 1) / gridDim.x);
    int lo = 0, hi = t.count - 1;  // the first tensor that ends behind p0
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (t.end[mid] > p0) hi = mid;
        else lo = mid + 1;
    }
    for (uint32_t p = p0; p < p1; p++) {
        while (p >= t.end[lo]) lo++;
        f(lo, p - (lo ? t.end[lo - 1] : 0u));
    }
}

__device__ __forceinline__ double wave_sum(double v)
{
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Of a workgroup, in every thread: the sum or the largest.
__device__ __forceinline__ double join(double v, int kind)
{
    __shared__ double part[kGradWaves];
    if (kind == GRAD_NORM_2) v = wave_sum(v);
    else
        for (int o = 32; o > 0; o >>= 1) {
            const double u = __shfl_xor(v, o, 64);
            v = u > v ? u : v;
        }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kGradWaves; w++) v = kind == GRAD_NORM_2 ? v + part[w] : (part[w] > v ? part[w] : v);
    __syncthreads();
    return v;
}

// Largest magnitudes travel as their bits: whole numbers, so that NaN are the largest.
__global__ __launch_bounds__(kGradThreads) void grad_sum_kernel(GradTable t, GradArgs a)
{
    Sum s;
    for_pieces(t, [&](int i, uint32_t piece) {
        auto add = [&](auto zero) {
            using T = decltype(zero);
            add_piece(s, Span<T>(t.data[i], t.n[i]), (long long)piece * (kPieceBytes / sizeof(T)), a.kind);
        };
        if (t.type[i] == DATA_F32) add(0.0f);
        else if (t.type[i] == DATA_F16) add((_Float16)0.0f);
        else add((__bf16)0.0f);
    });
    const double v = join(a.kind == GRAD_NORM_2 ? s.sq : (double)s.top, a.kind);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = v;
}

// The norm from the workgroups' sums, in every thread of a workgroup.
__device__ __forceinline__ float norm_of(const GradArgs& a)
{
    double v = 0.0;
    for (int i = threadIdx.x; i < a.num_sums; i += kGradThreads) {
        const double u = a.sums[i];
        v = a.kind == GRAD_NORM_2 ? v + u : (u > v ? u : v);
    }
    v = join(v, a.kind);
    const double n = a.kind == GRAD_NORM_2 ? sqrt(v) : (double)__builtin_bit_cast(float, (uint32_t)v);
    return (float)(n / (double)a.scale);
}

__global__ __launch_bounds__(kGradThreads) void grad_norm_kernel(GradArgs a)
{
    const float n = norm_of(a);
    if (threadIdx.x == 0) *a.norm_out = n;
}

template <class T>
__device__ __forceinline__ void clip_piece(const void* data, void* out, long long n, uint32_t piece, float factor, bool zero)
{
    constexpr int N = Span<T>::N, kPer = kPieceBytes / 16 / kGradThreads;
    const Span<T> t(data, n);
    T* const to = (T*)out - t.lo;
    const bool vec = ((uintptr_t)to & 15) == 0;
    const long long first = (long long)piece * (kPieceBytes / sizeof(T));
    auto scaled = [&](T v) { return zero ? (T)0.0f : factor == 1.0f ? v : (T)((float)v * factor); };
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const long long at = first + (i * kGradThreads + (int)threadIdx.x) * N;
        if (vec && at >= t.lo && at + N <= t.hi) {
            Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(t.base + at);
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = scaled(v[j]);
            *reinterpret_cast<Vec<T, N>*>(to + at) = v;
        } else {
            for (int j = 0; j < N; j++)
                if (at + j >= t.lo && at + j < t.hi) to[at + j] = scaled(t.base[at + j]);
        }
    }
}

__global__ __launch_bounds__(kGradThreads) void grad_clip_kernel(GradTable t, GradArgs a)
{
    const float n = a.norm_in ? *a.norm_in : norm_of(a);
    if (a.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = n;
    const bool finite = magnitude(n) < 0x7f800000u, zero = !finite && a.zero;
    const float factor = finite && n > a.max_norm ? a.max_norm / n : 1.0f;
    for_pieces(t, [&](int i, uint32_t piece) {
        void* const out = t.out[i];
        if (out == t.data[i] && factor == 1.0f && !zero) return;
        if (t.type[i] == DATA_F32) clip_piece<float>(t.data[i], out, t.n[i], piece, factor, zero);
        else if (t.type[i] == DATA_F16) clip_piece<_Float16>(t.data[i], out, t.n[i], piece, factor, zero);
        else clip_piece<__bf16>(t.data[i], out, t.n[i], piece, factor, zero);
    });
}

long long pieces_of(const GradTensor& t)
{
    const long long bytes = ((uintptr_t)t.data & 15) + t.n * data_bytes(t.dataType);
    return t.n ? (bytes + kPieceBytes - 1) / kPieceBytes : 0;
}

void check_list(const GradTensor* tensors, int count)
{
    require(count >= 0 && count <= 65536, "count must be 0..65536");
    require(tensors || count == 0, "null argument");
    for (int i = 0; i < count; i++) {
        const GradTensor& t = tensors[i];
        require_type(t.dataType);
        require(t.n >= 0 && t.n <= 1ll << 40, "n must be 0..2^40");
        require(t.data || t.n == 0, "null argument");
        const int mask = data_bytes(t.dataType) - 1;
        require(((uintptr_t)t.data & mask) == 0 && ((uintptr_t)t.out & mask) == 0, "tensors must be aligned to their elements");
    }
}

void check_norm(int norm, float scale, const float* d_norm)
{
    require(norm == GRAD_NORM_2 || norm == GRAD_NORM_MAX, "unknown norm");
    require(std::isfinite(scale) && scale > 0.0f, "gradScale must be finite and above 0");
    require(d_norm, "null argument");
}

// Nothing that is written is another tensor's.
void check_clip(const GradTensor* tensors, int count, float max_norm, int non_finite)
{
    require(max_norm >= 0.0f, "maxNorm must be >= 0");
    require(non_finite == GRAD_NONFINITE_KEEP || non_finite == GRAD_NONFINITE_ZERO, "unknown nonFinite");
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Range> all;
    all.reserve(2 * count);
    for (int i = 0; i < count; i++) {
        const GradTensor& t = tensors[i];
        if (t.n == 0) continue;
        const uintptr_t size = (uintptr_t)t.n * data_bytes(t.dataType), in = (uintptr_t)t.data, out = (uintptr_t)t.out;
        const bool in_place = !out || out == in;
        all.push_back({in, in + size, in_place});
        if (!in_place) all.push_back({out, out + size, true});
    }
    auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
    if (!std::is_sorted(all.begin(), all.end(), before)) std::sort(all.begin(), all.end(), before);
    uintptr_t read = 0, written = 0;  // where those so far end
    for (const Range& r : all) {
        require(r.lo >= written && (!r.written || r.lo >= read), "a tensor that is written overlaps another");
        (r.written ? written : read) = std::max(r.written ? written : read, r.hi);
    }
}

constexpr int kMostSums = 1024;

// f(table, workgroups) for the list in launches; all of them have kMostSums
// workgroups at most but for one more a launch.
template <class F>
void in_tables(const GradTensor* tensors, int count, F&& f)
{
    long long all = 0;
    for (int i = 0; i < count; i++) all += pieces_of(tensors[i]);
    GradTable t;
    t.count = 0;
    long long pieces = 0;
    auto flush = [&] {
        if (t.count) f(t, (unsigned)std::max(1ll, std::min(pieces, kMostSums * pieces / all)));
        t.count = 0;
        pieces = 0;
    };
    for (int i = 0; i < count; i++) {
        const GradTensor& g = tensors[i];
        const long long own = pieces_of(g);
        if (own == 0) continue;
        if (t.count == kMostTensors || pieces + own >= 1ll << 31) flush();
        t.data[t.count] = g.data;
        t.out[t.count] = g.out ? g.out : const_cast<void*>(g.data);
        t.n[t.count] = g.n;
        t.type[t.count] = (uint8_t)g.dataType;
        pieces += own;
        t.end[t.count] = (uint32_t)pieces;
        t.count++;
    }
    flush();
}

// The workgroups' sums; their number.
int sums(const GradTensor* tensors, int count, GradArgs& a, hipStream_t s)
{
    const size_t most = kMostSums + (size_t)count + 1;
    a.sums = (double*)stream_workspace(s).get(most * sizeof(double));
    int n = 0;
    in_tables(tensors, count, [&](const GradTable& t, unsigned wgs) {
        GradArgs b = a;
        b.sums += n;
        grad_sum_kernel<<<wgs, kGradThreads, 0, s>>>(t, b);
        GRAFT_LAUNCH_CHECK();
        n += (int)wgs;
    });
    return n;
}

void clip(const GradTensor* tensors, int count, GradArgs a, hipStream_t s)
{
    in_tables(tensors, count, [&](const GradTable& t, unsigned wgs) {
        grad_clip_kernel<<<wgs, kGradThreads, 0, s>>>(t, a);
        GRAFT_LAUNCH_CHECK();
    });
}

}  // namespace

void grad_norm(const GradTensor* tensors, int count, int norm, float scale, float* d_norm, hipStream_t s)
{
    check_list(tensors, count);
    check_norm(norm, scale, d_norm);
    GradArgs a{};
    a.kind = norm;
    a.scale = scale;
    a.norm_out = d_norm;
    a.num_sums = sums(tensors, count, a, s);
    grad_norm_kernel<<<1, kGradThreads, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

void grad_clip(const GradTensor* tensors, int count, float max_norm, int non_finite, const float* d_norm, hipStream_t s)
{
    check_list(tensors, count);
    check_clip(tensors, count, max_norm, non_finite);
    require(d_norm, "null argument");
    GradArgs a{};
    a.max_norm = max_norm;
    a.zero = non_finite == GRAD_NONFINITE_ZERO;
    a.norm_in = d_norm;
    clip(tensors, count, a, s);
}

void grad_norm_clip(const GradTensor* tensors, int count, int norm, float scale, float max_norm, int non_finite, float* d_norm,
                    hipStream_t s)
{
    check_list(tensors, count);
    check_norm(norm, scale, d_norm);
    check_clip(tensors, count, max_norm, non_finite);
    grad_norm(tensors, count, norm, scale, d_norm, s);
    grad_clip(tensors, count, max_norm, non_finite, d_norm, s);
}

}  // namespace graft
