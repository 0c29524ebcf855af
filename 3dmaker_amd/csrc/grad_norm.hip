// The norm over all elements of many tensors, and the tensors scaled to at most a
// given one, for gfx950:
//   n = sqrt(sum g^2) / scale  or  max |g| / scale;   g = g min(1, max / n)
// Bound by memory: one read for the norm, one read and one write for the clipping.
//
// The list of tensors goes to the kernels by value, kMostTensors to a launch, so
// that nothing has to be kept for it.  It is worked through in pieces of 64 bytes a
// thread; a workgroup (of few gradients: a wave of the only one) takes consecutive
// ones, so that it looks its first tensor up once.
// Squares of fp32 numbers are exact in 64 bits, and neither overflow nor vanish:
// the sum is off by 2^-53 an addition.  Sums of workgroups are joined in their
// order.
#include "grad_norm.h"

#include "lanes.h"

#include <algorithm>
#include <cmath>

namespace graft {

namespace {

constexpr int kGradThreads = 256, kSmallThreads = 1024;
constexpr int piece_bytes(int threads) { return threads * 64; }
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
    bool top;             // the largest magnitude
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

// A thread's sum of squares, or its largest magnitude as bits (NaN above all); four
// of them, so that an addition does not wait for the one before.
template <bool TOP>
struct Sum {
    double sq[4] = {};
    uint32_t top = 0;
    __device__ __forceinline__ void add(float v, int i)
    {
        if constexpr (TOP) top = max(top, magnitude(v));
        else sq[i & 3] = fma((double)v, (double)v, sq[i & 3]);
    }
    __device__ __forceinline__ double value() const { return TOP ? (double)top : (sq[0] + sq[1]) + (sq[2] + sq[3]); }
};

// f(first element, elements) of the thread's whole 16-byte parts of a piece, and
// g(element, its place in the part, value) for the elements of the tensor's first and
// last part, which are another's for the rest.  A part's loads are under way together.
template <int THREADS, class T, class F, class G>
__device__ __forceinline__ void for_parts(const Span<T>& t, uint32_t piece, F&& f, G&& g)
{
    constexpr int N = Span<T>::N, kPer = 4, kElements = piece_bytes(THREADS) / (int)sizeof(T);
    const int thread = threadIdx.x & (THREADS - 1);
    const long long first = (long long)piece * kElements;
    Vec<T, N> v[kPer];
    if (first >= t.lo && first + kElements <= t.hi) {
#pragma unroll
        for (int i = 0; i < kPer; i++) v[i] = *reinterpret_cast<const Vec<T, N>*>(t.base + first + (i * THREADS + thread) * N);
#pragma unroll
        for (int i = 0; i < kPer; i++) f(first + (i * THREADS + thread) * N, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const long long at = first + (i * THREADS + thread) * N;
            if (at >= t.lo && at + N <= t.hi) v[i] = *reinterpret_cast<const Vec<T, N>*>(t.base + at);
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const long long at = first + (i * THREADS + thread) * N;
            if (at >= t.lo && at + N <= t.hi) f(at, v[i]);
            else if (at + N > t.lo && at < t.hi) {
                T e[N];
#pragma unroll
                for (int j = 0; j < N; j++) e[j] = t.base[min(max(at + j, t.lo), t.hi - 1)];
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (at + j >= t.lo && at + j < t.hi) g(at + j, j, e[j]);
            }
        }
    }
}

template <int THREADS, class T, bool TOP>
__device__ __forceinline__ void add_piece(Sum<TOP>& s, const Span<T>& t, uint32_t piece)
{
    for_parts<THREADS>(
        t, piece,
        [&](long long, Vec<T, Span<T>::N> v) {
#pragma unroll
            for (int j = 0; j < Span<T>::N; j++) s.add((float)v[j], j);
        },
        [&](long long, int j, T v) { s.add((float)v, j); });
}

// f(tensor, piece of it) over the pieces of one of `workers`; BACK: from the last to
// the first, as what the pass for the norm has read last may still be in the cache
// for the one that clips.
template <bool BACK, class F>
__device__ __forceinline__ void for_pieces(const GradTable& t, uint32_t worker, uint32_t workers, F&& f)
{
    const uint32_t pieces = t.end[t.count - 1];
    const uint32_t p0 = (uint32_t)((uint64_t)pieces * worker / workers);
    const uint32_t p1 = (uint32_t)((uint64_t)pieces * (worker + 1) / workers);
    if (p0 == p1) return;
    const uint32_t start = BACK ? p1 - 1 : p0;
    // The first tensor that ends behind it, found by all lanes at once: a search in
    // steps waits for the kernel's arguments at each of them.
    static_assert(kMostTensors <= 128, "two a lane");
    const int lane = threadIdx.x & 63;
    int lo = __popcll(__ballot(lane < t.count && t.end[lane] <= start));
    lo += __popcll(__ballot(64 + lane < t.count && t.end[64 + lane] <= start));
    if (BACK) {
        for (uint32_t p = p1; p-- > p0;) {
            while (lo > 0 && p < t.end[lo - 1]) lo--;
            f(lo, p - (lo ? t.end[lo - 1] : 0u));
        }
    } else {
        for (uint32_t p = p0; p < p1; p++) {
            while (p >= t.end[lo]) lo++;
            f(lo, p - (lo ? t.end[lo - 1] : 0u));
        }
    }
}

// f(T{}) with the C++ type of a tensor.
template <class F>
__device__ __forceinline__ void with_type_of(int type, F&& f)
{
    if (type == DATA_F32) f(0.0f);
    else if (type == DATA_F16) f((_Float16)0.0f);
    else f((__bf16)0.0f);
}

__device__ __forceinline__ double wave_sum(double v)
{
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Of a workgroup, in every thread: the sum or the largest.
template <int THREADS>
__device__ __forceinline__ double join(double v, bool top)
{
    constexpr int kWaves = THREADS / 64;
    __shared__ double part[kWaves];
    if (!top) v = wave_sum(v);
    else
        for (int o = 32; o > 0; o >>= 1) {
            const double u = __shfl_xor(v, o, 64);
            v = u > v ? u : v;
        }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) v = !top ? v + part[w] : (part[w] > v ? part[w] : v);
    return v;
}

// Largest magnitudes travel as their bits: whole numbers, so that NaN are the largest.
template <int THREADS, bool TOP>
__device__ __forceinline__ double sum_of(const GradTable& t, uint32_t worker, uint32_t workers)
{
    Sum<TOP> s;
    for_pieces<false>(t, worker, workers, [&](int i, uint32_t piece) {
        with_type_of(t.type[i], [&](auto zero) { add_piece<THREADS>(s, Span<decltype(zero)>(t.data[i], t.n[i]), piece); });
    });
    return s.value();
}

__device__ __forceinline__ float norm_of_sum(const GradArgs& a, double v)
{
    const double n = a.top ? (double)__builtin_bit_cast(float, (uint32_t)v) : sqrt(v);
    return (float)(n / (double)a.scale);
}

template <bool TOP>
__global__ __launch_bounds__(kGradThreads) void grad_sum_kernel(GradTable t, GradArgs a)
{
    const double v = join<kGradThreads>(sum_of<kGradThreads, TOP>(t, blockIdx.x, gridDim.x), TOP);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = v;
}

// The norm from the workgroups' sums, in every thread of a workgroup.
__device__ __forceinline__ float norm_of_sums(const GradArgs& a)
{
    double v = 0.0;
    for (int i = threadIdx.x; i < a.num_sums; i += kGradThreads) {
        const double u = a.sums[i];
        v = !a.top ? v + u : (u > v ? u : v);
    }
    return norm_of_sum(a, join<kGradThreads>(v, a.top));
}

__global__ __launch_bounds__(kGradThreads) void grad_norm_kernel(GradArgs a)
{
    const float n = norm_of_sums(a);
    if (threadIdx.x == 0) *a.norm_out = n;
}

// What gradients are multiplied by: max / n, as v 2^e where it is below the normal
// numbers, whose few bits would be those of every gradient.
struct Factor {
    float v;
    int e;
    __device__ __forceinline__ Factor(float max_norm, float n)
    {
        v = n > max_norm ? max_norm / n : 1.0f;
        e = 0;
        if (v < 0x1p-126f && max_norm > 0.0f) {
            int max_e, n_e;
            v = frexpf(max_norm, &max_e) * 0.5f / frexpf(n, &n_e);  // at most 1: products stay finite
            e = max_e + 1 - n_e;
        }
    }
};

template <int THREADS, class T>
__device__ __forceinline__ void clip_piece(const void* data, void* out, long long n, uint32_t piece, Factor factor, bool zero)
{
    constexpr int N = Span<T>::N;
    const Span<T> t(data, n);
    T* const to = (T*)out - t.lo;
    auto scaled = [&](T v) { return zero ? (T)0.0f : (T)ldexpf((float)v * factor.v, factor.e); };
    auto one = [&](long long at, int, T v) { to[at] = scaled(v); };
    if (((uintptr_t)to & 15) == 0) {
        for_parts<THREADS>(
            t, piece,
            [&](long long at, Vec<T, N> v) {
                if (factor.v != 1.0f || zero) {
#pragma unroll
                    for (int j = 0; j < N; j++) v[j] = scaled(v[j]);
                }
                *reinterpret_cast<Vec<T, N>*>(to + at) = v;
            },
            one);
    } else {  // an output that starts elsewhere in 16 bytes than its input: element by element
        for_parts<THREADS>(
            t, piece,
            [&](long long at, Vec<T, N> v) {
#pragma unroll
                for (int j = 0; j < N; j++) to[at + j] = scaled(v[j]);
            },
            one);
    }
}

template <int THREADS>
__device__ __forceinline__ void clip_all(const GradTable& t, const GradArgs& a, float n, uint32_t worker, uint32_t workers)
{
    const bool finite = magnitude(n) < 0x7f800000u, zero = !finite && a.zero;
    const Factor factor(a.max_norm, finite ? n : 0.0f);
    for_pieces<true>(t, worker, workers, [&](int i, uint32_t piece) {
        void* const out = t.out[i];
        if (out == t.data[i] && factor.v == 1.0f && !zero) return;
        with_type_of(t.type[i], [&](auto z) { clip_piece<THREADS, decltype(z)>(t.data[i], out, t.n[i], piece, factor, zero); });
    });
}

__global__ __launch_bounds__(kGradThreads) void grad_clip_kernel(GradTable t, GradArgs a)
{
    const float n = a.norm_in ? *a.norm_in : norm_of_sums(a);
    if (a.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = n;
    clip_all<kGradThreads>(t, a, n, blockIdx.x, gridDim.x);
}

// Few gradients: one workgroup does all of it, its waves with pieces of their own.
template <bool TOP, bool CLIP>
__global__ __launch_bounds__(kSmallThreads) void grad_small_kernel(GradTable t, GradArgs a)
{
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = kSmallThreads / 64;
    const double v = t.count ? sum_of<64, TOP>(t, wave, waves) : 0.0;
    const float n = norm_of_sum(a, join<kSmallThreads>(v, TOP));
    if (threadIdx.x == 0) *a.norm_out = n;
    if (CLIP && t.count) clip_all<64>(t, a, n, wave, waves);
}

long long pieces_of(const GradTensor& t, int threads)
{
    const long long bytes = ((uintptr_t)t.data & 15) + t.n * data_bytes(t.dataType);
    return t.n ? (bytes + piece_bytes(threads) - 1) / piece_bytes(threads) : 0;
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

void check_norm_pointer(const float* d_norm)
{
    require(d_norm, "null argument");
    require(((uintptr_t)d_norm & 3) == 0, "d_norm must be aligned to its elements");
}

void check_norm(int norm, float scale, const float* d_norm)
{
    require(norm == GRAD_NORM_2 || norm == GRAD_NORM_MAX, "unknown norm");
    require(std::isfinite(scale) && scale > 0.0f, "gradScale must be finite and above 0");
    check_norm_pointer(d_norm);
}

// Nothing that is written is another tensor's, or the norm's.
void check_clip(const GradTensor* tensors, int count, float max_norm, int non_finite, const float* d_norm, bool norm_written)
{
    require(max_norm >= 0.0f, "maxNorm must be >= 0");
    require(non_finite == GRAD_NONFINITE_KEEP || non_finite == GRAD_NONFINITE_ZERO, "unknown nonFinite");
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Range> all;
    all.reserve(2 * (size_t)count);
    for (int i = 0; i < count; i++) {
        const GradTensor& t = tensors[i];
        if (t.n == 0) continue;
        const uintptr_t size = (uintptr_t)t.n * data_bytes(t.dataType), in = (uintptr_t)t.data, out = (uintptr_t)t.out;
        const bool in_place = !out || out == in;
        all.push_back({in, in + size, in_place});
        if (!in_place) all.push_back({out, out + size, true});
    }
    check_norm_pointer(d_norm);
    const uintptr_t norm_lo = (uintptr_t)d_norm, norm_hi = norm_lo + sizeof(float);
    for (const Range& t : all)
        require(norm_hi <= t.lo || t.hi <= norm_lo || !(norm_written || t.written), "d_norm overlaps a tensor");
    auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
    if (!std::is_sorted(all.begin(), all.end(), before)) std::sort(all.begin(), all.end(), before);
    uintptr_t read = 0, written = 0;  // where those so far end
    for (const Range& r : all) {
        require(r.lo >= written && (!r.written || r.lo >= read), "a tensor that is written overlaps another");
        (r.written ? written : read) = std::max(r.written ? written : read, r.hi);
    }
}

// Of a launch: four a CU (400,000,003 bf16 elements in 390 tensors, four launches: 516
// us for norm and clipping, 4.2 and 5.0 TB/s; with 1,024 over all of them 851).
constexpr int kMostWorkgroups = 1024;

void add_to(GradTable& t, const GradTensor& g, long long pieces)
{
    t.data[t.count] = g.data;
    t.out[t.count] = g.out ? g.out : const_cast<void*>(g.data);
    t.n[t.count] = g.n;
    t.type[t.count] = (uint8_t)g.dataType;
    t.end[t.count] = (uint32_t)pieces + (t.count ? t.end[t.count - 1] : 0u);
    t.count++;
}

// f(table, workgroups) for the list in launches.  Their number.
template <class F>
int in_tables(const GradTensor* tensors, int count, F&& f)
{
    GradTable t;
    t.count = 0;
    long long pieces = 0;
    int launches = 0;
    auto flush = [&] {
        if (t.count) f(t, (unsigned)std::min<long long>(pieces, kMostWorkgroups)), launches++;
        t.count = 0;
        pieces = 0;
    };
    for (int i = 0; i < count; i++) {
        const long long own = pieces_of(tensors[i], kGradThreads);
        if (own == 0) continue;
        if (t.count == kMostTensors || pieces + own >= 1ll << 31) flush();
        add_to(t, tensors[i], own);
        pieces += own;
    }
    flush();
    return launches;
}

// The whole list in one workgroup's hands where it is short: up to kSmallPieces of a
// wave, 4 KB each (norm and clipping of four tensors, us by one workgroup and by two
// launches of many: 32 KB in all 3.5 and 5.4, 128 KB 4.6 and 5.4, 192 KB 5.6 and 5.5; of
// 40 tensors of 3 KB, a piece each, 7.3 and 6.1).
constexpr int kSmallPieces = 32;
bool small_table(const GradTensor* tensors, int count, GradTable& t)
{
    t.count = 0;
    long long pieces = 0;
    for (int i = 0; i < count; i++) {
        const long long own = pieces_of(tensors[i], 64);
        if (own == 0) continue;
        pieces += own;
        if (pieces > kSmallPieces || t.count == kMostTensors) return false;
        add_to(t, tensors[i], own);
    }
    return true;
}

// The workgroups' sums, in how many launches.
int sums(const GradTensor* tensors, int count, GradArgs& a, hipStream_t s)
{
    size_t most = 0;
    in_tables(tensors, count, [&](const GradTable&, unsigned wgs) { most += wgs; });
    a.sums = (double*)stream_workspace(s).get(most * sizeof(double));
    return in_tables(tensors, count, [&](const GradTable& t, unsigned wgs) {
        GradArgs b = a;
        b.sums += a.num_sums;
        if (a.top) grad_sum_kernel<true><<<wgs, kGradThreads, 0, s>>>(t, b);
        else grad_sum_kernel<false><<<wgs, kGradThreads, 0, s>>>(t, b);
        GRAFT_LAUNCH_CHECK();
        a.num_sums += (int)wgs;
    });
}

void norm(const GradArgs& a, hipStream_t s)
{
    grad_norm_kernel<<<1, kGradThreads, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

void clip(const GradTensor* tensors, int count, const GradArgs& a, hipStream_t s)
{
    in_tables(tensors, count, [&](const GradTable& t, unsigned wgs) {
        grad_clip_kernel<<<wgs, kGradThreads, 0, s>>>(t, a);
        GRAFT_LAUNCH_CHECK();
    });
}

}  // namespace

void grad_norm(const GradTensor* tensors, int count, int norm_kind, float scale, float* d_norm, hipStream_t s)
{
    check_list(tensors, count);
    check_norm(norm_kind, scale, d_norm);
    GradArgs a{};
    a.top = norm_kind == GRAD_NORM_MAX;
    a.scale = scale;
    a.norm_out = d_norm;
    GradTable t;
    if (small_table(tensors, count, t)) {
        if (a.top) grad_small_kernel<true, false><<<1, kSmallThreads, 0, s>>>(t, a);
        else grad_small_kernel<false, false><<<1, kSmallThreads, 0, s>>>(t, a);
        GRAFT_LAUNCH_CHECK();
        return;
    }
    sums(tensors, count, a, s);
    norm(a, s);
}

void grad_clip(const GradTensor* tensors, int count, float max_norm, int non_finite, const float* d_norm, hipStream_t s)
{
    check_list(tensors, count);
    check_clip(tensors, count, max_norm, non_finite, d_norm, false);
    GradArgs a{};
    a.max_norm = max_norm;
    a.zero = non_finite == GRAD_NONFINITE_ZERO;
    a.norm_in = d_norm;
    clip(tensors, count, a, s);
}

void grad_norm_clip(const GradTensor* tensors, int count, int norm_kind, float scale, float max_norm, int non_finite,
                    float* d_norm, hipStream_t s)
{
    check_list(tensors, count);
    check_norm(norm_kind, scale, d_norm);
    check_clip(tensors, count, max_norm, non_finite, d_norm, true);
    GradArgs a{};
    a.top = norm_kind == GRAD_NORM_MAX;
    a.scale = scale;
    a.max_norm = max_norm;
    a.zero = non_finite == GRAD_NONFINITE_ZERO;
    a.norm_out = d_norm;
    GradTable t;
    if (small_table(tensors, count, t)) {
        if (a.top) grad_small_kernel<true, true><<<1, kSmallThreads, 0, s>>>(t, a);
        else grad_small_kernel<false, true><<<1, kSmallThreads, 0, s>>>(t, a);
        GRAFT_LAUNCH_CHECK();
        return;
    }
    // One launch's workgroups each form the norm from the sums; of several, a kernel
    // of its own does.
    if (sums(tensors, count, a, s) > 1) {
        norm(a, s);
        a.norm_in = d_norm;
        a.norm_out = nullptr;
    }
    clip(tensors, count, a, s);
}

}  // namespace graft
