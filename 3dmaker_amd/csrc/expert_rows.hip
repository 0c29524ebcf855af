// The experts' rows back to tokens, for gfx950:
//   combine   out[t] = sum_j w[t, j] rows[p[t, j]]
//   backward  dw[t, j] = <dout[t], rows[p[t, j]]>
// Both are bound by memory: each row of the experts is read once, in pieces of
// 16 bytes a lane.
//
// The rows' type R is that of the tokens, T, or fp32 on request.  16-bit rows are
// a rounding more, between the experts' products and this sum: half the bytes of
// the largest tensor of the block, for errors of a result about sqrt(2) of those
// of its own rounding (two experts, bf16: 0.0023 of its 2-norm, 0.0017 with fp32
// rows, for which 32,768 x 2 rows of 2,048 take 121 us instead of 75, and the
// product in front 327 instead of 213).
#include "experts.h"
#include "lanes.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kRowThreads = 256;

struct RowArgs {
    const void* rows;
    long long row_stride;
    const int* position;
    const float* weights;
    void* out;               // combine
    const void* dout;        // backward
    long long out_stride;    // of out or dout
    float* dweights;
    int dim, num_rows, tokens, topk;
    long long wg0;           // the launch's first workgroup
};

// N consecutive elements, in 16-byte loads where they are whole ones.
template <class R, int N>
struct Piece {
    static constexpr int P = 16 / sizeof(R) < N ? 16 / sizeof(R) : N;
    Vec<R, P> v[N / P];

    __device__ __forceinline__ void load(const R* p)
    {
#pragma unroll
        for (int i = 0; i < N / P; i++) v[i] = *reinterpret_cast<const Vec<R, P>*>(p + i * P);
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)v[i / P][i % P]; }
};

// A thread: N consecutive columns of a token (32,768 x 2 rows of 2,048 bf16:
// 75 us, 5.4 TB/s).
template <class R, class T, int N>
__global__ __launch_bounds__(kRowThreads) void combine_kernel(RowArgs a)
{
    const int chunks = (a.dim + N - 1) / N;
    const long long unit = (a.wg0 + blockIdx.x) * kRowThreads + threadIdx.x;
    const long long t = unit / chunks;
    const int col = (int)(unit % chunks) * N;
    if (t >= a.tokens) return;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = 0.0f;
    for (int j = 0; j < a.topk; j++) {
        const int p = a.position[t * a.topk + j];
        if ((unsigned)p >= (unsigned)a.num_rows) continue;
        const float w = a.weights ? a.weights[t * a.topk + j] : 1.0f;
        Piece<R, N> v;
        v.load((const R*)a.rows + (long long)p * a.row_stride + col);
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = fmaf(w, v[i], acc[i]);
    }
    Vec<T, N> o;
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = (T)acc[i];
    *reinterpret_cast<Vec<T, N>*>((T*)a.out + t * a.out_stride + col) = o;
}

// A wave: K slots of a token at a time, their rows' loads under way together.
// Positions outside read row 0 and count for nothing.  16,384 x 2 rows of 2,048
// fp16: 46 us, 4.4 TB/s.
template <class R, class T, int N, int K>
__global__ __launch_bounds__(kRowThreads) void combine_backward_kernel(RowArgs a)
{
    const long long t = (a.wg0 + blockIdx.x) * (kRowThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int lane = threadIdx.x & 63;
    if (t >= a.tokens) return;
    const T* d = (const T*)a.dout + t * a.out_stride;
    for (int j0 = 0; j0 < a.topk; j0 += K) {
        const R* row[K];
        bool there[K];
        float acc[K];
#pragma unroll
        for (int q = 0; q < K; q++) {
            const int p = j0 + q < a.topk ? a.position[t * a.topk + j0 + q] : -1;
            there[q] = (unsigned)p < (unsigned)a.num_rows;
            row[q] = (const R*)a.rows + (there[q] ? (long long)p * a.row_stride : 0);
            acc[q] = 0.0f;
        }
        if (a.num_rows > 0) {
#pragma unroll 2
            for (int c = lane * N; c < a.dim; c += 64 * N) {
                const Vec<T, N> dv = *reinterpret_cast<const Vec<T, N>*>(d + c);
                Piece<R, N> rv[K];
#pragma unroll
                for (int q = 0; q < K; q++) rv[q].load(row[q] + c);
#pragma unroll
                for (int q = 0; q < K; q++)
#pragma unroll
                    for (int i = 0; i < N; i++) acc[q] = fmaf((float)dv[i], rv[q][i], acc[q]);
            }
        }
#pragma unroll
        for (int q = 0; q < K; q++) {
            const float sum = lanes_sum<64>(acc[q]);
            if (lane == 0 && j0 + q < a.topk) a.dweights[t * a.topk + j0 + q] = there[q] ? sum : 0.0f;
        }
    }
}

RowArgs row_args(int dim, int type, const void* rows, int num_rows, long long row_stride, const int* position, int tokens,
                 int topK, long long out_stride)
{
    require(dim >= 1 && dim <= 1 << 23, "dim must be 1..2^23");
    require_type(type & ~COMBINE_ROWS_F32);
    require(tokens >= 0 && tokens <= kMaxRows && num_rows >= 0, "numTokens must be 0..2^30 and numRows >= 0");
    require(topK >= 1 && topK <= 32, "topK must be 1..32");
    require(row_stride >= dim && out_stride >= dim, "strides must be at least dim");
    require(tokens == 0 || (position && (rows || num_rows == 0)), "null argument");
    RowArgs a{};
    a.rows = rows;
    a.row_stride = row_stride;
    a.position = position;
    a.out_stride = out_stride;
    a.dim = dim;
    a.num_rows = num_rows;
    a.tokens = tokens;
    a.topk = topK;
    return a;
}

// f(R{}, T{}, number of elements of a thread's access)
template <class F>
void with_vec(int type, const RowArgs& a, const void* other, F&& f)
{
    const bool wide = type & COMBINE_ROWS_F32;
    type &= ~COMBINE_ROWS_F32;
    const int bytes = data_bytes(type), row_bytes = wide ? 4 : bytes;
    const bool vec = aligned16(a.rows) && aligned16(other) && a.dim * bytes % 16 == 0 && a.row_stride * row_bytes % 16 == 0 &&
                     a.out_stride * bytes % 16 == 0;
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        auto with_rows = [&](auto row) {
            if (vec) f(row, zero, std::integral_constant<int, 16 / (int)sizeof(T)>{});
            else f(row, zero, std::integral_constant<int, 1>{});
        };
        if (wide) with_rows(float{});
        else with_rows(zero);
    });
}

}  // namespace

void expert_combine(int dim, int type, const void* rows, int num_rows, long long row_stride, const int* position,
                    const float* weights, void* out, long long out_stride, int tokens, int topK, hipStream_t s)
{
    RowArgs a = row_args(dim, type, rows, num_rows, row_stride, position, tokens, topK, out_stride);
    if (tokens == 0) return;
    require(out, "null argument");
    a.weights = weights;
    a.out = out;
    with_vec(type, a, out, [&](auto row, auto zero, auto N) {
        constexpr int n = decltype(N)::value;
        const long long units = (long long)tokens * ((dim + n - 1) / n);
        in_launches((units + kRowThreads - 1) / kRowThreads, kRowThreads, [&](long long first, unsigned wgs) {
            a.wg0 = first;
            combine_kernel<decltype(row), decltype(zero), n><<<wgs, kRowThreads, 0, s>>>(a);
        });
    });
}

void expert_combine_backward(int dim, int type, const void* rows, int num_rows, long long row_stride, const int* position,
                             const void* dout, long long dout_stride, float* dweights, int tokens, int topK, hipStream_t s)
{
    RowArgs a = row_args(dim, type, rows, num_rows, row_stride, position, tokens, topK, dout_stride);
    if (tokens == 0) return;
    require(dout && dweights, "null argument");
    a.dout = dout;
    a.dweights = dweights;
    with_vec(type, a, dout, [&](auto row, auto zero, auto N) {
        using R = decltype(row);
        using T = decltype(zero);
        constexpr int n = decltype(N)::value;
        in_launches((tokens + 3ll) / 4, kRowThreads, [&](long long first, unsigned wgs) {
            a.wg0 = first;
            if (topK == 1) combine_backward_kernel<R, T, n, 1><<<wgs, kRowThreads, 0, s>>>(a);
            else if (topK == 2) combine_backward_kernel<R, T, n, 2><<<wgs, kRowThreads, 0, s>>>(a);
            else combine_backward_kernel<R, T, n, 4><<<wgs, kRowThreads, 0, s>>>(a);
        });
    });
}

}  // namespace graft
