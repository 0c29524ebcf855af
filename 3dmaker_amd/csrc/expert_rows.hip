// The experts' rows back to tokens, for gfx950:
//   combine   out[t] = sum_j w[t, j] rows[p[t, j]]
//   backward  dw[t, j] = <dout[t], rows[p[t, j]]>
// Both are bound by memory: each row of the experts is read once, in pieces of
// 16 bytes a lane.
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
};

// A thread: N consecutive columns of a token (32,768 x 2 rows of 2,048 bf16:
// 75 us, 5.4 TB/s).
template <class T, int N>
__global__ __launch_bounds__(kRowThreads) void combine_kernel(RowArgs a)
{
    const int chunks = (a.dim + N - 1) / N;
    const long long unit = (long long)blockIdx.x * kRowThreads + threadIdx.x;
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
        const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>((const T*)a.rows + (long long)p * a.row_stride + col);
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = fmaf(w, (float)v[i], acc[i]);
    }
    Vec<T, N> o;
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = (T)acc[i];
    *reinterpret_cast<Vec<T, N>*>((T*)a.out + t * a.out_stride + col) = o;
}

// A wave: K slots of a token at a time, their rows' loads under way together.
// Positions outside read row 0 and count for nothing.  16,384 x 2 rows of 2,048
// fp16: 46 us, 4.4 TB/s.
template <class T, int N, int K>
__global__ __launch_bounds__(kRowThreads) void combine_backward_kernel(RowArgs a)
{
    const long long t = (long long)blockIdx.x * (kRowThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int lane = threadIdx.x & 63;
    if (t >= a.tokens) return;
    const T* d = (const T*)a.dout + t * a.out_stride;
    for (int j0 = 0; j0 < a.topk; j0 += K) {
        const T* row[K];
        bool there[K];
        float acc[K];
#pragma unroll
        for (int q = 0; q < K; q++) {
            const int p = j0 + q < a.topk ? a.position[t * a.topk + j0 + q] : -1;
            there[q] = (unsigned)p < (unsigned)a.num_rows;
            row[q] = (const T*)a.rows + (there[q] ? (long long)p * a.row_stride : 0);
            acc[q] = 0.0f;
        }
        if (a.num_rows > 0) {
#pragma unroll 2
            for (int c = lane * N; c < a.dim; c += 64 * N) {
                const Vec<T, N> dv = *reinterpret_cast<const Vec<T, N>*>(d + c);
                Vec<T, N> rv[K];
#pragma unroll
                for (int q = 0; q < K; q++) rv[q] = *reinterpret_cast<const Vec<T, N>*>(row[q] + c);
#pragma unroll
                for (int q = 0; q < K; q++)
#pragma unroll
                    for (int i = 0; i < N; i++) acc[q] = fmaf((float)dv[i], (float)rv[q][i], acc[q]);
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
    require_type(type);
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

bool row_vec(const RowArgs& a, const void* other, int bytes)
{
    return aligned16(a.rows) && aligned16(other) && a.dim * bytes % 16 == 0 && a.row_stride * bytes % 16 == 0 &&
           a.out_stride * bytes % 16 == 0;
}

// f(T{}, number of elements of a thread's access)
template <class F>
void with_vec(int type, bool vec, F&& f)
{
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        if (vec) f(zero, std::integral_constant<int, 16 / (int)sizeof(T)>{});
        else f(zero, std::integral_constant<int, 1>{});
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
    with_vec(type, row_vec(a, out, data_bytes(type)), [&](auto zero, auto N) {
        constexpr int n = decltype(N)::value;
        const long long units = (long long)tokens * ((dim + n - 1) / n), wgs = (units + kRowThreads - 1) / kRowThreads;
        require(wgs <= 0x7fffffffll, "too many elements for one call");
        combine_kernel<decltype(zero), n><<<(unsigned)wgs, kRowThreads, 0, s>>>(a);
    });
    GRAFT_LAUNCH_CHECK();
}

void expert_combine_backward(int dim, int type, const void* rows, int num_rows, long long row_stride, const int* position,
                             const void* dout, long long dout_stride, float* dweights, int tokens, int topK, hipStream_t s)
{
    RowArgs a = row_args(dim, type, rows, num_rows, row_stride, position, tokens, topK, dout_stride);
    if (tokens == 0) return;
    require(dout && dweights, "null argument");
    a.dout = dout;
    a.dweights = dweights;
    with_vec(type, row_vec(a, dout, data_bytes(type)), [&](auto zero, auto N) {
        using T = decltype(zero);
        constexpr int n = decltype(N)::value;
        const unsigned wgs = (unsigned)((tokens + 3ll) / 4);
        if (topK == 1) combine_backward_kernel<T, n, 1><<<wgs, kRowThreads, 0, s>>>(a);
        else if (topK == 2) combine_backward_kernel<T, n, 2><<<wgs, kRowThreads, 0, s>>>(a);
        else combine_backward_kernel<T, n, 4><<<wgs, kRowThreads, 0, s>>>(a);
    });
    GRAFT_LAUNCH_CHECK();
}

}  // namespace graft
