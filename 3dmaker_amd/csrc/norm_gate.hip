// Norms behind and before a block, with its gate and the scaled residual, for
// gfx950:
//   u = postnorm(f),  y = alpha x + beta g u,  h = prenorm(y)
// The backward recomputes both norms from x and f:
//   dn2 = dh w2            d  = dy + r2 (dn2 - mean dn2 - n2 mean(dn2 n2))
//   dx  = alpha d          dg = beta d u        du = beta g d
//   dn1 = du w1            df = r1 (dn1 - mean dn1 - n1 mean(dn1 n1))
//   dw2 = sum dh n2, db2 = sum dh, dw1 = sum du n1, db1 = sum du over the rows
// (the mean of dn only for layer norms).  Bound by memory: a row stays in
// registers between its passes (but for gradients of rows above 4,096 elements),
// statistics in fp32.
#include "experts.h"
#include "lanes.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kMaxDim = 8192;

struct NormArgs {
    const void *x, *f, *gate;
    const float *post_w, *post_b, *pre_w, *pre_b;
    void *y, *h;
    long long sx, sf, sg, sy, sh;
    int rows, dim, gate_rows, post, pre;
    float alpha, beta, eps, inv_dim;
    long long row0;  // the launch's first row (forward)
    // backward
    const void *dy, *dh;
    void *dx, *df, *dgate;
    float* sums;      // [parts][arrays][dim] or the outputs' own
    float* dst[4];    // dw1, db1, dw2, db2
    int parts, span, chunk, per_span;
    int gate_mode;
    float* gate_sums;  // [parts][dim]
};

enum { kGateNone, kGateRow, kGateWhole, kGatePart };

// The thread's elements of a row: PER pieces of VEC, THREADS * VEC apart.
template <class T, int VEC, int THREADS, int PER>
struct Row {
    static constexpr int N = VEC * PER;
    float v[N];

    __device__ __forceinline__ void load(const T* p, int sub, int dim)
    {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int c = (i * THREADS + sub) * VEC;
            if (c < dim) {
                const Vec<T, VEC> w = *reinterpret_cast<const Vec<T, VEC>*>(p + c);
#pragma unroll
                for (int j = 0; j < VEC; j++) v[i * VEC + j] = (float)w[j];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[i * VEC + j] = 0.0f;
            }
        }
    }

    __device__ __forceinline__ void store(T* p, int sub, int dim) const
    {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int c = (i * THREADS + sub) * VEC;
            if (c < dim) {
                Vec<T, VEC> w;
#pragma unroll
                for (int j = 0; j < VEC; j++) w[j] = (T)v[i * VEC + j];
                *reinterpret_cast<Vec<T, VEC>*>(p + c) = w;
            }
        }
    }
};

// A row's pieces as they lie in memory: what is fetched ahead.  Pieces behind the
// row are never loaded and stay zero.
template <class T, int VEC, int THREADS, int PER>
struct Raw {
    Vec<T, VEC> v[PER] = {};

    __device__ __forceinline__ void load(const T* p, int sub, int dim)
    {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int c = (i * THREADS + sub) * VEC;
            if (c < dim) v[i] = *reinterpret_cast<const Vec<T, VEC>*>(p + c);
        }
    }
    __device__ __forceinline__ void widen(float (&to)[VEC * PER]) const
    {
#pragma unroll
        for (int i = 0; i < PER; i++)
#pragma unroll
            for (int j = 0; j < VEC; j++) to[i * VEC + j] = (float)v[i][j];
    }
};

// The thread's elements of a parameter (fp32), `none` where there is no
// parameter.  In pieces of 16 bytes where the rows' are.
template <int VEC, int THREADS, int PER>
struct Param {
    float v[VEC * PER];

    __device__ __forceinline__ void load(const float* p, float none, int sub, int dim)
    {
#pragma unroll
        for (int i = 0; i < VEC * PER; i++) v[i] = none;
        if (!p) return;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int c = (i * THREADS + sub) * VEC;
            if (c < dim) {
                constexpr int P = VEC < 4 ? VEC : 4;
#pragma unroll
                for (int j = 0; j < VEC; j += P) {
                    const Vec<float, P> w = *reinterpret_cast<const Vec<float, P>*>(p + c + j);
#pragma unroll
                    for (int q = 0; q < P; q++) v[i * VEC + j + q] = w[q];
                }
            }
        }
    }
};

// f(element, column) over the thread's pieces that lie in the row (a piece is
// whole: rows in pieces of more than one element are multiples of it).
template <int VEC, int THREADS, int PER, class F>
__device__ __forceinline__ void each(int sub, int dim, F&& f)
{
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int c = (i * THREADS + sub) * VEC;
        if (c < dim) {
#pragma unroll
            for (int j = 0; j < VEC; j++) f(i * VEC + j, c + j);
        }
    }
}

// Sums over the THREADS of a row, in the same order for all of them.  Calls that
// follow each other use different slots: the barrier of one is what keeps the
// next use of another's slot behind its last read.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float (*lds)[THREADS / 64], int slot)
{
    v = lanes_sum<64>(v);
    if constexpr (THREADS > 64) {
        constexpr int W = THREADS / 64;
        if ((threadIdx.x & 63) == 0) lds[slot][threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) v += lds[slot][i];
    }
    return v;
}

template <int THREADS>
__device__ __forceinline__ void row_sum2(float& u, float& v, float (*lds)[THREADS / 64], int slot)
{
    u = lanes_sum<64>(u);
    v = lanes_sum<64>(v);
    if constexpr (THREADS > 64) {
        constexpr int W = THREADS / 64;
        if ((threadIdx.x & 63) == 0) lds[slot][threadIdx.x >> 6] = u, lds[slot + 1][threadIdx.x >> 6] = v;
        __syncthreads();
        u = v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) u += lds[slot][i], v += lds[slot + 1][i];
    }
}

// n = normalised v (in place) and 1 / its deviation; v's elements behind the
// row stay zero.
template <int VEC, int THREADS, int PER>
__device__ __forceinline__ float normalise(float (&v)[VEC * PER], int kind, int sub, int dim, float inv_dim, float eps,
                                           float (*lds)[THREADS / 64], int slot)
{
    if (kind == NORM_NONE) return 1.0f;
    if (kind == NORM_LAYER) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC * PER; i++) sum += v[i];
        const float mean = row_sum<THREADS>(sum, lds, slot) * inv_dim;
        each<VEC, THREADS, PER>(sub, dim, [&](int i, int) { v[i] -= mean; });
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC * PER; i++) sq = fmaf(v[i], v[i], sq);
    const float r = rsqrtf(row_sum<THREADS>(sq, lds, slot + 1) * inv_dim + eps);
#pragma unroll
    for (int i = 0; i < VEC * PER; i++) v[i] *= r;
    return r;
}

// v = v w + b
template <int VEC, int THREADS, int PER>
__device__ __forceinline__ void affine(float (&v)[VEC * PER], const float* w, const float* b, int sub, int dim)
{
    Param<VEC, THREADS, PER> p;
    if (w) {
        p.load(w, 1.0f, sub, dim);
#pragma unroll
        for (int i = 0; i < VEC * PER; i++) v[i] *= p.v[i];
    }
    if (b) {
        p.load(b, 0.0f, sub, dim);
#pragma unroll
        for (int i = 0; i < VEC * PER; i++) v[i] += p.v[i];
    }
}

// A wave or a workgroup a row, which is read once (32,769 x 2,048 bf16: 117 us,
// 4.6 TB/s; with the parameters read element by element 322).
template <class T, int VEC, int THREADS, int PER>
__global__ __launch_bounds__(256) void norm_gate_kernel(NormArgs a)
{
    __shared__ float lds[4][THREADS / 64];
    using R = Row<T, VEC, THREADS, PER>;
    const int sub = threadIdx.x & (THREADS - 1);
    const long long row = a.row0 + (long long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
    if (row >= a.rows) return;  // a row's threads return together; only whole workgroups meet at a barrier
    R y;
    y.load((const T*)a.x + row * a.sx, sub, a.dim);
    if (a.f) {
        R u;
        u.load((const T*)a.f + row * a.sf, sub, a.dim);
        normalise<VEC, THREADS, PER>(u.v, a.post, sub, a.dim, a.inv_dim, a.eps, lds, 0);
        affine<VEC, THREADS, PER>(u.v, a.post_w, a.post_b, sub, a.dim);
        if (a.gate) {
            R g;
            g.load((const T*)a.gate + row / a.gate_rows * a.sg, sub, a.dim);
#pragma unroll
            for (int i = 0; i < R::N; i++) u.v[i] *= g.v[i];
        }
#pragma unroll
        for (int i = 0; i < R::N; i++) y.v[i] = fmaf(a.alpha, y.v[i], a.beta * u.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < R::N; i++) y.v[i] *= a.alpha;
    }
    if (a.y) y.store((T*)a.y + row * a.sy, sub, a.dim);
    if (!a.h) return;
    normalise<VEC, THREADS, PER>(y.v, a.pre, sub, a.dim, a.inv_dim, a.eps, lds, 2);
    affine<VEC, THREADS, PER>(y.v, a.pre_w, a.pre_b, sub, a.dim);
    y.store((T*)a.h + row * a.sh, sub, a.dim);
}

// dL/dinput (in place of d) of a norm whose normalised input is n and 1 /
// deviation r; the parameters' sums of this row added.  w: its weights.
template <int VEC, int THREADS, int PER>
__device__ __forceinline__ void norm_back(float (&d)[VEC * PER], const float (&n)[VEC * PER], float r, int kind,
                                          const float (&w)[VEC * PER], float (&dw)[VEC * PER], float (&db)[VEC * PER],
                                          int sub, int dim, float inv_dim, float (*lds)[THREADS / 64], int slot)
{
    constexpr int N = VEC * PER;
    if (kind == NORM_NONE) return;
    float m = 0.0f, p = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {  // d and n are zero behind the row
        dw[i] = fmaf(d[i], n[i], dw[i]);
        db[i] += d[i];
        d[i] *= w[i];
        m += d[i];
        p = fmaf(d[i], n[i], p);
    }
    row_sum2<THREADS>(m, p, lds, slot);
    m = kind == NORM_LAYER ? m * inv_dim * r : 0.0f;
    p *= inv_dim * r;
    each<VEC, THREADS, PER>(sub, dim, [&](int i, int) { d[i] = fmaf(-n[i], p, fmaf(d[i], r, -m)); });
}

// A workgroup: `chunk` rows of a span, its row groups (waves for THREADS 64) in
// turn; sums over its rows go to sums[part], or for one part to the outputs.  The
// next row is fetched while this one is worked on: without that a row waits for
// four tensors one after the other (16,389 x 1,280 fp16, layer norms: 237 us;
// 67 now, 3.8 TB/s).  Bound by about 600 instructions a thread and row, at three
// waves a SIMD: 168 registers are the most for these, and aligned 16-bit rows of
// 128 to 512 threads take 166.  16-bit rows of 64 threads take 169, fp32 and
// unaligned ones 185 to 256: two waves (fp32 16,389 x 1,280: 122 us, 4.1 TB/s;
// 8,195 x 4,096: 173 us, 4.7 TB/s; 16-bit 65,539 x 256: 86 us, 2.3 TB/s; 16,389 x
// 1,281: 133 us, 1.9 TB/s).  Rows above 4,096 elements have 1,024 threads of 128
// registers, and spill 176 bytes a lane (16 bits), 344 (fp32) or 480 to 524
// (unaligned): 4,099 x 8,192 bf16 345 us, 1.2 TB/s, fp32 642.
template <class T, int VEC, int THREADS, int PER, int WG>
__global__ __launch_bounds__(WG) void norm_gate_backward_kernel(NormArgs a)
{
    constexpr int kGroups = WG / THREADS, N = VEC * PER;
    constexpr bool kKeep = WG <= 512;  // parameters in registers for all rows, where there are enough
    using R = Row<T, VEC, THREADS, PER>;
    using W = Raw<T, VEC, THREADS, PER>;
    using P = Param<VEC, THREADS, PER>;
    __shared__ float lds[8][THREADS / 64];
    __shared__ float join[kGroups > 1 ? kGroups : 1][kGroups > 1 ? THREADS * N : 1];
    const int sub = threadIdx.x % THREADS, group = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    const long long span0 = (long long)(blockIdx.x / a.per_span) * a.span;
    const long long begin = span0 + (long long)(blockIdx.x % a.per_span) * a.chunk;
    const int span_end = (int)(span0 + a.span < a.rows ? span0 + a.span : a.rows);
    const int r0 = (int)(begin < span_end ? begin : span_end), r1 = r0 + a.chunk < span_end ? r0 + a.chunk : span_end;
    float dw1[N], db1[N], dw2[N], db2[N], dg[N];
#pragma unroll
    for (int i = 0; i < N; i++) dw1[i] = db1[i] = dw2[i] = db2[i] = dg[i] = 0.0f;

    // The groups' sums of a column array, in group order; the first group has them.
    auto joined = [&](float (&v)[N]) {
        if constexpr (kGroups > 1) {
            __syncthreads();
            each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) { join[group][c] = v[i]; });
            __syncthreads();
            if (group == 0)
                each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) {
                    float s = 0.0f;
#pragma unroll
                    for (int g = 0; g < kGroups; g++) s += join[g][c];
                    v[i] = s;
                });
        }
    };
    W rx, rf, rg, rdy, rdh;
    auto fetch = [&](int row) {
        rx.load((const T*)a.x + (long long)row * a.sx, sub, a.dim);
        if (a.f) rf.load((const T*)a.f + (long long)row * a.sf, sub, a.dim);
        if (a.gate) rg.load((const T*)a.gate + (long long)(row / a.gate_rows) * a.sg, sub, a.dim);
        if (a.dh) rdh.load((const T*)a.dh + (long long)row * a.sh, sub, a.dim);
        if (a.dy) rdy.load((const T*)a.dy + (long long)row * a.sy, sub, a.dim);
    };
    P w1, b1, w2;
    auto parameters = [&] {
        w1.load(a.post_w, 1.0f, sub, a.dim);
        b1.load(a.post_b, 0.0f, sub, a.dim);
        w2.load(a.pre_w, 1.0f, sub, a.dim);
    };
    if (kKeep) parameters();

    int row = r0 + group;
    if (row < r1) fetch(row);
    int next_flush = a.gate_mode == kGateWhole ? r0 + a.gate_rows : 0x7fffffff;
    for (int base = r0; base < r1;) {
        const int stop = next_flush < r1 ? next_flush : r1;
        while (row < stop) {
            float n1[N], n2[N], d[N], g[N], dy[N];
            rx.widen(n2);
            if (a.f) rf.widen(n1);
            if (a.gate) rg.widen(g);
            if (a.dh) rdh.widen(d);
            if (a.dy) rdy.widen(dy);
            if (row + kGroups < r1) fetch(row + kGroups);
            if (!kKeep) parameters();
            float r_1 = 1.0f;
            if (a.f) {
                r_1 = normalise<VEC, THREADS, PER>(n1, a.post, sub, a.dim, a.inv_dim, a.eps, lds, 0);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    g[i] = a.gate ? a.beta * g[i] : a.beta;  // the block's factor
                    n2[i] = fmaf(g[i], fmaf(n1[i], w1.v[i], b1.v[i]), a.alpha * n2[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) n2[i] *= a.alpha;
            }
            if (a.dh) {
                const float r_2 = normalise<VEC, THREADS, PER>(n2, a.pre, sub, a.dim, a.inv_dim, a.eps, lds, 2);
                norm_back<VEC, THREADS, PER>(d, n2, r_2, a.pre, w2.v, dw2, db2, sub, a.dim, a.inv_dim, lds, 4);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) d[i] = 0.0f;
            }
            if (a.dy) {
#pragma unroll
                for (int i = 0; i < N; i++) d[i] += dy[i];
            }
            R out;
            if (a.dx) {
#pragma unroll
                for (int i = 0; i < N; i++) out.v[i] = a.alpha * d[i];
                out.store((T*)a.dx + (long long)row * a.sx, sub, a.dim);
            }
            if (a.f) {
                if (a.gate) {  // beta comes in where the sums are stored
#pragma unroll
                    for (int i = 0; i < N; i++) dg[i] = fmaf(d[i], fmaf(n1[i], w1.v[i], b1.v[i]), dg[i]);
                    if (a.gate_mode == kGateRow) {
#pragma unroll
                        for (int i = 0; i < N; i++) out.v[i] = a.beta * dg[i], dg[i] = 0.0f;
                        out.store((T*)a.dgate + (long long)row * a.sg, sub, a.dim);
                    }
                }
#pragma unroll
                for (int i = 0; i < N; i++) d[i] *= g[i];
                norm_back<VEC, THREADS, PER>(d, n1, r_1, a.post, w1.v, dw1, db1, sub, a.dim, a.inv_dim, lds, 6);
                if (a.df) {
#pragma unroll
                    for (int i = 0; i < N; i++) out.v[i] = d[i];
                    out.store((T*)a.df + (long long)row * a.sf, sub, a.dim);
                }
            }
            row += kGroups;
        }
        base = stop;
        if (a.gate_mode == kGateWhole) {
            joined(dg);
            if (group == 0) {
                R out;
#pragma unroll
                for (int i = 0; i < N; i++) out.v[i] = a.beta * dg[i];
                out.store((T*)a.dgate + (long long)((stop - 1) / a.gate_rows) * a.sg, sub, a.dim);
            }
#pragma unroll
            for (int i = 0; i < N; i++) dg[i] = 0.0f;
            next_flush = stop + a.gate_rows;
        }
    }
    float* own = a.sums + (long long)blockIdx.x * 4 * a.dim;
    auto finish = [&](float (&v)[N], int k) {
        if (!a.dst[k]) return;
        joined(v);
        float* to = a.parts > 1 ? own + (long long)k * a.dim : a.dst[k];
        if (group == 0) each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) { to[c] = v[i]; });
    };
    finish(dw1, 0);
    finish(db1, 1);
    finish(dw2, 2);
    finish(db2, 3);
    if (a.gate_mode == kGatePart) {
        joined(dg);
        if (group == 0)
            each<VEC, THREADS, PER>(sub, a.dim,
                                    [&](int i, int c) { a.gate_sums[(long long)blockIdx.x * a.dim + c] = a.beta * dg[i]; });
    }
}

// Sums of `parts` rows of src (stride apart) in a fixed order: 32 columns (a line)
// a workgroup, 8 interleaved shares of the parts.
constexpr int kSumColumns = 32, kSumShares = 256 / kSumColumns;
template <class T>
__device__ __forceinline__ void sum_parts(const float* src, long long stride, int parts, int dim, T* out, int column0)
{
    __shared__ float share[kSumShares][kSumColumns];
    const int lane = threadIdx.x % kSumColumns, w = threadIdx.x / kSumColumns, c = column0 + lane;
    float s[8] = {};
    if (c < dim) {
        int p = w;
        for (; p + 7 * kSumShares < parts; p += 8 * kSumShares)
#pragma unroll
            for (int q = 0; q < 8; q++) s[q] += src[(p + kSumShares * q) * stride + c];
        for (; p < parts; p += kSumShares) s[0] += src[p * stride + c];
    }
    share[w][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (w == 0 && c < dim) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kSumShares; i++) sum += share[i][lane];
        out[c] = (T)sum;
    }
}

// blockIdx.y: the parameters' four arrays, then the gate's groups (one launch:
// the two would run one after the other, 9 and 5 us at 1,037 parts of 1,280).
template <class T>
__global__ __launch_bounds__(256) void norm_sum_kernel(NormArgs a)
{
    const int y = blockIdx.y, column = blockIdx.x * kSumColumns;
    if (y >= 4)
        sum_parts(a.gate_sums + (y - 4ll) * a.per_span * a.dim, (long long)a.dim, a.per_span, a.dim,
                  (T*)a.dgate + (y - 4ll) * a.sg, column);
    else if (a.dst[y] && a.parts > 1)
        sum_parts(a.sums + (long long)y * a.dim, 4ll * a.dim, a.parts, a.dim, a.dst[y], column);
}

NormArgs norm_args(const NormGateOption& o, const NormGateTensors& t, int rows)
{
    require(o.dim >= 1 && o.dim <= kMaxDim, "dim must be 1..8192");
    require(o.postNorm >= NORM_NONE && o.postNorm <= NORM_LAYER && o.preNorm >= NORM_NONE && o.preNorm <= NORM_LAYER,
            "unknown norm");
    require_type(o.dataType);
    require(rows >= 0 && rows <= kMaxRows, "numRows must be 0..2^30");
    require(o.gateRows >= 0, "gateRows must be >= 0");
    require(o.epsilon >= 0.0f, "epsilon must be >= 0");
    require(t.f || (o.postNorm == NORM_NONE && o.gateRows == 0), "a post norm and a gate need f");
    require(o.postNorm != NORM_NONE || (!t.post_w && !t.post_b), "a post weight or bias needs a post norm");
    require(o.preNorm != NORM_NONE || (!t.pre_w && !t.pre_b), "a pre weight or bias needs a pre norm");
    require(rows == 0 || (o.gateRows > 0) == (t.gate != nullptr), "a gate needs gateRows >= 1, and gateRows a gate");
    require(o.strideX >= o.dim && (!t.f || o.strideF >= o.dim) && (o.gateRows == 0 || o.strideGate >= o.dim),
            "strides must be at least dim");
    require(rows == 0 || t.x, "null argument");
    NormArgs a{};
    a.x = t.x;
    a.f = t.f;
    a.gate = t.gate;
    a.post_w = t.post_w;
    a.post_b = t.post_b;
    a.pre_w = t.pre_w;
    a.pre_b = t.pre_b;
    a.sx = o.strideX;
    a.sf = o.strideF;
    a.sg = o.strideGate;
    a.sy = o.strideY;
    a.sh = o.strideH;
    a.rows = rows;
    a.dim = o.dim;
    a.gate_rows = o.gateRows > 0 ? std::min(o.gateRows, std::max(rows, 1)) : 1;
    a.post = o.postNorm;
    a.pre = o.preNorm;
    a.alpha = o.residualScale;
    a.beta = o.blockScale;
    a.eps = o.epsilon;
    a.inv_dim = (float)(1.0 / o.dim);
    return a;
}

struct Access {
    const void* p;
    long long stride;
};

bool norm_vec(int dim, int bytes, std::initializer_list<Access> all)
{
    bool ok = dim * bytes % 16 == 0;  // then the parameters' pieces are whole too
    for (const Access& x : all) ok = ok && (!x.p || (aligned16(x.p) && x.stride * bytes % 16 == 0));
    return ok;
}

template <class T, int VEC, int THREADS, int PER>
void forward_launch(NormArgs a, hipStream_t s)
{
    constexpr int kPerWg = 256 / THREADS;
    in_launches((a.rows + kPerWg - 1) / kPerWg, 256, [&](long long first, unsigned wgs) {
        a.row0 = first * kPerWg;
        norm_gate_kernel<T, VEC, THREADS, PER><<<wgs, 256, 0, s>>>(a);
    });
}

// A wave holds a row of up to 32 elements a lane; longer rows take a workgroup.
template <class T, int VEC>
void forward_rows(const NormArgs& a, hipStream_t s)
{
    const int pieces = (a.dim + VEC - 1) / VEC;
    constexpr int P = 32 / VEC;  // pieces of a thread at most
    if (pieces <= 16 * P) forward_launch<T, VEC, 64, (P + 3) / 4>(a, s);
    else if (pieces <= 32 * P) forward_launch<T, VEC, 64, P / 2>(a, s);
    else if (pieces <= 64 * P) forward_launch<T, VEC, 64, P>(a, s);
    else if (pieces <= 128 * P) forward_launch<T, VEC, 256, P / 2>(a, s);
    else forward_launch<T, VEC, 256, P>(a, s);
}

template <class T, int VEC, int THREADS, int PER, int WG>
void backward_launch(const NormArgs& a, hipStream_t s)
{
    norm_gate_backward_kernel<T, VEC, THREADS, PER, WG><<<a.parts, WG, 0, s>>>(a);
}

// Eight elements a thread: the five sums over rows, the row's own arrays and the
// next row stay in registers, up to 512 threads.  Whole waves, as few as hold the
// row.  The rows are dealt to twelve waves a CU, as many as are resident of aligned
// 16-bit rows; of most others eight are, and a third of the workgroups wait.
int backward_threads(int dim, int vec)
{
    const int lanes = ((dim + vec - 1) / vec + 8 / vec - 1) / (8 / vec);
    for (int t : {64, 128, 192, 256, 384}) {
        if (lanes <= t) return t;
    }
    return lanes <= 512 ? 512 : 1024;
}

template <class T, int VEC>
void backward_rows(const NormArgs& a, hipStream_t s)
{
    constexpr int P = 8 / VEC;
    switch (backward_threads(a.dim, VEC)) {
        case 64: return backward_launch<T, VEC, 64, P, 256>(a, s);
        case 128: return backward_launch<T, VEC, 128, P, 128>(a, s);
        case 192: return backward_launch<T, VEC, 192, P, 192>(a, s);
        case 256: return backward_launch<T, VEC, 256, P, 256>(a, s);
        case 384: return backward_launch<T, VEC, 384, P, 384>(a, s);
        case 512: return backward_launch<T, VEC, 512, P, 512>(a, s);
        default: return backward_launch<T, VEC, 1024, P, 1024>(a, s);
    }
}

}  // namespace

void norm_gate(const NormGateOption& o, const NormGateTensors& t, void* y, void* h, int rows, hipStream_t s)
{
    NormArgs a = norm_args(o, t, rows);
    require((!y || o.strideY >= o.dim) && (!h || o.strideH >= o.dim), "strides must be at least dim");
    if (rows == 0) return;
    require(y || h, "y and h are both NULL");
    require(y != t.x || o.strideY == o.strideX, "y in x's place needs x's stride");
    a.y = y;
    a.h = h;
    const int bytes = data_bytes(o.dataType);
    const bool vec = norm_vec(o.dim, bytes, {{t.x, a.sx}, {t.f, a.sf}, {t.gate, a.sg}, {y, a.sy}, {h, a.sh}, {t.post_w, 16}, {t.post_b, 16},
                                               {t.pre_w, 16}, {t.pre_b, 16}});
    with_type(o.dataType, [&](auto zero) {
        using T = decltype(zero);
        if (vec) forward_rows<T, 16 / (int)sizeof(T)>(a, s);
        else forward_rows<T, 1>(a, s);
    });
}

void norm_gate_backward(const NormGateOption& o, const NormGateTensors& t, const void* dy, const void* dh,
                        const NormGateGrads& g, int rows, hipStream_t s)
{
    NormArgs a = norm_args(o, t, rows);
    require((!dy || o.strideY >= o.dim) && (!dh || o.strideH >= o.dim), "strides must be at least dim");
    require(t.f || (!g.df && !g.dgate && !g.dpost_w && !g.dpost_b), "gradients of a block's side need f");
    require(!g.dgate || o.gateRows > 0, "dgate needs a gate");
    require(o.postNorm != NORM_NONE || (!g.dpost_w && !g.dpost_b), "post norm gradients need a post norm");
    require(o.preNorm != NORM_NONE || (!g.dpre_w && !g.dpre_b), "pre norm gradients need a pre norm");
    a.dy = dy;
    a.dh = dh;
    a.dx = g.dx;
    a.df = g.df;
    a.dgate = g.dgate;
    a.dst[0] = g.dpost_w;
    a.dst[1] = g.dpost_b;
    a.dst[2] = g.dpre_w;
    a.dst[3] = g.dpre_b;
    const int bytes = data_bytes(o.dataType);
    const bool vec = norm_vec(o.dim, bytes,
                              {{t.x, a.sx}, {t.f, a.sf}, {t.gate, a.sg}, {dy, a.sy}, {dh, a.sh}, {g.dx, a.sx}, {g.df, a.sf},
                               {g.dgate, a.sg}, {t.post_w, 16}, {t.post_b, 16}, {t.pre_w, 16}, {t.pre_b, 16}});
    const bool sums = g.dpost_w || g.dpost_b || g.dpre_w || g.dpre_b;
    // Rows of a workgroup: whole groups of the gate, or an even part of one, so
    // that no workgroup has rows of two gates whose sums it cannot finish; the
    // same ones whether the gate's gradient is asked for or not.
    const int threads = backward_threads(o.dim, vec ? 16 / bytes : 1), wg = threads == 64 ? 256 : threads;
    const int most = std::min(num_cus() * std::max(1, 768 / wg), std::max(1, rows / 4));
    int chunk = std::max(1, (rows + most - 1) / most);
    a.gate_mode = !t.gate ? kGateNone : a.gate_rows == 1 ? kGateRow : kGateWhole;
    if (a.gate_mode != kGateWhole || a.gate_rows >= rows) {
        a.span = std::max(rows, 1);
        a.per_span = std::max(1, (rows + chunk - 1) / chunk);
        if (a.gate_mode == kGateWhole && a.per_span > 1) a.gate_mode = kGatePart;
    } else if (a.gate_rows <= chunk) {
        chunk = round_up(chunk, a.gate_rows);
        a.span = chunk;
        a.per_span = 1;
    } else {
        a.per_span = (a.gate_rows + chunk - 1) / chunk;
        chunk = (a.gate_rows + a.per_span - 1) / a.per_span;
        a.span = a.gate_rows;
        if (a.per_span > 1) a.gate_mode = kGatePart;
    }
    if (!g.dgate) a.gate_mode = kGateNone;
    a.chunk = chunk;
    const int spans = std::max(1, (int)(((long long)rows + a.span - 1) / a.span));
    a.parts = spans * a.per_span;
    const bool to_scratch = (sums && a.parts > 1) || a.gate_mode == kGatePart;
    if (to_scratch) {
        const size_t columns = (size_t)a.parts * a.dim;
        a.sums = (float*)stream_workspace(s).get(columns * 5 * sizeof(float));
        a.gate_sums = a.sums + columns * 4;
    }
    with_type(o.dataType, [&](auto zero) {
        using T = decltype(zero);
        if (vec) backward_rows<T, 16 / (int)sizeof(T)>(a, s);
        else backward_rows<T, 1>(a, s);
        GRAFT_LAUNCH_CHECK();
        const int columns = (a.dim + kSumColumns - 1) / kSumColumns;
        if (to_scratch) norm_sum_kernel<T><<<dim3(columns, 4 + (a.gate_mode == kGatePart ? spans : 0)), 256, 0, s>>>(a);
    });
    GRAFT_LAUNCH_CHECK();
}

}  // namespace graft
