// Norms behind and before a block, with its gate and the scaled residual, for
// gfx950:
//   u = postnorm(f),  y = alpha x + beta g u,  h = prenorm(y)
// The backward recomputes both norms from x and f:
//   dn2 = dh w2            d  = dy + r2 (dn2 - mean dn2 - n2 mean(dn2 n2))
//   dx  = alpha d          dg = beta d u        du = beta g d
//   dn1 = du w1            df = r1 (dn1 - mean dn1 - n1 mean(dn1 n1))
//   dw2 = sum dh n2, db2 = sum dh, dw1 = sum du n1, db1 = sum du over the rows
// (the mean of dn only for layer norms).  Bound by memory: a row stays in
// registers between its passes, statistics in fp32.
#include "experts.h"
#include "lanes.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kMaxDim = 8192;
constexpr int kMaxParts = 1024;  // workgroups of a backward, each with its sums over rows

struct NormArgs {
    const void *x, *f, *gate;
    const float *post_w, *post_b, *pre_w, *pre_b;
    void *y, *h;
    long long sx, sf, sg, sy, sh;
    int rows, dim, gate_rows, post, pre;
    float alpha, beta, eps;
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

template <int VEC, int THREADS, int PER, class F>
__device__ __forceinline__ void each(int sub, int dim, F&& f)
{
#pragma unroll
    for (int i = 0; i < PER; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int c = (i * THREADS + sub) * VEC + j;
            if (c < dim) f(i * VEC + j, c);
        }
}

// Sum over the THREADS of a row, in the same order for all of them.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* lds)
{
    v = lanes_sum<64>(v);
    if constexpr (THREADS > 64) {
        constexpr int W = THREADS / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) v += lds[i];
    }
    return v;
}

// n = normalised v (in place) and 1 / its deviation; v's elements behind the
// row stay zero.
template <int VEC, int THREADS, int PER>
__device__ __forceinline__ float normalise(float (&v)[VEC * PER], int kind, int sub, int dim, float eps, float* lds)
{
    if (kind == NORM_NONE) return 1.0f;
    if (kind == NORM_LAYER) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC * PER; i++) sum += v[i];
        const float mean = row_sum<THREADS>(sum, lds) / (float)dim;
        each<VEC, THREADS, PER>(sub, dim, [&](int i, int) { v[i] -= mean; });
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC * PER; i++) sq = fmaf(v[i], v[i], sq);
    const float r = 1.0f / sqrtf(row_sum<THREADS>(sq, lds) / (float)dim + eps);
#pragma unroll
    for (int i = 0; i < VEC * PER; i++) v[i] *= r;
    return r;
}

template <class T, int VEC, int THREADS, int PER>
__global__ __launch_bounds__(256) void norm_gate_kernel(NormArgs a)
{
    __shared__ float lds[4];
    using R = Row<T, VEC, THREADS, PER>;
    const int sub = threadIdx.x & (THREADS - 1);
    const long long row = (long long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
    if (row >= a.rows) return;  // a row's threads return together; only whole workgroups meet at a barrier
    R y;
    y.load((const T*)a.x + row * a.sx, sub, a.dim);
    if (a.f) {
        R u;
        u.load((const T*)a.f + row * a.sf, sub, a.dim);
        normalise<VEC, THREADS, PER>(u.v, a.post, sub, a.dim, a.eps, lds);
        each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) {
            if (a.post_w) u.v[i] *= a.post_w[c];
            if (a.post_b) u.v[i] += a.post_b[c];
        });
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
    normalise<VEC, THREADS, PER>(y.v, a.pre, sub, a.dim, a.eps, lds);
    each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) {
        if (a.pre_w) y.v[i] *= a.pre_w[c];
        if (a.pre_b) y.v[i] += a.pre_b[c];
    });
    y.store((T*)a.h + row * a.sh, sub, a.dim);
}

// dL/dinput (in place of d) of a norm whose normalised input is n and 1 /
// deviation r; the parameters' sums of this row added.
template <int VEC, int THREADS, int PER>
__device__ __forceinline__ void norm_back(float (&d)[VEC * PER], const float (&n)[VEC * PER], float r, int kind,
                                          const float* w, float (&dw)[VEC * PER], float (&db)[VEC * PER], int sub, int dim,
                                          float* lds)
{
    if (kind == NORM_NONE) return;
    float m = 0.0f, p = 0.0f;
    each<VEC, THREADS, PER>(sub, dim, [&](int i, int c) {
        dw[i] = fmaf(d[i], n[i], dw[i]);
        db[i] += d[i];
        if (w) d[i] *= w[c];
        m += d[i];
        p = fmaf(d[i], n[i], p);
    });
    m = kind == NORM_LAYER ? row_sum<THREADS>(m, lds) / (float)dim : 0.0f;
    p = row_sum<THREADS>(p, lds) / (float)dim;
    each<VEC, THREADS, PER>(sub, dim, [&](int i, int) { d[i] = r * (d[i] - m - n[i] * p); });
}

// A workgroup: `chunk` rows of a span, its row groups (waves for THREADS 64)
// in turn; sums over its rows go to sums[part], or for one part to the outputs.
template <class T, int VEC, int THREADS, int PER, int WG>
__global__ __launch_bounds__(WG) void norm_gate_backward_kernel(NormArgs a)
{
    constexpr int kGroups = WG / THREADS;
    using R = Row<T, VEC, THREADS, PER>;
    __shared__ float lds[WG / 64];
    __shared__ float join[kGroups > 1 ? kGroups : 1][kGroups > 1 ? THREADS * VEC * PER : 1];
    const int sub = threadIdx.x & (THREADS - 1), group = threadIdx.x / THREADS;
    const long long span0 = (long long)(blockIdx.x / a.per_span) * a.span;
    const long long begin = span0 + (long long)(blockIdx.x % a.per_span) * a.chunk;
    const int span_end = (int)(span0 + a.span < a.rows ? span0 + a.span : a.rows);
    const int r0 = (int)(begin < span_end ? begin : span_end), r1 = r0 + a.chunk < span_end ? r0 + a.chunk : span_end;
    float dw1[R::N], db1[R::N], dw2[R::N], db2[R::N], dg[R::N];
#pragma unroll
    for (int i = 0; i < R::N; i++) dw1[i] = db1[i] = dw2[i] = db2[i] = dg[i] = 0.0f;

    // The groups' sums of a column array, in group order; the first group has them.
    auto joined = [&](float (&v)[R::N]) {
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

    int next_flush = a.gate_mode == kGateWhole ? r0 + a.gate_rows : 0x7fffffff;
    for (int base = r0; base < r1;) {
        const int stop = next_flush < r1 ? next_flush : r1;
        for (int row = base + group; row < stop; row += kGroups) {
            R n1, n2, d;
            float r_1 = 1.0f;
            n2.load((const T*)a.x + (long long)row * a.sx, sub, a.dim);
            const T* grow = a.gate ? (const T*)a.gate + (long long)(row / a.gate_rows) * a.sg : nullptr;
            if (a.f) {
                n1.load((const T*)a.f + (long long)row * a.sf, sub, a.dim);
                r_1 = normalise<VEC, THREADS, PER>(n1.v, a.post, sub, a.dim, a.eps, lds);
                R g;
                if (grow) g.load(grow, sub, a.dim);
                each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) {
                    float u = n1.v[i];
                    if (a.post_w) u *= a.post_w[c];
                    if (a.post_b) u += a.post_b[c];
                    if (grow) u *= g.v[i];
                    n2.v[i] = fmaf(a.alpha, n2.v[i], a.beta * u);
                });
            } else {
#pragma unroll
                for (int i = 0; i < R::N; i++) n2.v[i] *= a.alpha;
            }
            if (a.dh) {
                const float r_2 = normalise<VEC, THREADS, PER>(n2.v, a.pre, sub, a.dim, a.eps, lds);
                d.load((const T*)a.dh + (long long)row * a.sh, sub, a.dim);
                norm_back<VEC, THREADS, PER>(d.v, n2.v, r_2, a.pre, a.pre_w, dw2, db2, sub, a.dim, lds);
            } else {
#pragma unroll
                for (int i = 0; i < R::N; i++) d.v[i] = 0.0f;
            }
            if (a.dy) {
                R e;
                e.load((const T*)a.dy + (long long)row * a.sy, sub, a.dim);
#pragma unroll
                for (int i = 0; i < R::N; i++) d.v[i] += e.v[i];
            }
            if (a.dx) {
                R e;
#pragma unroll
                for (int i = 0; i < R::N; i++) e.v[i] = a.alpha * d.v[i];
                e.store((T*)a.dx + (long long)row * a.sx, sub, a.dim);
            }
            if (!a.f) continue;
            if (grow) {
                R g, own;
                g.load(grow, sub, a.dim);
#pragma unroll
                for (int i = 0; i < R::N; i++) own.v[i] = 0.0f;
                each<VEC, THREADS, PER>(sub, a.dim, [&](int i, int c) {
                    float u = n1.v[i];
                    if (a.post_w) u *= a.post_w[c];
                    if (a.post_b) u += a.post_b[c];
                    own.v[i] = a.beta * d.v[i] * u;
                    dg[i] += own.v[i];
                    d.v[i] *= a.beta * g.v[i];
                });
                if (a.gate_mode == kGateRow) own.store((T*)a.dgate + (long long)row * a.sg, sub, a.dim);
            } else {
#pragma unroll
                for (int i = 0; i < R::N; i++) d.v[i] *= a.beta;
            }
            norm_back<VEC, THREADS, PER>(d.v, n1.v, r_1, a.post, a.post_w, dw1, db1, sub, a.dim, lds);
            if (a.df) d.store((T*)a.df + (long long)row * a.sf, sub, a.dim);
        }
        base = stop;
        if (a.gate_mode == kGateWhole) {
            joined(dg);
            if (group == 0) {
                R out;
#pragma unroll
                for (int i = 0; i < R::N; i++) out.v[i] = dg[i];
                out.store((T*)a.dgate + (long long)((stop - 1) / a.gate_rows) * a.sg, sub, a.dim);
            }
#pragma unroll
            for (int i = 0; i < R::N; i++) dg[i] = 0.0f;
            next_flush = stop + a.gate_rows;
        }
    }
    float* own = a.sums + (long long)blockIdx.x * 4 * a.dim;
    auto finish = [&](float (&v)[R::N], int k) {
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
                                    [&](int i, int c) { a.gate_sums[(long long)blockIdx.x * a.dim + c] = dg[i]; });
    }
}

// Sums of `parts` rows of src (stride apart) in a fixed order: 64 columns a
// workgroup, four interleaved quarters of the parts.
template <class T>
__device__ __forceinline__ void sum_parts(const float* src, long long stride, int parts, int dim, T* out, int column0)
{
    __shared__ float quarter[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = column0 + lane;
    float s = 0.0f;
    if (c < dim)
        for (int p = w; p < parts; p += 4) s += src[p * stride + c];
    quarter[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < dim) out[c] = (T)(quarter[0][lane] + quarter[1][lane] + quarter[2][lane] + quarter[3][lane]);
}

__global__ __launch_bounds__(256) void norm_sum_kernel(NormArgs a)
{
    float* dst = a.dst[blockIdx.y];
    if (!dst) return;
    sum_parts(a.sums + (long long)blockIdx.y * a.dim, 4ll * a.dim, a.parts, a.dim, dst, blockIdx.x * 64);
}

template <class T>
__global__ __launch_bounds__(256) void gate_sum_kernel(NormArgs a)
{
    sum_parts(a.gate_sums + (long long)blockIdx.y * a.per_span * a.dim, (long long)a.dim, a.per_span, a.dim,
              (T*)a.dgate + (long long)blockIdx.y * a.sg, blockIdx.x * 64);
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
    return a;
}

struct Access {
    const void* p;
    long long stride;
};

bool norm_vec(int dim, int bytes, std::initializer_list<Access> all)
{
    bool ok = dim * bytes % 16 == 0;
    for (const Access& x : all) ok = ok && (!x.p || (aligned16(x.p) && x.stride * bytes % 16 == 0));
    return ok;
}

template <class T, int VEC, int THREADS, int PER>
void forward_launch(const NormArgs& a, hipStream_t s)
{
    const int per_wg = 256 / THREADS;
    norm_gate_kernel<T, VEC, THREADS, PER><<<(a.rows + per_wg - 1) / per_wg, 256, 0, s>>>(a);
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

// Sixteen elements a thread at most: five sums over rows and the row's own
// arrays stay in registers.
template <class T, int VEC>
void backward_rows(const NormArgs& a, hipStream_t s)
{
    const int pieces = (a.dim + VEC - 1) / VEC;
    constexpr int P = 16 / VEC;
    if (pieces <= 32 * P) backward_launch<T, VEC, 64, P / 2, 256>(a, s);
    else if (pieces <= 64 * P) backward_launch<T, VEC, 64, P, 256>(a, s);
    else if (pieces <= 128 * P) backward_launch<T, VEC, 256, P / 2, 256>(a, s);
    else if (pieces <= 256 * P) backward_launch<T, VEC, 256, P, 256>(a, s);
    else backward_launch<T, VEC, 512, P, 512>(a, s);
}

}  // namespace

void norm_gate(const NormGateOption& o, const NormGateTensors& t, void* y, void* h, int rows, hipStream_t s)
{
    NormArgs a = norm_args(o, t, rows);
    require((!y || o.strideY >= o.dim) && (!h || o.strideH >= o.dim), "strides must be at least dim");
    if (rows == 0) return;
    require(y || h, "y and h are both NULL");
    a.y = y;
    a.h = h;
    const int bytes = data_bytes(o.dataType);
    const bool vec = norm_vec(o.dim, bytes, {{t.x, a.sx}, {t.f, a.sf}, {t.gate, a.sg}, {y, a.sy}, {h, a.sh}});
    with_type(o.dataType, [&](auto zero) {
        using T = decltype(zero);
        if (vec) forward_rows<T, 16 / (int)sizeof(T)>(a, s);
        else forward_rows<T, 1>(a, s);
    });
    GRAFT_LAUNCH_CHECK();
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
    const bool sums = g.dpost_w || g.dpost_b || g.dpre_w || g.dpre_b;
    // Rows of a workgroup: whole groups of the gate, or an even part of one, so
    // that no workgroup has rows of two gates whose sums it cannot finish; the
    // same ones whether the gate's gradient is asked for or not.
    const int most = std::min(kMaxParts, std::max(1, rows / 4));
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
    const int bytes = data_bytes(o.dataType);
    const bool vec = norm_vec(o.dim, bytes,
                              {{t.x, a.sx}, {t.f, a.sf}, {t.gate, a.sg}, {dy, a.sy}, {dh, a.sh}, {g.dx, a.sx}, {g.df, a.sf},
                               {g.dgate, a.sg}});
    with_type(o.dataType, [&](auto zero) {
        using T = decltype(zero);
        if (vec) backward_rows<T, 16 / (int)sizeof(T)>(a, s);
        else backward_rows<T, 1>(a, s);
        GRAFT_LAUNCH_CHECK();
        const int columns = (a.dim + 63) / 64;
        if (sums && a.parts > 1) norm_sum_kernel<<<dim3(columns, 4), 256, 0, s>>>(a);
        if (a.gate_mode == kGatePart) gate_sum_kernel<T><<<dim3(columns, spans), 256, 0, s>>>(a);
    });
    GRAFT_LAUNCH_CHECK();
}

}  // namespace graft
