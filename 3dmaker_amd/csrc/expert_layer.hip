// The whole layer of experts for few tokens, for gfx950:
//   z = x R^T;  (e_j, w_j) = route(z);  a_j = act(W1_{e_j} x) [* (U1_{e_j} x)];
//   y = sum_j w_j W2_{e_j} a_j
// Bound by the weights' bytes: each selected expert's matrices are read once, for
// all tokens that take it.  Weights are widened to bf16 with their scales, which is
// exact, and go to v_mfma_f32_16x16x32_bf16 as 16 rows by 32 of k; tokens are its
// 16 columns, few or many, at the same cost.  Tokens and a_j are split into as many
// bf16 terms as they need (16-bit tokens are exact in one or two, fp32 ones in
// three; a_j has two, 16 bits, or three under fp32 tokens), so that nothing is
// rounded to 8 bits on the way.
#include "product.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kLayerThreads = 512, kLayerWaves = kLayerThreads / 64;
constexpr int kMaxTokens = EXPERT_LAYER_TOKENS;

struct LayerArgs {
    const void *x, *router;
    const float* bias;
    const uint8_t *w1, *s1, *w2, *s2;
    void* out;
    long long stride_x, stride_out;
    int tokens, experts, topk, dim, hidden, activation;
    bool gated, vec_x, vec_router, vec_out;
    int scale_shift;  // rows of a scale, as a shift
    int dim_pad, hidden_pad;  // filled up to whole blocks of 128
    // scratch
    float *logits, *weights;  // [tokens][experts], [tokens][topk]
    int *indices, *active;    // [tokens][topk]; number of experts that a token takes, and which
    uint8_t* place;           // [active][kMaxTokens]: the token's place for that expert, or kNone
    __bf16* acts;             // [tokens * topk][terms][hidden_pad]
};

constexpr int kNone = 255;

template <class T>
struct Terms {
    static constexpr int kX = sizeof(T) == 4 ? 3 : std::is_same_v<T, __bf16> ? 1 : 2;  // of a token
    static constexpr int kA = sizeof(T) == 4 ? 3 : 2;                                  // of a hidden activation
};

// v as N bf16 numbers: the first N - 1 cut, so that what is left over is exact, the
// last rounded.  Infinities and NaN are the first alone.
template <int N>
__device__ __forceinline__ void split(float v, __bf16 (&t)[N])
{
#pragma unroll
    for (int i = 0; i < N - 1; i++) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, v);
        if ((bits & 0x7f800000u) == 0x7f800000u) {
            t[i] = (__bf16)v;
            v = 0.0f;
        } else {
            const float cut = __builtin_bit_cast(float, bits & 0xffff0000u);
            t[i] = (__bf16)cut;
            v -= cut;
        }
    }
    t[N - 1] = (__bf16)v;
}

// Eight consecutive elements, zero from the n-th on.
template <class T>
__device__ __forceinline__ void load8(T (&v)[8], const T* p, int n, bool vec)
{
    if (vec && n >= 8) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            const Vec<T, N> w = *reinterpret_cast<const Vec<T, N>*>(p + i);
#pragma unroll
            for (int j = 0; j < N; j++) v[i + j] = w[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < n ? p[j] : (T)0.0f;
    }
}

// Logits of eight tokens and a wave's expert.
constexpr int kRouterTokens = 8;
template <class T, class R>
__global__ __launch_bounds__(256) void layer_logits_kernel(LayerArgs a)
{
    const int e = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, t0 = blockIdx.y * kRouterTokens;
    if (e >= a.experts) return;
    float acc[kRouterTokens];
#pragma unroll
    for (int t = 0; t < kRouterTokens; t++) acc[t] = 0.0f;
    const R* r = (const R*)a.router + (long long)e * a.dim;
    for (int d = lane * 8; d < a.dim; d += 512) {
        R w[8];
        load8(w, r + d, a.dim - d, a.vec_router);
#pragma unroll
        for (int t = 0; t < kRouterTokens; t++) {
            if (t0 + t >= a.tokens) break;
            T x[8];
            load8(x, (const T*)a.x + (t0 + t) * a.stride_x + d, a.dim - d, a.vec_x);
#pragma unroll
            for (int j = 0; j < 8; j++) acc[t] = fmaf((float)x[j], (float)w[j], acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < kRouterTokens; t++) {
        const float z = lanes_sum<64>(acc[t]);
        if (lane == 0 && t0 + t < a.tokens) a.logits[(long long)(t0 + t) * a.experts + e] = z;
    }
}

// The experts that some token takes, in their order, and the tokens' places for
// them.  One workgroup.
__global__ __launch_bounds__(256) void layer_plan_kernel(LayerArgs a)
{
    __shared__ uint32_t taken[32];
    __shared__ int before[32];
    if (threadIdx.x < 32) taken[threadIdx.x] = 0;
    __syncthreads();
    const int slots = a.tokens * a.topk;
    for (int i = threadIdx.x; i < slots; i += 256) {
        const int e = a.indices[i];
        if ((unsigned)e < (unsigned)a.experts) atomicOr(&taken[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int n = threadIdx.x < 32 ? __popc(taken[threadIdx.x]) : 0, up = lanes_scan(n);
        if (threadIdx.x < 32) before[threadIdx.x] = up - n;
        if (threadIdx.x == 63) a.active[0] = up;
    }
    __syncthreads();
    auto number = [&](int e) { return before[e >> 5] + __popc(taken[e >> 5] & ((1u << (e & 31)) - 1)); };
    const int count = before[31] + __popc(taken[31]);
    for (int e = threadIdx.x; e < a.experts; e += 256)
        if (taken[e >> 5] >> (e & 31) & 1) a.active[1 + number(e)] = e;
    for (int i = threadIdx.x; i < count * (kMaxTokens / 4); i += 256) reinterpret_cast<uint32_t*>(a.place)[i] = 0xffffffffu;
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += 256) {
        const int e = a.indices[i];
        if ((unsigned)e < (unsigned)a.experts) a.place[number(e) * kMaxTokens + i / a.topk] = (uint8_t)(i % a.topk);
    }
}

// A lane's 32 of the 128 k of a row: those from 32 quad on, eight to a matrix
// instruction.
template <int FORMAT>
struct Piece;

template <>
struct Piece<EXPERT_FP8> {
    i4v v[2];
    int byte;
    __device__ __forceinline__ void load(const uint8_t* row, const uint8_t* scales, int kb, int quad)
    {
        v[0] = *reinterpret_cast<const i4v*>(row + kb * 128 + quad * 32);
        v[1] = *reinterpret_cast<const i4v*>(row + kb * 128 + quad * 32 + 16);
        byte = scales[kb];
    }
    __device__ __forceinline__ bf16x8 operator()(int q) const
    {
        return widen(v[q >> 1][2 * (q & 1)], v[q >> 1][2 * (q & 1) + 1], scale_of(byte));
    }
};

template <>
struct Piece<EXPERT_FP4> {
    i4v v;
    int byte;
    __device__ __forceinline__ void load(const uint8_t* row, const uint8_t* scales, int kb, int quad)
    {
        v = *reinterpret_cast<const i4v*>(row + kb * 64 + quad * 16);
        byte = scales[kb * 4 + quad];
    }
    __device__ __forceinline__ bf16x8 operator()(int q) const
    {
        const float scale = byte == 255 ? __builtin_bit_cast(float, 0x7fc00000) : scale_of(byte);
        const uint32_t w = (uint32_t)v[q];
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
        const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
        return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

template <int FORMAT>
__device__ __forceinline__ long long pitch_of(int pad) { return FORMAT == EXPERT_FP4 ? pad / 2 : pad; }
template <int FORMAT>
__device__ __forceinline__ long long scale_pitch_of(int pad) { return FORMAT == EXPERT_FP4 ? pad / 32 : (pad / 128 + 3) / 4 * 4; }

// Rows and scale rows of expert e's matrix [rows x pad].
template <int FORMAT>
__device__ __forceinline__ const uint8_t* row_of(const uint8_t* w, int e, int rows, int pad, int row)
{
    return w + ((long long)e * rows + row) * pitch_of<FORMAT>(pad);
}
template <int FORMAT>
__device__ __forceinline__ const uint8_t* scales_of(const uint8_t* s, int e, int rows, int pad, int row, int shift)
{
    return s + ((long long)e * ((rows + (1 << shift) - 1) >> shift) + (row >> shift)) * scale_pitch_of<FORMAT>(pad);
}

__device__ __forceinline__ float activate(int kind, float v)
{
    switch (kind) {
        case EXPERT_RELU: return v < 0.0f ? 0.0f : v;  // NaN stays
        case EXPERT_SILU: return v / (1.0f + expf(-v));
        case EXPERT_GELU: return 0.5f * v * (1.0f + erff(v * 0.707106781f));
        default: return v;
    }
}

// The hidden activations of 16 rows for all tokens of an active expert: waves share
// out k.
template <int FORMAT, class T, int MT>
__global__ __launch_bounds__(kLayerThreads) void layer_hidden_kernel(LayerArgs a)
{
    constexpr int X = Terms<T>::kX, A = Terms<T>::kA;
    __shared__ f4 sums[kLayerWaves][2][MT][64];
    __shared__ int slots[kMaxTokens];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4, n0 = blockIdx.x * 16;
    if ((int)blockIdx.y >= a.active[0]) return;
    const int e = a.active[1 + blockIdx.y];
    const int place = lane < a.tokens ? a.place[blockIdx.y * kMaxTokens + lane] : kNone;
    const uint64_t mask = __ballot(place != kNone);
    const int count = __popcll(mask);
    if (wave == 0 && place != kNone) slots[__popcll(mask & ((1ull << lane) - 1))] = lane * a.topk + place;
    __syncthreads();
    const T* x[MT];
#pragma unroll
    for (int j = 0; j < MT; j++)
        x[j] = j * 16 + col < count ? (const T*)a.x + slots[j * 16 + col] / a.topk * a.stride_x + quad * 32 : nullptr;
    const int rows = a.gated ? 2 * a.hidden : a.hidden, row = min(n0 + col, a.hidden - 1);
    const uint8_t *W[2], *S[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
        const int r = g && a.gated ? a.hidden + row : row;
        W[g] = row_of<FORMAT>(a.w1, e, rows, a.dim_pad, r);
        S[g] = scales_of<FORMAT>(a.s1, e, rows, a.dim_pad, r, a.scale_shift);
    }
    f4 acc[2][MT];
#pragma unroll
    for (int j = 0; j < MT; j++) acc[0][j] = acc[1][j] = f4zero();
    for (int kb = wave; kb < a.dim_pad / 128; kb += kLayerWaves) {
        Piece<FORMAT> w[2];
        w[0].load(W[0], S[0], kb, quad);
        if (a.gated) w[1].load(W[1], S[1], kb, quad);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            bf16x8 t[MT][X];
#pragma unroll
            for (int j = 0; j < MT; j++) {
                T v[8];
                if (x[j]) load8(v, x[j] + kb * 128 + q * 8, a.dim - (kb * 128 + quad * 32 + q * 8), a.vec_x);
                else {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = (T)0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    __bf16 s[X];
                    if constexpr (X == 1) s[0] = v[i];
                    else split((float)v[i], s);
#pragma unroll
                    for (int u = 0; u < X; u++) t[j][u][i] = s[u];
                }
            }
#pragma unroll
            for (int g = 0; g < 2; g++) {
                if (g && !a.gated) break;
                const bf16x8 b = w[g](q);
#pragma unroll
                for (int j = 0; j < MT; j++) {
                    if (j * 16 >= count) break;
#pragma unroll
                    for (int u = 0; u < X; u++) acc[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, t[j][u], acc[g][j], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MT; j++) sums[wave][0][j][lane] = acc[0][j], sums[wave][1][j][lane] = acc[1][j];
    __syncthreads();
    for (int j = wave; j < MT; j += kLayerWaves) {
        if (j * 16 + col >= count) continue;
        f4 v = sums[0][0][j][lane], u = sums[0][1][j][lane];
        for (int w = 1; w < kLayerWaves; w++) v += sums[w][0][j][lane], u += sums[w][1][j][lane];
        Vec<__bf16, 4> o[A];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float h = activate(a.activation, v[i]);
            if (a.gated) h *= u[i];
            if (n0 + quad * 4 + i >= a.hidden) h = 0.0f;
            __bf16 s[A];
            split(h, s);
#pragma unroll
            for (int t = 0; t < A; t++) o[t][i] = s[t];
        }
        __bf16* to = a.acts + (long long)slots[j * 16 + col] * A * a.hidden_pad + n0 + quad * 4;
#pragma unroll
        for (int t = 0; t < A; t++) *reinterpret_cast<Vec<__bf16, 4>*>(to + (long long)t * a.hidden_pad) = o[t];
    }
}

// 16 columns of the outputs for all tokens: waves share out the active experts' k.
// An expert's sums are kept apart, so that its NaN reach its own tokens alone.
template <int FORMAT, class T, int MT>
__global__ __launch_bounds__(kLayerThreads) void layer_out_kernel(LayerArgs a)
{
    constexpr int A = Terms<T>::kA;
    __shared__ f4 sums[kLayerWaves][MT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4, d0 = blockIdx.x * 16;
    const int blocks = a.hidden_pad / 128, items = a.active[0] * blocks;  // at most 2^10 * 2^7
    const int first = items * wave / kLayerWaves, last = items * (wave + 1) / kLayerWaves;
    const int row = min(d0 + col, a.dim - 1);
    f4 acc[MT], own[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) acc[j] = f4zero();
    for (int n = first / blocks; n * blocks < last; n++) {
        const int e = a.active[1 + n];
        const __bf16* act[MT];
        float weight[MT];
        bool some[MT];
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int t = j * 16 + col, place = t < a.tokens ? a.place[n * kMaxTokens + t] : kNone;
            const int slot = t * a.topk + place;
            act[j] = place != kNone ? a.acts + (long long)slot * A * a.hidden_pad + quad * 32 : nullptr;
            weight[j] = place != kNone ? a.weights[slot] : 0.0f;
            some[j] = __ballot(place != kNone) != 0;
            own[j] = f4zero();
        }
        const uint8_t* W = row_of<FORMAT>(a.w2, e, a.dim, a.hidden_pad, row);
        const uint8_t* S = scales_of<FORMAT>(a.s2, e, a.dim, a.hidden_pad, row, a.scale_shift);
        for (int kb = max(first - n * blocks, 0); kb < min(last - n * blocks, blocks); kb++) {
            Piece<FORMAT> w;
            w.load(W, S, kb, quad);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const bf16x8 b = w(q);
#pragma unroll
                for (int j = 0; j < MT; j++) {
                    if (!some[j]) continue;
#pragma unroll
                    for (int u = 0; u < A; u++) {
                        bf16x8 t{};
                        if (act[j]) t = *reinterpret_cast<const bf16x8*>(act[j] + (long long)u * a.hidden_pad + kb * 128 + q * 8);
                        own[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, t, own[j], 0, 0, 0);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[j][i] = act[j] ? fmaf(weight[j], own[j][i], acc[j][i]) : acc[j][i];
    }
#pragma unroll
    for (int j = 0; j < MT; j++) sums[wave][j][lane] = acc[j];
    __syncthreads();
    for (int j = wave; j < MT; j += kLayerWaves) {
        f4 v = sums[0][j][lane];
        for (int w = 1; w < kLayerWaves; w++) v += sums[w][j][lane];
        const int t = j * 16 + col, d = d0 + quad * 4;
        if (t >= a.tokens) continue;
        T* to = (T*)a.out + t * a.stride_out + d;
        if (a.vec_out && d + 4 <= a.dim) {
            Vec<T, 4> o;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = (T)v[i];
            *reinterpret_cast<Vec<T, 4>*>(to) = o;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (d + i < a.dim) to[i] = (T)v[i];
        }
    }
}

template <int FORMAT, class T, int MT>
void layer_launch(const LayerArgs& a, hipStream_t s)
{
    const unsigned most = (unsigned)std::min(a.experts, a.tokens * a.topk);
    layer_hidden_kernel<FORMAT, T, MT><<<dim3(a.hidden_pad / 16, most), kLayerThreads, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
    layer_out_kernel<FORMAT, T, MT><<<(a.dim + 15) / 16, kLayerThreads, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

}  // namespace

void expert_layer(const ExpertLayerOption& o, const ExpertLayerTensors& t, void* out, int tokens, hipStream_t s)
{
    check_route_option(o.route);
    require(o.route.logitsType == DATA_F32, "route.logitsType must be DATA_F32");
    require(tokens >= 0 && tokens <= kMaxTokens, "numTokens must be 0..64");
    require(o.dim >= 1 && o.dim <= 16384 && o.hidden >= 1 && o.hidden <= 16384, "dim and hidden must be 1..16384");
    require(o.activation >= EXPERT_LINEAR && o.activation <= EXPERT_GELU, "unknown activation");
    require(o.weightFormat == EXPERT_FP8 || o.weightFormat == EXPERT_FP4, "unknown weightFormat");
    require(o.scaleRows == 1 || (o.scaleRows == 128 && o.weightFormat == EXPERT_FP8),
            "scaleRows must be 1, or 128 with EXPERT_FP8");
    require_type(o.dataType);
    require_type(o.routerType);
    require(o.strideX >= o.dim && o.strideOut >= o.dim, "strides must be at least dim");
    if (tokens == 0) return;
    require(t.x && t.router && t.w1 && t.w1_scales && t.w2 && t.w2_scales && out, "null argument");
    require(aligned16(t.w1) && aligned16(t.w2) && ((uintptr_t)t.w1_scales & 3) == 0 && ((uintptr_t)t.w2_scales & 3) == 0,
            "weights must be 16-byte aligned and scales 4-byte aligned");
    LayerArgs a{};
    a.x = t.x;
    a.router = t.router;
    a.bias = t.bias;
    a.w1 = t.w1;
    a.s1 = t.w1_scales;
    a.w2 = t.w2;
    a.s2 = t.w2_scales;
    a.out = out;
    a.stride_x = o.strideX;
    a.stride_out = o.strideOut;
    a.tokens = tokens;
    a.experts = o.route.numExperts;
    a.topk = o.route.topK;
    a.dim = o.dim;
    a.hidden = o.hidden;
    a.activation = o.activation;
    a.gated = o.gated != 0;
    const int bytes = data_bytes(o.dataType);
    a.vec_x = aligned16(t.x) && o.strideX * bytes % 16 == 0;
    a.vec_router = aligned16(t.router) && (long long)o.dim * data_bytes(o.routerType) % 16 == 0;
    a.vec_out = aligned16(out) && o.strideOut * bytes % 16 == 0;
    a.scale_shift = o.scaleRows == 128 ? 7 : 0;
    a.dim_pad = round_up(o.dim, 128);
    a.hidden_pad = round_up(o.hidden, 128);
    const int slots = tokens * a.topk, most = std::min(a.experts, slots);
    size_t size = 0;
    auto take = [&](size_t n) {
        const size_t at = size;
        size += round_up<size_t>(n, 256);
        return at;
    };
    const size_t at_logits = take((size_t)tokens * a.experts * 4), at_weights = take((size_t)slots * 4);
    const size_t at_indices = take((size_t)slots * 4), at_active = take((size_t)(most + 1) * 4);
    const size_t at_place = take((size_t)most * kMaxTokens);
    const size_t at_acts = take((size_t)slots * (o.dataType == DATA_F32 ? 3 : 2) * a.hidden_pad * 2);
    char* ws = (char*)stream_workspace(s).get(size);
    a.logits = (float*)(ws + at_logits);
    a.weights = (float*)(ws + at_weights);
    a.indices = (int*)(ws + at_indices);
    a.active = (int*)(ws + at_active);
    a.place = (uint8_t*)(ws + at_place);
    a.acts = (__bf16*)(ws + at_acts);
    with_type(o.dataType, [&](auto x) {
        using T = decltype(x);
        with_type(o.routerType, [&](auto r) {
            layer_logits_kernel<T, decltype(r)>
                <<<dim3((a.experts + 3) / 4, (tokens + kRouterTokens - 1) / kRouterTokens), 256, 0, s>>>(a);
        });
        GRAFT_LAUNCH_CHECK();
        route_experts(o.route, a.logits, a.experts, a.bias, a.indices, a.weights, tokens, s);
        layer_plan_kernel<<<1, 256, 0, s>>>(a);
        GRAFT_LAUNCH_CHECK();
        auto with_tiles = [&](auto F) {
            constexpr int format = decltype(F)::value;
            if (tokens <= 16) layer_launch<format, T, 1>(a, s);
            else if (tokens <= 32) layer_launch<format, T, 2>(a, s);
            else layer_launch<format, T, 4>(a, s);
        };
        if (o.weightFormat == EXPERT_FP8) with_tiles(std::integral_constant<int, EXPERT_FP8>{});
        else with_tiles(std::integral_constant<int, EXPERT_FP4>{});
    });
}

}  // namespace graft
