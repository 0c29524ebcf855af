// The whole layer of experts for few tokens, for gfx950:
//   z = x R^T;  (e_j, w_j) = route(z);  a_j = act(W1_{e_j} x) [* (U1_{e_j} x)];
//   y = sum_j w_j W2_{e_j} a_j
// Bound by the weights' bytes: each selected expert's matrices are read once, for
// all tokens that take it.  Weights are widened to bf16 with their scales, which is
// exact, and go to v_mfma_f32_16x16x32_bf16 as 16 rows by 32 of k; an expert's slots
// (a token's place for it) are its 16 columns, few or many, at the same cost.  Tokens
// and a_j are split into as many bf16 terms as they need (16-bit tokens are exact in
// one or two, fp32 ones in three; a_j has two, 16 bits, or three under fp32 tokens),
// so that nothing is rounded to 8 bits on the way.
//
// Three launches: routing (the last workgroup to have its logits ready routes all
// tokens), the hidden activations, the outputs.
#include "product.h"
#include "route_math.h"

#include <algorithm>

namespace graft {

namespace {

constexpr int kLayerThreads = 512, kLayerWaves = kLayerThreads / 64;
constexpr int kRouteThreads = 1024, kRouteWaves = kRouteThreads / 64;
constexpr int kMaxTokens = EXPERT_LAYER_TOKENS;

struct LayerArgs {
    const void *x, *router;
    const float* bias;
    const uint8_t *w1, *s1, *w2, *s2;
    void* out;
    long long stride_x, stride_out;
    int tokens, experts, topk, dim, hidden, activation;
    int groups, kept, group_best;
    float scale;
    bool sigmoid, renorm, gated, vec_x, vec_router, vec_out;
    int scale_shift;          // rows of a scale, as a shift
    int dim_pad, hidden_pad;  // filled up to whole blocks of 128
    // scratch
    float *logits, *weights;  // [tokens][experts], [slots]
    int* active;              // number of experts that some token takes, and which
    int *first, *slots;       // where their slots begin in the list of slots, and its end
    __bf16 *xs, *acts;        // [tokens][terms][dim_pad], [slots][terms][hidden_pad]
    float* parts;             // [parts][tokens][dim], of more than one part
    uint32_t *route_ticket, *out_tickets;
};

template <class T>
struct Terms {
    static constexpr int kX = sizeof(T) == 4 ? 3 : std::is_same_v<T, __bf16> ? 1 : 2;  // of a token or a router's row
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

template <class T, int N = Terms<T>::kX>
__device__ __forceinline__ void split8(const T (&v)[8], bf16x8 (&t)[N])
{
#pragma unroll
    for (int i = 0; i < 8; i++) {
        __bf16 s[N];
        if constexpr (N == 1) s[0] = v[i];
        else split((float)v[i], s);
#pragma unroll
        for (int u = 0; u < N; u++) t[u][i] = s[u];
    }
}

// ---------------------------------------------------------------------------
// routing
// ---------------------------------------------------------------------------

// A token by a wave: lane l has experts PER l .. PER l + PER - 1, so that lane order
// is index order.  scores, and keys with groups: LDS of the wave, one an expert.
template <int PER>
__device__ __forceinline__ void route_token(const LayerArgs& a, int t, float* scores, uint32_t* keys)
{
    const int lane = threadIdx.x & 63, first = lane * PER, n = a.experts - first;
    float s[PER];
    uint32_t key[PER];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float z = i < n ? a.logits[(long long)t * a.experts + first + i] : -INFINITY;
        s[i] = z > -INFINITY ? fminf(z, 3.402823466e38f) : -INFINITY;  // NaN: none
        top = fmaxf(top, s[i]);
    }
    float sum = 0.0f;
    top = lanes_max<64>(top);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        key[i] = s[i] > -INFINITY;
        if (a.sigmoid) {
            const float e = exp_neg(-fabsf(s[i])), r = __builtin_amdgcn_rcpf(1.0f + e);
            s[i] = key[i] ? (s[i] >= 0.0f ? r : e * r) : 0.0f;
        } else {
            s[i] = key[i] ? exp_neg(s[i] - top) : 0.0f;
            sum += s[i];
        }
    }
    if (!a.sigmoid) {
        sum = lanes_sum<64>(sum);
        sum = sum > 0.0f ? 1.0f / sum : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (!a.sigmoid) s[i] *= sum;
        const float c = s[i] + (a.bias && i < n ? a.bias[first + i] : 0.0f);
        key[i] = key[i] && c > -INFINITY ? key_of(c) : 0u;
        if (i < n) scores[first + i] = s[i];
    }
    if (a.groups > 1) {
        const int size = a.experts / a.groups;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (i < n) keys[first + i] = key[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        uint32_t b1 = 0, b2 = 0;  // lane g: the best two of group g
        if (lane < a.groups)
            for (int i = 0; i < size; i++) {
                const uint32_t k = keys[lane * size + i];
                b2 = max(b2, min(b1, k));
                b1 = max(b1, k);
            }
        uint32_t g = b1;
        if (a.group_best == 2 && b2 != 0) g = key_of(of_key(b1) + of_key(b2));
        int ahead = 0;
        for (int o = 0; o < a.groups; o++) {
            const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)g, o);
            ahead += k > g || (k == g && o < lane);
        }
        const uint64_t kept = __ballot(lane < a.groups && ahead < a.kept);
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (i < n && !(kept >> ((first + i) / size) & 1)) key[i] = 0;
        __builtin_amdgcn_wave_barrier();
    }
    int mine = -1;  // lane j: the j-th pick
#pragma unroll 1
    for (int j = 0; j < a.topk; j++) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < PER; i++) best = max(best, key[i]);
        const uint32_t all = lanes_umax<64>(best);
        if (all == 0) break;
        const int l = __ffsll((unsigned long long)__ballot(best == all)) - 1;
        int at = 0;
#pragma unroll
        for (int i = PER - 1; i >= 0; i--) at = key[i] == all ? i : at;
#pragma unroll
        for (int i = 0; i < PER; i++) key[i] = lane == l && i == at ? 0u : key[i];
        const int e = __builtin_amdgcn_readlane(first + at, l);
        mine = lane == j ? e : mine;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float score = mine >= 0 ? scores[mine] : 0.0f;
    __builtin_amdgcn_wave_barrier();
    if (a.renorm) {
        const float total = lanes_sum<64>(score);
        score *= a.scale / (total + 1e-20f);
    } else score *= a.scale;
    if (lane < a.topk) {
        a.weights[t * a.topk + lane] = score;
        a.slots[t * a.topk + lane] = mine;  // for now the slot's expert
    }
}

// The experts that some token takes, in their order, and the list of their slots.
__device__ __forceinline__ void plan(const LayerArgs& a, int* lds)
{
    int* const count = lds;              // [experts]: slots; then where the expert's next goes
    int* const expert = lds + a.experts; // [slots]
    const int slots = a.tokens * a.topk;
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) count[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += kRouteThreads) {
        expert[i] = a.slots[i];
        if (expert[i] >= 0) atomicAdd(&count[expert[i]], 1);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        int number = 0, begin = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int e = e0 + threadIdx.x, n = e < a.experts ? count[e] : 0;
            const int upn = lanes_scan(n > 0), ups = lanes_scan(n);
            if (n > 0) {
                a.active[1 + number + upn - 1] = e;
                a.first[number + upn - 1] = begin + ups - n;
                count[e] = begin + ups - n;
            }
            number += __shfl(upn, 63);
            begin += __shfl(ups, 63);
        }
        if (threadIdx.x == 0) a.active[0] = number, a.first[number] = begin;
    }
    __syncthreads();
    // an expert's slots in any order: each has a column of its own
    for (int i = threadIdx.x; i < slots; i += kRouteThreads)
        if (expert[i] >= 0) a.slots[atomicAdd(&count[expert[i]], 1)] = i;
}

// Logits of 16 experts, waves sharing out k; the tokens' terms on the way; routing
// and plan by the workgroup that is last.  Products of terms are exact; those of
// 2^-24 of a product and less are left out.
template <class T, class R, int MT>
__global__ __launch_bounds__(kRouteThreads) void layer_route_kernel(LayerArgs a)
{
    constexpr int X = Terms<T>::kX, Y = Terms<R>::kX;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ bool last;
    f4* const sums = reinterpret_cast<f4*>(lds);  // [waves][MT][64]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4, e0 = blockIdx.x * 16;
    const int blocks = a.dim_pad / 128;
    f4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) acc[j] = f4zero();
    const R* r = (const R*)a.router + (long long)min(e0 + col, a.experts - 1) * a.dim;
    for (int kb = wave; kb < blocks; kb += kRouteWaves) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int k = kb * 128 + quad * 32 + q * 8;
            R v[8];
            bf16x8 y[Y];
            load8(v, r + k, a.dim - k, a.vec_router);
            split8(v, y);
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const int t = j * 16 + col;
                T u[8];
                bf16x8 x[X];
                load8(u, (const T*)a.x + min(t, a.tokens - 1) * a.stride_x + k, a.dim - k, a.vec_x);
                split8(u, x);
#pragma unroll
                for (int m = 0; m < X; m++)
#pragma unroll
                    for (int n = 0; n < Y; n++)
                        if (m + n < 3) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[n], x[m], acc[j], 0, 0, 0);
                // each workgroup stores some blocks of the terms
                if (kb % gridDim.x == blockIdx.x && t < a.tokens) {
#pragma unroll
                    for (int m = 0; m < X; m++)
                        *reinterpret_cast<bf16x8*>(a.xs + ((long long)t * X + m) * a.dim_pad + k) = x[m];
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MT; j++) sums[(wave * MT + j) * 64 + lane] = acc[j];
    __syncthreads();
    if (wave < MT) {
        f4 v = sums[wave * 64 + lane];
        for (int w = 1; w < kRouteWaves; w++) v += sums[(w * MT + wave) * 64 + lane];
        const int t = wave * 16 + col;
        if (t < a.tokens) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e0 + quad * 4 + i < a.experts) a.logits[(long long)t * a.experts + e0 + quad * 4 + i] = v[i];
        }
    }
    __syncthreads();
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) {
            __threadfence();
            last = atomicAdd(a.route_ticket, 1u) == gridDim.x - 1;
        }
        __syncthreads();
        if (!last) return;
        if (threadIdx.x == 0) *a.route_ticket = 0;
        __threadfence();
    }
    if (a.out_tickets)
        for (int i = threadIdx.x; i < (a.dim + 15) / 16; i += kRouteThreads) a.out_tickets[i] = 0;
    float* const scores = reinterpret_cast<float*>(lds) + wave * a.experts;
    uint32_t* const keys = reinterpret_cast<uint32_t*>(lds) + (kRouteWaves + wave) * a.experts;
    for (int t = wave; t < a.tokens; t += kRouteWaves) {
        if (a.experts <= 64) route_token<1>(a, t, scores, keys);
        else if (a.experts <= 128) route_token<2>(a, t, scores, keys);
        else if (a.experts <= 256) route_token<4>(a, t, scores, keys);
        else route_token<16>(a, t, scores, keys);
    }
    __syncthreads();
    plan(a, reinterpret_cast<int*>(lds));
}

// ---------------------------------------------------------------------------
// the experts' products
// ---------------------------------------------------------------------------

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

// The hidden activations of 16 NT rows for the slots of an active expert, 16 CT at a
// time: waves share out k, and their sums are joined in LDS in wave order.  A lane
// whose column has no slot works on the first one's for nothing.
template <int FORMAT, class T, int G, int NT, int CT>
__global__ __launch_bounds__(kLayerThreads) void layer_hidden_kernel(LayerArgs a)
{
    constexpr int X = Terms<T>::kX, A = Terms<T>::kA, F = G * NT;
    __shared__ f4 sums[kLayerWaves][F][CT][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int col = lane & 15, quad = lane >> 4, n0 = blockIdx.x * 16 * NT, n = blockIdx.y;
    if (n >= a.active[0]) return;
    const int e = a.active[1 + n], first = a.first[n], count = a.first[n + 1] - first;
    const uint8_t *W[F], *S[F];
#pragma unroll
    for (int f = 0; f < F; f++) {
        const int row = min(n0 + f % NT * 16 + col, a.hidden - 1) + f / NT * a.hidden;
        W[f] = row_of<FORMAT>(a.w1, e, G * a.hidden, a.dim_pad, row);
        S[f] = scales_of<FORMAT>(a.s1, e, G * a.hidden, a.dim_pad, row, a.scale_shift);
    }
    const int blocks = a.dim_pad / 128;
    for (int s0 = 0; s0 < count; s0 += 16 * CT) {
        int slot[CT];
        const __bf16* x[CT];
        f4 acc[F][CT];
#pragma unroll
        for (int j = 0; j < CT; j++) {
            const int c = s0 + j * 16 + col;
            slot[j] = c < count ? a.slots[first + c] : -1;
            x[j] = a.xs + (long long)(max(slot[j], 0) / a.topk) * X * a.dim_pad + quad * 32;
#pragma unroll
            for (int f = 0; f < F; f++) acc[f][j] = f4zero();
        }
        auto load = [&](Piece<FORMAT>(&w)[F], int kb) {
#pragma unroll
            for (int f = 0; f < F; f++) w[f].load(W[f], S[f], kb, quad);
        };
        auto work = [&](const Piece<FORMAT>(&w)[F], int kb) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                bf16x8 t[CT][X];
#pragma unroll
                for (int j = 0; j < CT; j++)
#pragma unroll
                    for (int u = 0; u < X; u++)
                        t[j][u] = *reinterpret_cast<const bf16x8*>(x[j] + (long long)u * a.dim_pad + kb * 128 + q * 8);
#pragma unroll
                for (int f = 0; f < F; f++) {
                    const bf16x8 b = w[f](q);
#pragma unroll
                    for (int j = 0; j < CT; j++)
#pragma unroll
                        for (int u = 0; u < X; u++)
                            acc[f][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, t[j][u], acc[f][j], 0, 0, 0);
                }
            }
        };
        Piece<FORMAT> w0[F], w1[F];
        int kb = wave;
        if (kb < blocks) load(w0, kb);
        while (kb < blocks) {
            if (kb + waves < blocks) load(w1, kb + waves);
            work(w0, kb);
            kb += waves;
            if (kb >= blocks) break;
            if (kb + waves < blocks) load(w0, kb + waves);
            work(w1, kb);
            kb += waves;
        }
        if (s0 > 0) __syncthreads();
#pragma unroll
        for (int f = 0; f < F; f++)
#pragma unroll
            for (int j = 0; j < CT; j++) sums[wave][f][j][lane] = acc[f][j];
        __syncthreads();
#pragma unroll
        for (int f = 0; f < NT; f++)
#pragma unroll
            for (int j = 0; j < CT; j++) {
                if ((f * CT + j) % waves != wave || slot[j] < 0) continue;
                f4 v = sums[0][f][j][lane], u = f4zero();
                for (int w = 1; w < waves; w++) v += sums[w][f][j][lane];
                if (G == 2)
                    for (int w = 0; w < waves; w++) u += sums[w][F - NT + f][j][lane];
                const int row = n0 + f * 16 + quad * 4;
                Vec<__bf16, 4> o[A];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float h = activate(a.activation, v[i]);
                    if (G == 2) h *= u[i];
                    if (row + i >= a.hidden) h = 0.0f;
                    __bf16 s[A];
                    split(h, s);
#pragma unroll
                    for (int t = 0; t < A; t++) o[t][i] = s[t];
                }
                __bf16* to = a.acts + (long long)slot[j] * A * a.hidden_pad + row;
#pragma unroll
                for (int t = 0; t < A; t++) *reinterpret_cast<Vec<__bf16, 4>*>(to + (long long)t * a.hidden_pad) = o[t];
            }
    }
}

// 16 NT columns of the outputs for all tokens, and a part of the active experts' k:
// its waves share that out in runs of one expert's, whose sums go, weighted, to the
// tokens' in LDS.  Where k is in more than one part, the last workgroup of a tile
// joins them in their order.
template <int FORMAT, class T, int NT, int CT>
__global__ __launch_bounds__(kLayerThreads) void layer_out_kernel(LayerArgs a)
{
    constexpr int A = Terms<T>::kA;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ bool last;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int col = lane & 15, quad = lane >> 4, d0 = blockIdx.x * 16 * NT;
    const int slots = a.tokens * a.topk, most = min(a.experts, slots);
    f4* const sums = reinterpret_cast<f4*>(lds);  // [waves][tokens][4 NT]
    int* const active = reinterpret_cast<int*>(sums + waves * a.tokens * 4 * NT);
    int *const first = active + most, *const list = first + most + 1;
    const int number = a.active[0];
    for (int i = threadIdx.x; i < number; i += blockDim.x) active[i] = a.active[1 + i];
    for (int i = threadIdx.x; i <= number; i += blockDim.x) first[i] = a.first[i];
    for (int i = threadIdx.x; i < slots; i += blockDim.x) list[i] = a.slots[i];
    for (int i = threadIdx.x; i < waves * a.tokens * 4 * NT; i += blockDim.x) sums[i] = f4zero();
    __syncthreads();
    const int blocks = a.hidden_pad / 128, items = number * blocks;  // at most 2^10 * 2^7
    const int workers = waves * gridDim.y, worker = blockIdx.y * waves + wave;
    const int begin = (int)((long long)items * worker / workers), end = (int)((long long)items * (worker + 1) / workers);
    int row[NT];
#pragma unroll
    for (int f = 0; f < NT; f++) row[f] = min(d0 + f * 16 + col, a.dim - 1);

    // Where the wave is: block kb of up to `to` of expert `at`, for its slots from s0 on.
    struct Cursor {
        int at, kb, from, to, s0;
    };
    auto enter = [&](int n) {
        Cursor c{n, 0, max(begin - n * blocks, 0), min(end - n * blocks, blocks), 0};
        c.kb = c.from;
        return c;
    };
    auto after = [&](Cursor c) {  // past the end: to <= from
        if (c.kb + 1 < c.to) c.kb++;
        else if (c.s0 + 16 * CT < __builtin_amdgcn_readfirstlane(first[c.at + 1] - first[c.at])) c.s0 += 16 * CT, c.kb = c.from;
        else if ((c.at + 1) * blocks < end) c = enter(c.at + 1);
        else c.to = c.from;
        return c;
    };
    auto load = [&](Piece<FORMAT>(&w)[NT], const Cursor& c) {
        const int e = __builtin_amdgcn_readfirstlane(active[c.at]);
#pragma unroll
        for (int f = 0; f < NT; f++)
            w[f].load(row_of<FORMAT>(a.w2, e, a.dim, a.hidden_pad, row[f]),
                      scales_of<FORMAT>(a.s2, e, a.dim, a.hidden_pad, row[f], a.scale_shift), c.kb, quad);
    };
    f4 own[NT][CT];
    int slot[CT];
    const __bf16* act[CT];
    auto start = [&](const Cursor& c) {
        const int f0 = first[c.at], count = first[c.at + 1] - f0;
#pragma unroll
        for (int j = 0; j < CT; j++) {
            const int i = c.s0 + j * 16 + col;
            slot[j] = i < count ? list[f0 + i] : -1;
            act[j] = a.acts + (long long)(slot[j] >= 0 ? slot[j] : list[f0]) * A * a.hidden_pad + quad * 32;
#pragma unroll
            for (int f = 0; f < NT; f++) own[f][j] = f4zero();
        }
    };
    auto finish_run = [&] {
#pragma unroll
        for (int j = 0; j < CT; j++) {
            if (slot[j] < 0) continue;
            const float w = a.weights[slot[j]];
            f4* to = sums + (wave * a.tokens + slot[j] / a.topk) * 4 * NT + quad;
#pragma unroll
            for (int f = 0; f < NT; f++) {
                f4 v = to[f * 4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = fmaf(w, own[f][j][i], v[i]);
                to[f * 4] = v;
            }
        }
    };
    auto work = [&](const Piece<FORMAT>(&w)[NT], int kb) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            bf16x8 t[CT][A];
#pragma unroll
            for (int j = 0; j < CT; j++)
#pragma unroll
                for (int u = 0; u < A; u++)
                    t[j][u] = *reinterpret_cast<const bf16x8*>(act[j] + (long long)u * a.hidden_pad + kb * 128 + q * 8);
#pragma unroll
            for (int f = 0; f < NT; f++) {
                const bf16x8 b = w[f](q);
#pragma unroll
                for (int j = 0; j < CT; j++)
#pragma unroll
                    for (int u = 0; u < A; u++)
                        own[f][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, t[j][u], own[f][j], 0, 0, 0);
            }
        }
    };
    if (begin < end) {
        Cursor c = enter(begin / blocks);
        Piece<FORMAT> w0[NT], w1[NT];
        load(w0, c);
        start(c);
        auto step = [&](Piece<FORMAT>(&w)[NT], Piece<FORMAT>(&ahead)[NT]) {
            const Cursor d = after(c);
            const bool more = d.to > d.from;
            if (more) load(ahead, d);
            work(w, c.kb);
            if (!more || d.at != c.at || d.s0 != c.s0) {
                finish_run();
                if (more) start(d);
            }
            c = d;
            return more;
        };
        while (step(w0, w1) && step(w1, w0)) {}
    }
    __syncthreads();
    // Of token t, columns d .. d + 3.
    auto store = [&](int t, int d, f4 v) {
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
    };
    const int pieces = a.tokens * 4 * NT;
    const long long plane = (long long)gridDim.x * pieces;
    f4* const parts = reinterpret_cast<f4*>(a.parts) + (long long)blockIdx.x * pieces;
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
        f4 v = sums[i];
        for (int w = 1; w < waves; w++) v += sums[w * pieces + i];
        if (gridDim.y == 1) store(i / (4 * NT), d0 + i % (4 * NT) * 4, v);
        else parts[blockIdx.y * plane + i] = v;
    }
    if (gridDim.y == 1) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(a.out_tickets + blockIdx.x, 1u) == gridDim.y - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
        f4 v = parts[i];
        for (unsigned p = 1; p < gridDim.y; p++) v += parts[p * plane + i];
        store(i / (4 * NT), d0 + i % (4 * NT) * 4, v);
    }
}

// What a call launches, by its sizes.
struct LayerPlan {
    bool many;       // several slots an expert
    int hidden_waves, out_tiles, out_parts, out_waves;
};

LayerPlan layer_plan(const LayerArgs& a)
{
    LayerPlan p{};
    const int slots = a.tokens * a.topk, experts = std::min(a.experts, slots);
    p.many = slots >= 4 * experts;
    p.hidden_waves = std::min(kLayerWaves, a.dim_pad / 128);
    const int nt = p.many ? 2 : 1, items = experts * (a.hidden_pad / 128);
    p.out_tiles = (a.dim + 16 * nt - 1) / (16 * nt);
    p.out_waves = std::min(kLayerWaves, items);
    p.out_parts = std::max(1, std::min((2 * num_cus() + p.out_tiles - 1) / p.out_tiles, items / (4 * kLayerWaves)));
    return p;
}

// More dynamic LDS than any kernel may have has to be asked for.
void allow_lds(const void* kernel, size_t lds)
{
    if (lds > 64 * 1024) GRAFT_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
}

template <int FORMAT, class T, int G, int NT, int CT>
void hidden_launch(const LayerArgs& a, const LayerPlan& p, hipStream_t s)
{
    const unsigned most = (unsigned)std::min(a.experts, a.tokens * a.topk);
    layer_hidden_kernel<FORMAT, T, G, NT, CT><<<dim3(a.hidden_pad / (16 * NT), most), p.hidden_waves * 64, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

template <int FORMAT, class T, int NT, int CT>
void out_launch(const LayerArgs& a, const LayerPlan& p, hipStream_t s)
{
    const int slots = a.tokens * a.topk, most = std::min(a.experts, slots);
    const size_t lds = (size_t)p.out_waves * a.tokens * 64 * NT + (size_t)(2 * most + 1 + slots) * 4;
    allow_lds((const void*)layer_out_kernel<FORMAT, T, NT, CT>, lds);
    layer_out_kernel<FORMAT, T, NT, CT><<<dim3(p.out_tiles, p.out_parts), p.out_waves * 64, lds, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

template <class T, class R, int MT>
void route_launch(const LayerArgs& a, hipStream_t s)
{
    const size_t scores = (size_t)kRouteWaves * a.experts * 4 * (a.groups > 1 ? 2 : 1);
    const size_t lds = std::max({(size_t)kRouteWaves * MT * 1024, scores, (size_t)(a.experts + a.tokens * a.topk) * 4});
    allow_lds((const void*)layer_route_kernel<T, R, MT>, lds);
    layer_route_kernel<T, R, MT><<<(a.experts + 15) / 16, kRouteThreads, lds, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

template <int FORMAT, class T>
void products(const LayerArgs& a, const LayerPlan& p, hipStream_t s)
{
    if (p.many) {
        if (a.gated) hidden_launch<FORMAT, T, 2, 2, 2>(a, p, s);
        else hidden_launch<FORMAT, T, 1, 4, 2>(a, p, s);
        out_launch<FORMAT, T, 2, 2>(a, p, s);
    } else {
        if (a.gated) hidden_launch<FORMAT, T, 2, 1, 1>(a, p, s);
        else hidden_launch<FORMAT, T, 1, 1, 1>(a, p, s);
        out_launch<FORMAT, T, 1, 1>(a, p, s);
    }
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
    a.groups = o.route.numGroups;
    a.kept = o.route.topGroups;
    a.group_best = o.route.groupScore;
    a.scale = o.route.scale;
    a.sigmoid = o.route.scoreType == ROUTE_SIGMOID;
    a.renorm = o.route.renormalize != 0;
    a.gated = o.gated != 0;
    const int bytes = data_bytes(o.dataType);
    a.vec_x = aligned16(t.x) && o.strideX * bytes % 16 == 0;
    a.vec_router = aligned16(t.router) && (long long)o.dim * data_bytes(o.routerType) % 16 == 0;
    a.vec_out = aligned16(out) && o.strideOut * bytes % 16 == 0;
    a.scale_shift = o.scaleRows == 128 ? 7 : 0;
    a.dim_pad = round_up(o.dim, 128);
    a.hidden_pad = round_up(o.hidden, 128);
    const LayerPlan p = layer_plan(a);
    const int slots = tokens * a.topk, most = std::min(a.experts, slots);
    size_t size = 0;
    auto take = [&](size_t n) {
        const size_t at = size;
        size += round_up<size_t>(n, 256);
        return at;
    };
    const size_t x_terms = o.dataType == DATA_F32 ? 3 : o.dataType == DATA_BF16 ? 1 : 2, a_terms = o.dataType == DATA_F32 ? 3 : 2;
    const size_t at_logits = take((size_t)tokens * a.experts * 4), at_weights = take((size_t)slots * 4);
    const size_t at_active = take((size_t)(most + 1) * 4), at_first = take((size_t)(most + 1) * 4), at_slots = take((size_t)slots * 4);
    const size_t at_xs = take((size_t)tokens * x_terms * a.dim_pad * 2), at_acts = take((size_t)slots * a_terms * a.hidden_pad * 2);
    const bool split = p.out_parts > 1;
    const size_t at_parts = take(split ? (size_t)p.out_parts * p.out_tiles * tokens * (p.many ? 32 : 16) * 4 : 0);
    const size_t at_tickets = take(split ? (size_t)(o.dim + 15) / 16 * 4 : 0);
    a.route_ticket = stream_tickets(s);
    char* ws = (char*)stream_workspace(s).get(size);
    a.logits = (float*)(ws + at_logits);
    a.weights = (float*)(ws + at_weights);
    a.active = (int*)(ws + at_active);
    a.first = (int*)(ws + at_first);
    a.slots = (int*)(ws + at_slots);
    a.xs = (__bf16*)(ws + at_xs);
    a.acts = (__bf16*)(ws + at_acts);
    if (split) {
        a.parts = (float*)(ws + at_parts);
        a.out_tickets = (uint32_t*)(ws + at_tickets);
    }
    with_type(o.dataType, [&](auto x) {
        using T = decltype(x);
        with_type(o.routerType, [&](auto r) {
            if (tokens <= 16) route_launch<T, decltype(r), 1>(a, s);
            else route_launch<T, decltype(r), 4>(a, s);
        });
        if (o.weightFormat == EXPERT_FP8) products<EXPERT_FP8, T>(a, p, s);
        else products<EXPERT_FP4, T>(a, p, s);
    });
}

}  // namespace graft
