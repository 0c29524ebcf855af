// The whole layer of experts for few tokens, for gfx950:
//   z = x R^T;  (e_j, w_j) = route(z);  a_j = act(W1_{e_j} x) [* (U1_{e_j} x)];
//   y = sum_j w_j W2_{e_j} a_j
// Bound by the weights' bytes: each selected expert's matrices are read once, for
// all tokens that take it.  Weights are widened to bf16 with their scales, which is
// exact, and go to v_mfma_f32_16x16x32_bf16 as 16 rows by 32 of k; an expert's slots
// (a token's place for it) are its 16 columns, few or many, at the same cost.  Tokens
// and a_j are split into as many bf16 terms as they need (16-bit tokens are exact in
// one or two, fp32 ones in three; a_j has two, 17 bits, or three, all of fp32),
// so that nothing is rounded to 8 bits on the way.
//
// Three launches: routing (the last workgroup to have its logits ready routes all
// tokens), the hidden activations, the outputs; one more to gather tokens where experts
// have many slots each.
//
// Measured, us for routing, hidden activations, outputs: 7 bf16 tokens, top 6 of 64,
// gated 2048 x 1024 fp4: 9, 20.5, 16.7 (107 MB of weights at 2.3 TB/s in all); 27
// tokens, top 8 of 128, gated 2048 x 768 fp8: 16, 52, 34 (498 MB, 5.8 TB/s in the
// products); 64 fp32 tokens, top 2 of 8, 4096 x 2048 fp8: 14 and 5 for the gathering,
// 31, 29 (134 MB: there the three terms of values, five times the weights' bytes from
// the L2, and registers for two waves a SIMD bound it).
#include "product.h"
#include "route_math.h"

#include <algorithm>
#include <type_traits>

namespace graft {

namespace {

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
    bool sigmoid, renorm, gated, fp4, vec_x, vec_router, vec_out;
    int scale_shift;          // rows of a scale, as a shift
    int dim_pad, hidden_pad;  // filled up to whole blocks of 128
    // scratch
    float *logits, *weights;  // [parts][tokens][experts], [slots]
    int* active;              // number of experts that some token takes, and which
    int *first, *slots;       // where their slots begin in the list of slots, and its end
    __bf16 *xs, *acts;        // [tokens][terms][dim_pad], [slots][terms][hidden_pad] or fragments
    __bf16* frags;            // [fragments][dim_pad / 128][4][64][8]
    float* sums;              // [parts][tiles][tokens][columns of a tile], of more than one part
    uint32_t *route_ticket, *out_tickets;
    int out_tiles;
};

template <class T>
struct Terms {
    static constexpr int kX = sizeof(T) == 4 ? 3 : std::is_same_v<T, __bf16> ? 1 : 2;  // of a token or a router's row
};

// Of a hidden activation, A below: two under 16-bit tokens, three under fp32 ones and on
// request (us with two and with three: 27 tokens, top 8 of 128, gated 2048 x 768 fp8 107
// and 115; 64, top 2 of 8, gated 2048 x 1024 fp8 37.7 and 40.4; 7, top 6 of 64, fp4 45
// and 46).
constexpr int a_terms_of(bool f32) { return f32 ? 3 : 2; }

// v as N bf16 numbers, each what is nearest to what those before it leave, which is
// exact: two keep 17 bits of v, three all of an fp32 number.  Where rounding would
// give an infinity for a finite v, the first is cut.  An infinity is the first alone,
// a NaN also the last.  Not SAFE: infinities, and what rounds to them, become NaN.
template <bool SAFE = true, int N>
__device__ __forceinline__ void split(float v, __bf16 (&t)[N])
{
#pragma unroll
    for (int i = 0; i < N - 1; i++) {
        float near = (float)(__bf16)v;
        if (SAFE && i == 0 && __builtin_isinf(near)) near = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u);
        t[i] = (__bf16)near;
        v = SAFE && i == 0 && __builtin_isinf(near) ? 0.0f : v - near;
    }
    t[N - 1] = (__bf16)v;
}

// Where eight consecutive k, k % 8 == 0, of a block of 128 stand among a token's terms
// or a slot's activations: the order in which the lanes load them beside the weights,
// so that a load of 16 rows takes 64 consecutive bytes of each.  Lane quarter `quad`
// has bytes 16 quad .. 16 quad + 15 of 64 of a row of weights: 16 k of e4m3, 32 of fp4.
__device__ __forceinline__ int place_of(int k, bool fp4)
{
    const int in = k & 127;
    return k - in + (fp4 ? (in / 8 % 4) * 32 + in / 32 * 8 : (in / 64 * 2 + in / 8 % 2) * 32 + in / 16 % 4 * 8);
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

// v but for its infinities, which are zero.
__device__ __forceinline__ bf16x8 finite8(bf16x8 v)
{
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __builtin_isinf((float)v[i]) ? (__bf16)0.0f : v[i];
    return v;
}

template <bool SAFE, class T, int N = Terms<T>::kX>
__device__ __forceinline__ void split8(const T (&v)[8], bf16x8 (&t)[N])
{
#pragma unroll
    for (int i = 0; i < 8; i++) {
        __bf16 s[N];
        if constexpr (N == 1) s[0] = v[i];
        else split<SAFE>((float)v[i], s);
#pragma unroll
        for (int u = 0; u < N; u++) t[u][i] = s[u];
    }
}

// What workgroups of a launch leave for the last of them goes past the L2, which the
// XCDs do not share, word by word as atomics of the device's scope.  A release fence,
// which writes back all of an L2, took 256 workgroups 11 us and 512 of them 21.
__device__ __forceinline__ void store_past(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float load_past(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Whether the workgroup is the last of `number` to come here.  Its stores have been
// made by then: the memory counter says when they are.
__device__ __forceinline__ bool is_last(uint32_t* ticket, uint32_t number, bool* shared)
{
    __builtin_amdgcn_s_waitcnt(kCopiesDone);
    __syncthreads();
    if (threadIdx.x == 0) *shared = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == number - 1;
    __syncthreads();
    return *shared;
}

// ---------------------------------------------------------------------------
// routing
// ---------------------------------------------------------------------------

// Tokens by LANES lanes of a wave, lane l of them with experts PER l .. PER l + PER - 1,
// so that lane order is index order.  Logits are in LDS or the sum of `parts` in
// memory; scores, and with groups keys, are LDS for PER experts of each thread, and
// group_keys of one.  Bound by instructions: some 400 a wave and round, on one CU.
template <int LANES, int PER>
__device__ __forceinline__ void route_tokens(const LayerArgs& a, const float* logits, int parts, float* lds, int* expert)
{
    const int threads = blockDim.x, lane = threadIdx.x & 63, sub = lane & (LANES - 1), local = threadIdx.x / LANES;
    const int first = sub * PER, n = a.experts - first, size = a.experts / a.groups;
    const uint64_t lanes = (LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1)) << (lane - sub);  // the token's
    float* const scores = lds + local * (LANES * PER);
    uint32_t* const keys = reinterpret_cast<uint32_t*>(lds) + (threads + local * LANES) * PER;
    uint32_t* const group_keys = reinterpret_cast<uint32_t*>(lds) + 2 * threads * PER + local * LANES;
    float bias[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) bias[i] = a.bias && i < n ? a.bias[first + i] : 0.0f;
    for (int t0 = 0; t0 < a.tokens; t0 += threads / LANES) {
        const int t = min(t0 + local, a.tokens - 1);  // behind the last token: that once more
        float s[PER];
        uint32_t key[PER];
        if (logits) {
#pragma unroll
            for (int i = 0; i < PER; i++) s[i] = i < n ? logits[t * a.experts + first + i] : -INFINITY;
        } else {
            const float* z = a.logits + (long long)t * a.experts + first;
#pragma unroll
            for (int i = 0; i < PER; i++) s[i] = i < n ? load_past(z + i) : -INFINITY;
            for (int p = 1; p < parts; p++) {
                z += (long long)a.tokens * a.experts;
#pragma unroll
                for (int i = 0; i < PER; i++) s[i] += i < n ? load_past(z + i) : 0.0f;
            }
        }
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            s[i] = s[i] > -INFINITY ? fminf(s[i], 3.402823466e38f) : -INFINITY;  // NaN: none
            top = fmaxf(top, s[i]);
        }
        if (!a.sigmoid) top = lanes_max<LANES>(top);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool live = s[i] > -INFINITY;
            const float e = exp_neg(a.sigmoid ? -fabsf(s[i]) : s[i] - top), r = __builtin_amdgcn_rcpf(1.0f + e);
            key[i] = live;
            s[i] = !live ? 0.0f : !a.sigmoid ? e : s[i] >= 0.0f ? r : e * r;
            sum += s[i];
        }
        if (!a.sigmoid) {
            sum = lanes_sum<LANES>(sum);
            const float r = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
            for (int i = 0; i < PER; i++) s[i] *= r;
        }
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const float c = s[i] + bias[i];
            key[i] = key[i] && c > -INFINITY ? key_of(c) : 0u;
            if (i < n) scores[first + i] = s[i];
        }
        if (a.groups > 1) {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (i < n) keys[first + i] = key[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            uint32_t g = 0;  // lane l: group l, by the best one or two of it
            if (sub < a.groups) {
                uint32_t b2 = 0;
#pragma unroll 8
                for (int i = 0; i < size; i++) {
                    const uint32_t k = keys[sub * size + i];
                    b2 = max(b2, min(g, k));
                    g = max(g, k);
                }
                if (a.group_best == 2 && b2 != 0) g = key_of(of_key(g) + of_key(b2));
                group_keys[sub] = g;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            int ahead = 0;
#pragma unroll 4
            for (int o = 0; o < a.groups; o++) {
                const uint32_t k = group_keys[o];
                ahead += k > g || (k == g && o < sub);
            }
            const uint64_t kept = __ballot(sub < a.groups && ahead < a.kept) >> (lane - sub);
            const float r = 1.0f / (float)size;
#pragma unroll
            for (int i = 0; i < PER; i++)  // of at most 1,024 experts: the quotient's error is far below 1 / 2 size
                if (i < n && !(kept >> (int)(((float)(first + i) + 0.5f) * r) & 1)) key[i] = 0;
        }
#pragma unroll 1
        for (int j = 0; j < a.topk; j++) {
            uint32_t best = key[0];
#pragma unroll
            for (int i = 1; i < PER; i++) best = max(best, key[i]);
            const uint32_t all = lanes_umax<LANES>(best);
            const uint64_t have = __ballot(best == all) & lanes;
            const bool mine = lane == __ffsll((unsigned long long)have) - 1;  // the lowest
            int at = 0;
#pragma unroll
            for (int i = PER - 1; i >= 0; i--) at = key[i] == all ? i : at;
#pragma unroll
            for (int i = 0; i < PER; i++) key[i] = mine && i == at ? 0u : key[i];
            if (mine) expert[t * a.topk + j] = all ? first + at : -1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int e = sub < a.topk ? expert[t * a.topk + sub] : -1;  // topk is at most LANES
        float score = e >= 0 ? scores[e] : 0.0f, factor = a.scale;
        if (a.renorm) factor /= lanes_sum<LANES>(score) + 1e-20f;
        if (sub < a.topk) a.weights[t * a.topk + sub] = score * factor;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// f(lanes of a token, experts of a lane): as many tokens a wave as leave a lane at most
// four experts (or 16, of more than 256) and a lane for each group and pick.
template <class F>
__host__ __device__ inline void with_lanes(const LayerArgs& a, F&& f)
{
    using std::integral_constant;
    const int per_group_or_pick = a.groups > a.topk ? a.groups : a.topk;
    if (a.experts <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (a.experts <= 64 && per_group_or_pick <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    else if (a.experts <= 128 && per_group_or_pick <= 32) f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
    else if (a.experts <= 256) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

// The experts that some token takes, in their order, and the list of their slots,
// from the slots' experts and count [experts] in LDS.
__device__ __forceinline__ void plan(const LayerArgs& a, const int* expert, int* count)
{
    const int slots = a.tokens * a.topk;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) count[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += blockDim.x)
        if (expert[i] >= 0) atomicAdd(&count[expert[i]], 1);
    __syncthreads();
    if (threadIdx.x < 64) {  // count: where the expert's next slot goes
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
    for (int i = threadIdx.x; i < slots; i += blockDim.x)
        if (expert[i] >= 0) a.slots[atomicAdd(&count[expert[i]], 1)] = i;
}

// LDS of the routing kernel: sums of its waves, then scores and keys, then the plan's
// counts, in one place; the slots' experts; the logits, if there is room for them: they
// are read token by token if not.
constexpr int kLdsBytes = 160 * 1024 - 64;  // with what the kernel declares itself
struct RouteLds {
    int experts_at, logits_at, size;
    bool logits;
};
__host__ __device__ inline RouteLds route_lds(const LayerArgs& a, int waves, int tiles)
{
    int scores = 0;
    with_lanes(a, [&](auto, auto P) { scores = waves * 64 * 4 * (a.groups > 1 ? 2 * decltype(P)::value + 1 : decltype(P)::value); });
    const int sums = waves * tiles * 1024, counts = a.experts * 4;
    RouteLds l;
    l.experts_at = sums > scores ? sums : scores;
    if (counts > l.experts_at) l.experts_at = counts;
    l.logits_at = l.experts_at + a.tokens * a.topk * 4;
    l.logits = l.logits_at + a.tokens * a.experts * 4 <= kLdsBytes;
    l.size = l.logits_at + (l.logits ? a.tokens * a.experts * 4 : 0);
    return l;
}

// Logits of 16 experts over a part of k that the waves share out; the tokens' terms on
// the way; routing and plan by the workgroup that is last.  Products of terms are
// exact; a second term is at most 2^-8 of its number and a third 2^-17, so that the
// products that are left out come to 2^-24 of the whole one at most, of either sign.
// Bound by round trips.  A
// part is two blocks of k, a quarter of one for each of eight waves, while that makes
// no more than 128 workgroups, so that reading and splitting tokens is spread (64 fp32
// tokens of 4096 by 8 experts: 14.2 us, 19.9 with four blocks, 13.0 with one; 27 of
// 2048 by 128: 15.6, 16.5 and 17.3).
template <class T, class R, int MT>
__global__ __launch_bounds__(kRouteThreads) void layer_route_kernel(LayerArgs a)
{
    constexpr int X = Terms<T>::kX, Y = Terms<R>::kX;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ bool last;
    f4* const sums = reinterpret_cast<f4*>(lds);  // [waves][MT][64]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int col = lane & 15, quad = lane >> 4, e0 = blockIdx.x * 16;
    const int blocks = a.dim_pad / 128, parts = gridDim.y;
    const int kb0 = blocks * blockIdx.y / parts, kb1 = blocks * (blockIdx.y + 1) / parts;
    const bool alone = gridDim.x * parts == 1;
    const RouteLds at = route_lds(a, waves, MT);
    int* const expert = reinterpret_cast<int*>(lds + at.experts_at);
    const int all = a.tokens * a.experts;
    float* const logits = at.logits ? reinterpret_cast<float*>(lds + at.logits_at) : nullptr;
    f4 acc[MT];
    const R* r = (const R*)a.router + (long long)min(e0 + col, a.experts - 1) * a.dim;
#pragma unroll
    for (int j = 0; j < MT; j++) acc[j] = f4zero();
    auto load_x = [&](T(&w)[8], int j, int k) {
        load8(w, (const T*)a.x + min(j * 16 + col, a.tokens - 1) * a.stride_x + k, a.dim - k, a.vec_x);
    };
    auto store_x = [&](const bf16x8(&x)[X], int j, int k) {  // each workgroup of a part stores some blocks of the terms
        const int t = j * 16 + col;
        if (k / 128 % gridDim.x != blockIdx.x || t >= a.tokens) return;
#pragma unroll
        for (int m = 0; m < X; m++) *reinterpret_cast<bf16x8*>(a.xs + ((long long)t * X + m) * a.dim_pad + place_of(k, a.fp4)) = x[m];
    };
    for (int u = 4 * kb0 + wave; u < 4 * kb1; u += waves) {  // a quarter of a block at a time
        const int k = u / 4 * 128 + quad * 32 + u % 4 * 8;
        R v[8];
        bf16x8 y[Y];
        load8(v, r + k, a.dim - k, a.vec_router);
        T w[MT][8];
#pragma unroll
        for (int j = 0; j < MT; j++)
            if (j * 16 < a.tokens) load_x(w[j], j, k);
        split8<false>(v, y);
#pragma unroll
        for (int j = 0; j < MT; j++) {
            if (j * 16 >= a.tokens) break;
            bf16x8 x[X];
            split8<false>(w[j], x);
#pragma unroll
            for (int m = 0; m < X; m++)
#pragma unroll
                for (int n = 0; n < Y; n++)
                    if (m + n < 3) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[n], x[m], acc[j], 0, 0, 0);
            store_x(x, j, k);
        }
    }
    // An infinity has become a NaN, which it would also with the other operand's second
    // term where that is zero or of the other sign.  Where there is a NaN all of it again,
    // infinities as first terms, which meet the other operand's first term alone.
    if constexpr (X * Y > 1) {
        float any = 0.0f;
#pragma unroll
        for (int j = 0; j < MT; j++) any += (acc[j][0] + acc[j][1]) + (acc[j][2] + acc[j][3]);
        const bool again = __any(__builtin_isnan(any));
#pragma unroll
        for (int j = 0; j < MT; j++) {
            if (!again || j * 16 >= a.tokens) break;
            acc[j] = f4zero();
#pragma unroll 1
            for (int u = 4 * kb0 + wave; u < 4 * kb1; u += waves) {
                const int k = u / 4 * 128 + quad * 32 + u % 4 * 8;
                R v[8];
                T w[8];
                bf16x8 x[X], y[Y];
                load8(v, r + k, a.dim - k, a.vec_router);
                load_x(w, j, k);
                split8<true>(v, y);
                split8<true>(w, x);
                const bf16x8 first_x = finite8(x[0]), first_y = finite8(y[0]);
#pragma unroll
                for (int m = 0; m < X; m++)
#pragma unroll
                    for (int n = 0; n < Y; n++)
                        if (m + n < 3)
                            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n == 0 && m > 0 ? first_y : y[n],
                                                                             m == 0 && n > 0 ? first_x : x[m], acc[j], 0, 0, 0);
                store_x(x, j, k);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MT; j++) sums[(wave * MT + j) * 64 + lane] = acc[j];
    __syncthreads();
    for (int j = wave; j * 16 < a.tokens; j += waves) {
        f4 v = sums[j * 64 + lane];
        for (int w = 1; w < min(waves, 4 * (kb1 - kb0)); w++) v += sums[(w * MT + j) * 64 + lane];
        const int t = j * 16 + col;
        if (t < a.tokens) {
            float* to = alone ? logits : a.logits + (long long)blockIdx.y * all;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = e0 + quad * 4 + i;
                if (e >= a.experts) continue;
                if (alone) to[t * a.experts + e] = v[i];
                else store_past(to + t * a.experts + e, v[i]);
            }
        }
    }
    if (alone) __syncthreads();
    else {
        if (!is_last(a.route_ticket, gridDim.x * parts, &last)) return;
        if (threadIdx.x == 0) *a.route_ticket = 0;
        if (logits) {  // all parts' loads together
            for (int i0 = threadIdx.x; i0 < all; i0 += 4 * blockDim.x) {
                float v[4] = {};
                for (int p0 = 0; p0 < parts; p0 += 8) {
                    float z[4][8];
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int p = 0; p < 8; p++)
                            z[u][p] = load_past(a.logits + min(p0 + p, parts - 1) * all + min(i0 + u * (int)blockDim.x, all - 1));
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int p = 0; p < 8; p++) v[u] += p0 + p < parts ? z[u][p] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (i0 + u * (int)blockDim.x < all) logits[i0 + u * blockDim.x] = v[u];
            }
            __syncthreads();
        }
    }
    if (a.out_tickets)
        for (int i = threadIdx.x; i < a.out_tiles; i += blockDim.x) a.out_tickets[i] = 0;
    with_lanes(a, [&](auto L, auto P) {
        route_tokens<decltype(L)::value, decltype(P)::value>(a, logits, parts, reinterpret_cast<float*>(lds), expert);
    });
    __syncthreads();
    plan(a, expert, reinterpret_cast<int*>(lds));
}

// ---------------------------------------------------------------------------
// the experts' products
// ---------------------------------------------------------------------------

// A wave's copies of weights: 16 rows by 64 bytes each, four consecutive lanes a row, so
// that the vector memory unit takes 16 cycles for them.  A load in the order of the
// matrix instruction, whose consecutive lanes have rows of their own, takes it 64,
// which bounded these kernels (7 tokens, top 6 of 64, 2048 x 1024 fp4: 26 and 19 us
// for hidden activations and outputs, 20.6 and 16.9 this way; 27 tokens, top 8 of 128,
// 2048 x 768 fp8: 55 and 40, 52 and 35).  Piece p of row r goes to place p ^ key(r) of
// the row's four: a quarter of a 16-byte read from LDS then meets each bank once.
constexpr int kCopyBytes = 1024;
__device__ __forceinline__ int copy_key(int row) { return -(row >> 2) & 3; }

// A lane's 32 of the 128 k of a row, from the copies of a block; eight to a matrix
// instruction: which eight is place_of's order.
template <int FORMAT>
struct Piece;

template <>
struct Piece<EXPERT_FP8> {
    static constexpr int kCopies = 2;
    i4v v[2];
    __device__ __forceinline__ void read(const uint8_t* lds, int at)
    {
        v[0] = *reinterpret_cast<const i4v*>(lds + at);
        v[1] = *reinterpret_cast<const i4v*>(lds + at + kCopyBytes);
    }
    static __device__ __forceinline__ int four_scales(const uint8_t* scales, int kb) { return *(const int*)(scales + (kb & ~3)); }
    static __device__ __forceinline__ int shift(int kb, int) { return 8 * (kb & 3); }
    __device__ __forceinline__ bf16x8 operator()(int q, int byte) const
    {
        return widen(v[q >> 1][2 * (q & 1)], v[q >> 1][2 * (q & 1) + 1], scale_of(byte));
    }
};

template <>
struct Piece<EXPERT_FP4> {
    static constexpr int kCopies = 1;
    i4v v;
    __device__ __forceinline__ void read(const uint8_t* lds, int at) { v = *reinterpret_cast<const i4v*>(lds + at); }
    static __device__ __forceinline__ int four_scales(const uint8_t* scales, int kb) { return *(const int*)(scales + kb * 4); }
    static __device__ __forceinline__ int shift(int, int quad) { return 8 * quad; }
    __device__ __forceinline__ bf16x8 operator()(int q, int byte) const
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

#ifdef __HIP_DEVICE_COMPILE__  // the host pass does not know the type
// Rows of weights, with zeros behind them; the same for all lanes.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t weights_from(const uint8_t* p, int bytes)
{
    const uint64_t at = (uint64_t)p;
    const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t)at), high = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)high << 32 | low), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}
#endif

__device__ __forceinline__ float activate(int kind, float v)
{
    switch (kind) {
        case EXPERT_RELU: return v < 0.0f ? 0.0f : v;  // NaN stays
        case EXPERT_SILU: return v / (1.0f + expf(-v));
        case EXPERT_GELU: return 0.5f * v * (1.0f + erff(v * 0.707106781f));
        default: return v;
    }
}

// The 16 columns of a matrix instruction are SLOTS slots by TERMS terms, one term of
// all slots behind the other: a value's terms are products of their own, added up at
// the end.
template <int TERMS>
struct Columns {
    static constexpr int kSlots = 16 / TERMS;
    int slot, term;
    __device__ __forceinline__ explicit Columns(int col)
    {
        term = col / kSlots;
        slot = term < TERMS ? col - term * kSlots : kSlots;  // none behind the last term's
    }
};

// 128 of k of a wave's CT fragments of tokens or hidden activations, from where the
// lane's are: 32 elements to a row of STEP.  With one fragment they are in rows; with
// several, which cost more than the weights, as fragments: the lanes' pieces of 16
// bytes one behind the other, 1 KB to a load.
template <int CT>
struct Values {
    static constexpr int kStep = CT == 1 ? 32 : 512, kBlock = 4 * kStep;  // to the next load's, to the next block's
    bf16x8 t[CT][4];
    __device__ __forceinline__ void load(const __bf16* const (&from)[CT], int kb)
    {
#pragma unroll
        for (int j = 0; j < CT; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) t[j][q] = *reinterpret_cast<const bf16x8*>(from[j] + (long long)kb * kBlock + q * kStep);
    }
};

// Fragments of an expert's slots, the n-th active one's, whose slots begin at `first`:
// the first fragment's number.  No two experts' meet: the sum of ceil(c / SLOTS) over
// the first n of them is less than first / SLOTS + n.
template <int SLOTS>
__device__ __forceinline__ int fragment_of(int first, int n) { return first / SLOTS + n; }

// The blocks of a wave, one under way ahead of the one that is worked on, in two
// places: first(place), then load(place) and work(place) while more() says so, and
// end(place).  What is under way is the same on every path to a wait: where loads
// depend on a condition, the compiler has the wait for the older block wait for them.
template <class More, class First, class Load, class Work, class End>
__device__ __forceinline__ void in_two_places(More&& more, First&& first, Load&& load, Work&& work, End&& end)
{
    const std::integral_constant<int, 0> a;
    const std::integral_constant<int, 1> b;
    first(a);
    while (true) {
        if (!more()) {
            end(a);
            return;
        }
        load(b);
        work(a);
        if (!more()) {
            end(b);
            return;
        }
        load(a);
        work(b);
    }
}

// The scales of F fragments of weights, four bytes at a time.  They are loaded behind
// the copies of those: when they are there, so are the copies.
template <int FORMAT, int F>
struct Scales {
    int four[F];
    __device__ __forceinline__ void load(const uint8_t* const (&from)[F], int kb)
    {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int f = 0; f < F; f++) four[f] = Piece<FORMAT>::four_scales(from[f], kb);
    }
    __device__ __forceinline__ void arrive()
    {
#pragma unroll
        for (int f = 0; f < F; f++) asm volatile("" : "+v"(four[f])::"memory");
    }
};

// lds: the copies of the block, those of a fragment behind the other's; at: the lane's
// place in a copy; shift: to its scale.
template <int FORMAT, int F, int CT>
__device__ __forceinline__ void multiply(f4 (&acc)[F][CT], const uint8_t* lds, int at, const Scales<FORMAT, F>& s, int shift,
                                         const Values<CT>& v)
{
    Piece<FORMAT> w[F];
#pragma unroll
    for (int f = 0; f < F; f++) w[f].read(lds + f * (Piece<FORMAT>::kCopies * kCopyBytes), at);
#pragma unroll
    for (int u = 0; u < 4 * F; u++) {  // with few fragments of values the weights' in turn, so that sums wait less for each other
        const int f = CT > 1 ? u / 4 : u % F, q = CT > 1 ? u % 4 : u / F;
        const bf16x8 b = w[f](q, s.four[f] >> shift & 255);
#pragma unroll
        for (int j = 0; j < CT; j++) acc[f][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, v.t[j][q], acc[f][j], 0, 0, 0);
    }
}

// Tokens' terms as fragments, block by block.
template <class T>
__global__ __launch_bounds__(256) void layer_gather_kernel(LayerArgs a)
{
    constexpr int X = Terms<T>::kX, kSlots = Columns<X>::kSlots;
    const int n = blockIdx.y, kb = blockIdx.x, lane = threadIdx.x & 63, q = threadIdx.x >> 6;
    if (n >= a.active[0]) return;
    const int first = a.first[n], count = a.first[n + 1] - first;
    const Columns<X> mine(lane & 15);
    __bf16* to = a.frags + ((long long)fragment_of<kSlots>(first, n) * gridDim.x + kb) * 2048 + threadIdx.x * 8;
    for (int s0 = 0; s0 < count; s0 += kSlots, to += gridDim.x * 2048) {
        if (mine.slot >= kSlots || s0 + mine.slot >= count) continue;
        const int token = a.slots[first + s0 + mine.slot] / a.topk;
        *reinterpret_cast<bf16x8*>(to) = *reinterpret_cast<const bf16x8*>(
            a.xs + ((long long)token * X + mine.term) * a.dim_pad + kb * 128 + q * 32 + (lane >> 4) * 8);
    }
}

// The hidden activations of 16 NT rows (with their gate's: G 2) for the slots of an
// active expert, as many at a time as CT fragments have: waves share out k, and their
// sums are joined in LDS in wave order.  A lane whose column has no slot works on the
// first one's for nothing.  Bound by the weights' trips from memory, of which many
// waves a CU have more under way than few that look far ahead: four waves with two
// blocks in LDS took 20.6 us where four blocks took 22.7 and six 25.2 (7 tokens, top 6
// of 64, 2048 x 1024 fp4), 52.2, 68.8 and 98 (27 tokens, top 8 of 128, 2048 x 768 fp8).
constexpr int kHiddenWaves = 4;

template <int FORMAT, class T, int A, int G, int NT, int CT>
__global__ __launch_bounds__(kHiddenWaves * 64, CT == 4 ? 2 : CT == 2 ? 3 : 4) void layer_hidden_kernel(LayerArgs a)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host pass needs the kernel's name alone
    constexpr int WAVES = kHiddenWaves;
    constexpr int X = Terms<T>::kX, F = G * NT, kSlots = Columns<X>::kSlots;
    constexpr int kCopies = Piece<FORMAT>::kCopies, kBlock = F * kCopies * kCopyBytes;
    constexpr int kSums = WAVES * F * CT * 1024, kRings = WAVES * 2 * kBlock;
    // One array: with two, the compiler waits for all copies before each LDS read.
    __shared__ __attribute__((aligned(128))) uint8_t lds[kSums > kRings ? kSums : kRings];
    f4(*const sums)[F][CT][64] = reinterpret_cast<f4(*)[F][CT][64]>(lds);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4, n0 = blockIdx.x * 16 * NT, n = blockIdx.y;
    // one round trip for all four; behind the active experts they are of no use
    const int number = a.active[0], at_e = a.active[1 + n], at_first = a.first[n], at_end = a.first[n + 1];
    if (n >= __builtin_amdgcn_readfirstlane(number)) return;
    const int e = __builtin_amdgcn_readfirstlane(at_e), first = __builtin_amdgcn_readfirstlane(at_first);
    const int count = __builtin_amdgcn_readfirstlane(at_end) - first;
    uint8_t* const ring = lds + wave * 2 * kBlock;
    const int pitch = (int)pitch_of<FORMAT>(a.dim_pad), rows = min(16 * NT, max(a.hidden - n0, 0));
    const uint32_t from = (lane >> 2) * pitch + ((lane & 3) ^ copy_key(lane >> 2)) * 16, at = col * 64 + (quad ^ copy_key(col)) * 16;
    const uint8_t* const w = row_of<FORMAT>(a.w1, e, G * a.hidden, a.dim_pad, min(n0, a.hidden));
    const __amdgpu_buffer_rsrc_t w0 = weights_from(w, rows * pitch), w1 = weights_from(w + (G - 1) * (long long)a.hidden * pitch, rows * pitch);
    const uint8_t* S[F];
#pragma unroll
    for (int f = 0; f < F; f++) {
        const int row = min(n0 + f % NT * 16 + col, a.hidden - 1) + f / NT * a.hidden;
        S[f] = scales_of<FORMAT>(a.s1, e, G * a.hidden, a.dim_pad, row, a.scale_shift);
    }
    const int blocks = a.dim_pad / 128;
    const Columns<X> mine(col);
    for (int s0 = 0; s0 < count; s0 += kSlots * CT) {
        int slot = 0;  // of rows
        const __bf16* x[CT];
        f4 acc[F][CT];
#pragma unroll
        for (int j = 0; j < CT; j++) {
            if (CT == 1) {
                const bool there = mine.slot < kSlots && s0 + mine.slot < count;
                slot = a.slots[first + (there ? s0 + mine.slot : 0)];
                x[j] = a.xs + ((long long)(slot / a.topk) * X + (there ? mine.term : 0)) * a.dim_pad + quad * 8;
            } else {
                const int j1 = min(j, (count - s0 - 1) / kSlots);  // behind the last fragment: that once more
                x[j] = a.frags + (long long)(fragment_of<kSlots>(first, n) + s0 / kSlots + j1) * blocks * 2048 + lane * 8;
            }
#pragma unroll
            for (int f = 0; f < F; f++) acc[f][j] = f4zero();
        }
        // Four fragments of values leave no registers for those of two blocks.
        constexpr bool kOne = CT == 4;
        Scales<FORMAT, F> scales[2];
        Values<CT> v[kOne ? 1 : 2];
        if (wave < blocks) {
            int ahead = wave, now = wave;
            auto weights = [&](auto D) {
                constexpr int d = decltype(D)::value;
                __builtin_amdgcn_s_waitcnt(kLdsDone);  // reads of the place that is copied to
#pragma unroll
                for (int f = 0; f < F; f++)
#pragma unroll
                    for (int h = 0; h < kCopies; h++)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(
                            f < NT ? w0 : w1, (__attribute__((address_space(3))) void*)(ring + d * kBlock + (f * kCopies + h) * kCopyBytes),
                            16, from + f % NT * 16 * pitch + (ahead * kCopies + h) * 64, 0, 0, 0);
                scales[d].load(S, ahead);
                ahead += WAVES;
            };
            auto work = [&](auto D) {
                constexpr int d = decltype(D)::value;
                scales[d].arrive();
                multiply(acc, ring + d * kBlock, at, scales[d], Piece<FORMAT>::shift(now, quad), v[kOne ? 0 : d]);
                if (kOne) __builtin_amdgcn_sched_barrier(0);  // the next values' loads stay behind: they have these' registers
                now += WAVES;
            };
            in_two_places(
                [&] { return ahead < blocks; },
                [&](auto D) {
                    if (!kOne) v[0].load(x, ahead);
                    weights(D);
                },
                [&](auto D) {
                    if (kOne) v[0].load(x, now);
                    else v[decltype(D)::value].load(x, ahead);
                    weights(D);
                },
                work,
                [&](auto D) {
                    if (kOne) v[0].load(x, now);
                    work(D);
                });
        }
        __syncthreads();  // sums take the rings' place
#pragma unroll
        for (int f = 0; f < F; f++)
#pragma unroll
            for (int j = 0; j < CT; j++) sums[wave][f][j][lane] = acc[f][j];
        __syncthreads();
        const int joined = min(WAVES, blocks);
        for (int c = wave; c < NT * CT; c += WAVES) {
            const int f = c / CT, j = c % CT, i = s0 + j * kSlots + mine.slot;
            if (mine.slot >= kSlots || i >= count || mine.term > 0) continue;
            f4 h[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                h[g] = f4zero();
                for (int u = 0; u < X; u++)
                    for (int w = 0; w < joined; w++) h[g] += sums[w][g * NT + f][j][lane + u * kSlots];
            }
            const int row = n0 + f * 16 + quad * 4;
            Vec<__bf16, 4> o[A];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float v = activate(a.activation, h[0][r]);
                if (G == 2) v *= h[G - 1][r];
                if (row + r >= a.hidden) v = 0.0f;
                __bf16 s[A];
                split(v, s);
#pragma unroll
                for (int t = 0; t < A; t++) o[t][r] = s[t];
            }
            const int k = place_of(row & ~7, FORMAT == EXPERT_FP4);
            constexpr int kOut = Columns<A>::kSlots;
            __bf16* const to = CT == 1 ? a.acts + (long long)slot * A * a.hidden_pad + k + (row & 4)
                                       : a.acts + (long long)(fragment_of<kOut>(first, n) + i / kOut) * a.hidden_pad * 16 +
                                             k / 32 * 512 + (k / 8 % 4 * 16 + i % kOut) * 8 + (row & 4);
#pragma unroll
            for (int t = 0; t < A; t++) *reinterpret_cast<Vec<__bf16, 4>*>(to + (CT == 1 ? (long long)t * a.hidden_pad : t * kOut * 8)) = o[t];
        }
        if (s0 + kSlots * CT < count) __syncthreads();
    }
#endif
}

// 16 NT columns of the outputs for all tokens and a part of the active experts' k, which
// its waves share out in runs of one expert's.  Their sums go, weighted, to the
// tokens' in the wave's part of LDS; those are joined in wave order, and the parts in
// their order by the workgroup of a tile that is last.  Bound as the hidden activations'
// kernel is: 16.7 us for 36 MB, 34 for 166 MB (4.9 TB/s).
constexpr int kOutWaves = 8;

template <int FORMAT, class T, int A, int NT, int CT>
__global__ __launch_bounds__(kOutWaves * 64) void layer_out_kernel(LayerArgs a)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host pass needs the kernel's name alone
    constexpr int WAVES = kOutWaves, kSlots = Columns<A>::kSlots;
    constexpr int kCopies = Piece<FORMAT>::kCopies, kBlock = NT * kCopies * kCopyBytes;
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4, d0 = blockIdx.x * 16 * NT;
    const int slots = a.tokens * a.topk, most = min(a.experts, slots);
    uint8_t* const ring = lds + wave * 2 * kBlock;
    f4* const sums = reinterpret_cast<f4*>(lds + WAVES * 2 * kBlock);  // [waves][tokens][4 NT]
    int* const active = reinterpret_cast<int*>(sums + WAVES * a.tokens * 4 * NT);
    int *const first = active + most, *const list = first + most + 1;
    float* const weights = reinterpret_cast<float*>(list + slots);  // in LDS as well: a load would wait for all that are ahead
    const int number = a.active[0];
    for (int i = threadIdx.x; i < most; i += WAVES * 64) active[i] = a.active[1 + i];
    for (int i = threadIdx.x; i <= most; i += WAVES * 64) first[i] = a.first[i];
    for (int i = threadIdx.x; i < slots; i += WAVES * 64) list[i] = a.slots[i], weights[i] = a.weights[i];
    for (int i = threadIdx.x; i < WAVES * a.tokens * 4 * NT; i += WAVES * 64) sums[i] = f4zero();
    __syncthreads();
    const int blocks = a.hidden_pad / 128, items = number * blocks;  // at most 2^10 * 2^7
    const int workers = WAVES * gridDim.y, worker = blockIdx.y * WAVES + wave;
    const int begin = (int)((long long)items * worker / workers), end = (int)((long long)items * (worker + 1) / workers);
    int row[NT];
#pragma unroll
    for (int f = 0; f < NT; f++) row[f] = min(d0 + f * 16 + col, a.dim - 1);
    const int pitch = (int)pitch_of<FORMAT>(a.hidden_pad), rows = min(16 * NT, a.dim - d0);
    const uint32_t copy_from = (lane >> 2) * pitch + ((lane & 3) ^ copy_key(lane >> 2)) * 16;
    const int at = col * 64 + (quad ^ copy_key(col)) * 16;
    const Columns<A> mine(col);

    // Block kb, from .. to - 1, of expert `at`, for its slots from s0 on.
    struct Cursor {
        int at, kb, from, to, s0;
        __device__ __forceinline__ bool valid() const { return kb < to; }
        __device__ __forceinline__ bool first_of_run() const { return kb == from; }
        __device__ __forceinline__ bool last_of_run() const { return kb + 1 == to; }
    };
    auto enter = [&](int n) {
        const int from = max(begin - n * blocks, 0);
        return Cursor{n, from, from, min(end - n * blocks, blocks), 0};
    };
    auto advance = [&](Cursor& c) {
        if (++c.kb < c.to) return;
        if (c.s0 + kSlots * CT < __builtin_amdgcn_readfirstlane(first[c.at + 1] - first[c.at])) {
            c.s0 += kSlots * CT;
            c.kb = c.from;
        } else if ((c.at + 1) * blocks < end) c = enter(c.at + 1);
    };
    auto slot_of = [&](const Cursor& c, int j) {  // of the lane's column, -1: none
        const int f0 = first[c.at], i = c.s0 + j * kSlots + mine.slot;
        return mine.slot < kSlots && i < first[c.at + 1] - f0 ? list[f0 + i] : -1;
    };
    Scales<FORMAT, NT> scales[2];
    __amdgpu_buffer_rsrc_t W;
    const uint8_t* S[NT];
    const __bf16* act[CT];
    auto load_weights = [&](int d, Scales<FORMAT, NT>& to, const Cursor& c) {
        if (c.first_of_run()) {
            const int e = __builtin_amdgcn_readfirstlane(active[c.at]);
            W = weights_from(row_of<FORMAT>(a.w2, e, a.dim, a.hidden_pad, d0), rows * pitch);
#pragma unroll
            for (int f = 0; f < NT; f++) S[f] = scales_of<FORMAT>(a.s2, e, a.dim, a.hidden_pad, row[f], a.scale_shift);
        }
#pragma unroll
        for (int f = 0; f < NT; f++)
#pragma unroll
            for (int h = 0; h < kCopies; h++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    W, (__attribute__((address_space(3))) void*)(ring + d * kBlock + (f * kCopies + h) * kCopyBytes), 16,
                    copy_from + f * 16 * pitch + (c.kb * kCopies + h) * 64, 0, 0, 0);
        to.load(S, c.kb);
    };
    auto load_values = [&](Values<CT>& v, const Cursor& c) {
        if (c.first_of_run()) {
#pragma unroll
            for (int j = 0; j < CT; j++) {
                if (CT == 1) {
                    const int slot = slot_of(c, j);
                    act[j] = a.acts + ((long long)(slot >= 0 ? slot : list[first[c.at]]) * A + (slot >= 0 ? mine.term : 0)) * a.hidden_pad +
                             quad * 8;
                } else {
                    const int f0 = __builtin_amdgcn_readfirstlane(first[c.at]), n = __builtin_amdgcn_readfirstlane(first[c.at + 1]) - f0;
                    const int j1 = min(j, (n - c.s0 - 1) / kSlots);  // behind the last fragment: that once more
                    act[j] = a.acts + (long long)(fragment_of<kSlots>(f0, c.at) + c.s0 / kSlots + j1) * a.hidden_pad * 16 + lane * 8;
                }
            }
        }
        v.load(act, c.kb);
    };
    f4 own[NT][CT];
    auto finish_run = [&](const Cursor& c) {
#pragma unroll
        for (int j = 0; j < CT; j++) {
            const int slot = slot_of(c, j);
            const bool takes = slot >= 0 && mine.term == 0;
            const float w = weights[max(slot, 0)];
            f4* to = sums + (wave * a.tokens + max(slot, 0) / a.topk) * 4 * NT + quad;
#pragma unroll
            for (int f = 0; f < NT; f++) {
                f4 v = own[f][j];
#pragma unroll
                for (int i = 0; i < 4; i++) {  // the other terms, kSlots lanes on
                    const float x = own[f][j][i];
                    const uint32_t u = __builtin_bit_cast(uint32_t, x);
                    if constexpr (A == 2) v[i] += __builtin_bit_cast(float, dpp_mov<0x108>(u));
                    if constexpr (A == 3)
                        v[i] += __builtin_bit_cast(float, dpp_mov<0x105>(u)) + __builtin_bit_cast(float, dpp_mov<0x10a>(u));
                }
                if (!takes) continue;
                f4 sum = to[f * 4];
#pragma unroll
                for (int i = 0; i < 4; i++) sum[i] = fmaf(w, v[i], sum[i]);
                to[f * 4] = sum;
            }
        }
    };
    if (begin < end) {
        Values<CT> v[2];
        Cursor ahead = enter(begin / blocks), now = ahead;
        auto load = [&](auto D) {
            constexpr int d = decltype(D)::value;
            __builtin_amdgcn_s_waitcnt(kLdsDone);  // reads of the place that is copied to
            load_values(v[d], ahead);
            load_weights(d, scales[d], ahead);
            advance(ahead);
        };
        auto work = [&](auto D) {
            constexpr int d = decltype(D)::value;
            if (now.first_of_run()) {
#pragma unroll
                for (int j = 0; j < CT; j++)
#pragma unroll
                    for (int f = 0; f < NT; f++) own[f][j] = f4zero();
            }
            scales[d].arrive();
            multiply(own, ring + d * kBlock, at, scales[d], Piece<FORMAT>::shift(now.kb, quad), v[d]);
            if (now.last_of_run()) finish_run(now);
            advance(now);
        };
        in_two_places([&] { return ahead.valid(); }, load, load, work, work);
    }
    // Zero already, unless calls that share the counter ran at once, against the rules:
    // then at least the stream's next one finds it so.
    if (blockIdx.x + blockIdx.y + threadIdx.x == 0) *a.route_ticket = 0;
    __syncthreads();
    const int pieces = a.tokens * 4 * NT;
    auto store = [&](int i, f4 v) {
        const int t = i / (4 * NT), d = d0 + i % (4 * NT) * 4;
        T* to = (T*)a.out + t * a.stride_out + d;
        if (a.vec_out && d + 4 <= a.dim) {
            Vec<T, 4> o;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = (T)v[j];
            *reinterpret_cast<Vec<T, 4>*>(to) = o;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (d + j < a.dim) to[j] = (T)v[j];
        }
    };
    const long long plane = (long long)gridDim.x * pieces * 4;
    float* const parts = a.sums + (long long)blockIdx.x * pieces * 4;
    for (int i = threadIdx.x; i < pieces; i += WAVES * 64) {
        f4 v = sums[i];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v += sums[w * pieces + i];
        if (gridDim.y == 1) store(i, v);
        else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                store_past(parts + blockIdx.y * plane + i * 4 + j, v[j]);
        }
    }
    if (gridDim.y == 1 || !is_last(a.out_tickets + blockIdx.x, gridDim.y, reinterpret_cast<bool*>(lds))) return;  // a ring's place
    for (int i = threadIdx.x; i < pieces; i += WAVES * 64) {
        f4 v = f4zero();
        for (unsigned p = 0; p < gridDim.y; p++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                v[j] += load_past(parts + p * plane + i * 4 + j);
        store(i, v);
    }
#endif
}

// What a call launches, by its sizes.
struct LayerPlan {
    int route_parts, route_waves;
    bool many;  // several slots an expert
    int out_tiles, out_parts;
};

LayerPlan layer_plan(const LayerArgs& a)
{
    LayerPlan p{};
    const int slots = a.tokens * a.topk, blocks = a.dim_pad / 128, groups = (a.experts + 15) / 16;
    p.route_parts = std::max(1, std::min({blocks / 2, 128 / groups, 32}));
    p.route_waves = std::min(kRouteWaves, std::max(4 * ((blocks + p.route_parts - 1) / p.route_parts), a.tokens));
    const int most = std::min(a.experts, slots);
    // Fragments cost a launch and the gathering, and pay where experts have many slots (64
    // tokens, top 2, gated 2048 x 1024 fp8, us as fragments and as rows: 8 slots an expert
    // fp32 tokens 63 and 70, bf16 51 and 49, with fp4 weights 42 and 45; 16 slots 50 and 61,
    // 37 and 38, 36 and 41; 4 slots 87 and 80, 72 and 61, 64 and 56).
    p.many = slots >= 8 * most;
    p.out_tiles = (a.dim + (p.many ? 31 : 15)) / (p.many ? 32 : 16);
    // A workgroup a CU, each wave with four blocks of k at least.  More parts cost more to
    // join than they help (7 tokens of 64 experts, top 6, 2048 x 1024: 19.1 us in two
    // parts, 20.1 in four, 23.6 in eight, 28 in one).
    p.out_parts = std::max(1, std::min((num_cus() + p.out_tiles - 1) / p.out_tiles, most * (a.hidden_pad / 128) / 32));
    return p;
}

// More dynamic LDS than any kernel may have has to be asked for.  The limit is the
// kernel's, not the call's: all ask for the same, so that none lowers what another
// thread's launch, or a captured one, needs.
void allow_lds(const void* kernel, size_t lds)
{
    if (lds > 64 * 1024) GRAFT_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes));
}

template <int FORMAT, class T, int A, int G, int NT, int CT>
void hidden_launch(const LayerArgs& a, hipStream_t s)
{
    const unsigned most = (unsigned)std::min(a.experts, a.tokens * a.topk);
    layer_hidden_kernel<FORMAT, T, A, G, NT, CT><<<dim3(a.hidden_pad / (16 * NT), most), kHiddenWaves * 64, 0, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

template <int FORMAT, class T, int A, int NT, int CT>
void out_launch(const LayerArgs& a, const LayerPlan& p, hipStream_t s)
{
    const int slots = a.tokens * a.topk, most = std::min(a.experts, slots);
    const size_t lds = kOutWaves * ((size_t)2 * NT * Piece<FORMAT>::kCopies * kCopyBytes + (size_t)a.tokens * 64 * NT) +
                       (size_t)(2 * most + 1 + 2 * slots) * 4;
    allow_lds((const void*)layer_out_kernel<FORMAT, T, A, NT, CT>, lds);
    layer_out_kernel<FORMAT, T, A, NT, CT><<<dim3(p.out_tiles, p.out_parts), kOutWaves * 64, lds, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

template <class T, class R, int MT>
void route_launch(const LayerArgs& a, const LayerPlan& p, hipStream_t s)
{
    const unsigned groups = (a.experts + 15) / 16;
    const size_t lds = route_lds(a, p.route_waves, MT).size;
    allow_lds((const void*)layer_route_kernel<T, R, MT>, lds);
    layer_route_kernel<T, R, MT><<<dim3(groups, p.route_parts), p.route_waves * 64, lds, s>>>(a);
    GRAFT_LAUNCH_CHECK();
}

template <int FORMAT, class T, int A>
void products(const LayerArgs& a, const LayerPlan& p, hipStream_t s)
{
    constexpr int CT = Terms<T>::kX == 3 ? 4 : 2;  // fragments: 20 slots of three terms, 16 or 32 of fewer
    if (p.many) {
        layer_gather_kernel<T><<<dim3(a.dim_pad / 128, std::min(a.experts, a.tokens * a.topk)), 256, 0, s>>>(a);
        GRAFT_LAUNCH_CHECK();
        if (a.gated) hidden_launch<FORMAT, T, A, 2, 1, CT>(a, s);
        else hidden_launch<FORMAT, T, A, 1, 2, CT>(a, s);
        out_launch<FORMAT, T, A, 2, A == 3 ? 4 : 2>(a, p, s);
    } else {
        if (a.gated) hidden_launch<FORMAT, T, A, 2, 1, 1>(a, s);
        else hidden_launch<FORMAT, T, A, 1, 1, 1>(a, s);
        out_launch<FORMAT, T, A, 1, 1>(a, p, s);
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
    const int type = o.dataType & ~EXPERT_HIDDEN_F32;
    const bool hidden_f32 = type == DATA_F32 || (o.dataType & EXPERT_HIDDEN_F32);
    require_type(type);
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
    a.fp4 = o.weightFormat == EXPERT_FP4;
    const int bytes = data_bytes(type);
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
    const size_t x_terms = type == DATA_F32 ? 3 : type == DATA_BF16 ? 1 : 2, a_terms = a_terms_of(hidden_f32);
    const size_t at_logits = take((size_t)p.route_parts * tokens * a.experts * 4), at_weights = take((size_t)slots * 4);
    const size_t at_active = take((size_t)(most + 1) * 4), at_first = take((size_t)(most + 1) * 4), at_slots = take((size_t)slots * 4);
    const size_t at_xs = take((size_t)tokens * x_terms * a.dim_pad * 2);
    auto fragments = [&](size_t terms) { return (size_t)(slots / (16 / terms) + most); };
    const size_t at_acts = take(p.many ? fragments(a_terms) * a.hidden_pad * 32 : (size_t)slots * a_terms * a.hidden_pad * 2);
    const size_t at_frags = take(p.many ? fragments(x_terms) * a.dim_pad * 32 : 0);
    const bool split = p.out_parts > 1;
    const size_t at_sums = take(split ? (size_t)p.out_parts * p.out_tiles * tokens * (p.many ? 32 : 16) * 4 : 0);
    const size_t at_tickets = take(split ? (size_t)p.out_tiles * 4 : 0);
    a.route_ticket = stream_ticket(s);
    char* ws = (char*)stream_workspace(s).get(size);
    a.logits = (float*)(ws + at_logits);
    a.weights = (float*)(ws + at_weights);
    a.active = (int*)(ws + at_active);
    a.first = (int*)(ws + at_first);
    a.slots = (int*)(ws + at_slots);
    a.xs = (__bf16*)(ws + at_xs);
    a.acts = (__bf16*)(ws + at_acts);
    a.frags = (__bf16*)(ws + at_frags);
    if (split) {
        a.sums = (float*)(ws + at_sums);
        a.out_tickets = (uint32_t*)(ws + at_tickets);
        a.out_tiles = p.out_tiles;
    }
    with_type(type, [&](auto x) {
        using T = decltype(x);
        with_type(o.routerType, [&](auto r) {
            if (tokens <= 16) route_launch<T, decltype(r), 1>(a, p, s);
            else route_launch<T, decltype(r), 4>(a, p, s);
        });
        auto of_format = [&](auto f) {
            constexpr int F = decltype(f)::value;
            if constexpr (sizeof(T) == 4) products<F, T, a_terms_of(true)>(a, p, s);
            else if (hidden_f32) products<F, T, a_terms_of(true)>(a, p, s);
            else products<F, T, a_terms_of(false)>(a, p, s);
        };
        if (o.weightFormat == EXPERT_FP8) of_format(std::integral_constant<int, EXPERT_FP8>{});
        else of_format(std::integral_constant<int, EXPERT_FP4>{});
    });
}

}  // namespace graft
