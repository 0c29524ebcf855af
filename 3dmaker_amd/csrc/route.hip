// Routing of tokens to experts and the plan of the experts' rows, for gfx950.
//
//   s = softmax(z) or sigmoid(z),  c = s + b;  the best groups by c, then the
//   k largest c in them, ties to the lowest index;  w = scale s / (sum s + 1e-20)
//
// A token lies on LPT lanes of a wave, every group of experts on LG of them,
// a lane's V experts next to each other, so that lane order is index order: the
// largest key of all lanes by a butterfly, then the lowest lane that has it and
// that lane's first place with it are the lowest index.
#include "experts.h"
#include "route_math.h"

#include <algorithm>
#include <cmath>

namespace graft {

namespace {

constexpr int kRouteThreads = 256;
constexpr int kMaxExperts = 1024;

struct RouteArgs {
    const void* logits;
    long long stride;
    const float* bias;
    int* indices;
    float* weights;
    int tokens, experts, topk, groups, kept, group_size, lanes_group, lanes_group_bits, group_best;
    int type;
    bool sigmoid, renorm, vec;
    float scale;
    int token0;  // the launch's first token
    // backward
    const float* dweights;
    void* dlogits;
    long long dstride;
};

template <class T, int V>
__device__ __forceinline__ void load_v(float (&z)[V], const T* p, int n, bool vec)
{
    if (vec) {
        constexpr int N = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
#pragma unroll
        for (int i = 0; i < V; i += N) {
            const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(p + i);
#pragma unroll
            for (int j = 0; j < N; j++) z[i + j] = (float)v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) z[i] = i < n ? (float)p[i] : 0.0f;
    }
}

// The lane's V logits: experts first .. first + n of the token (others and
// unavailable ones: live bit 0).
template <int V>
__device__ __forceinline__ uint32_t load_logits(float (&z)[V], const RouteArgs& a, int token, int first, int n)
{
    if (n > 0) {
        const long long at = (long long)token * a.stride + first;
        if (a.type == DATA_F32) load_v(z, (const float*)a.logits + at, n, a.vec);
        else if (a.type == DATA_F16) load_v(z, (const _Float16*)a.logits + at, n, a.vec);
        else load_v(z, (const __bf16*)a.logits + at, n, a.vec);
    }
    uint32_t live = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const bool ok = i < n && z[i] > -INFINITY;  // false for NaN
        live |= ok ? 1u << i : 0u;
        z[i] = ok ? fminf(z[i], 3.402823466e38f) : 0.0f;
    }
    return live;
}

// Scores of the lane's experts (0 where not live).
template <int V, int LPT>
__device__ __forceinline__ void scores_of(float (&s)[V], const float (&z)[V], uint32_t live, bool sigmoid)
{
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float t = exp_neg(-fabsf(z[i]));
            const float r = __builtin_amdgcn_rcpf(1.0f + t);
            s[i] = live >> i & 1 ? (z[i] >= 0.0f ? r : t * r) : 0.0f;
        }
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; i++) m = live >> i & 1 ? fmaxf(m, z[i]) : m;
        m = lanes_max<LPT>(m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            s[i] = live >> i & 1 ? exp_neg(z[i] - m) : 0.0f;
            sum += s[i];
        }
        sum = lanes_sum<LPT>(sum);
        const float r = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) s[i] *= r;
    }
}

// The largest key of a token's lanes.  A whole wave's is left in its last lane by
// the row broadcasts (six instructions, against ten for one that all lanes hold)
// and read from there.
template <int LPT>
__device__ __forceinline__ uint32_t largest(uint32_t v)
{
    if constexpr (LPT < 64) return lanes_umax<LPT>(v);
    v = lanes_umax<16>(v);
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x142, 0xa, 0xf, false));  // row_bcast:15
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x143, 0xc, 0xf, false));  // row_bcast:31
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Whether a lane is the lowest of its token's in the wave's mask.
template <int LPT>
__device__ __forceinline__ bool lowest_of(uint64_t mask, int lane)
{
    if constexpr (LPT == 64) return __ffsll((unsigned long long)mask) - 1 == lane;
    const uint64_t below = ((1ull << lane) - 1) & (((1ull << LPT) - 1) << (lane & ~(LPT - 1)));  // the same for all picks
    return (mask & below) == 0;
}

// The best two keys of the LG lanes of a group.
template <int LG>
__device__ __forceinline__ void best_two(uint32_t& b1, uint32_t& b2)
{
    auto join = [&](uint32_t o1, uint32_t o2) {
        b2 = max(min(b1, o1), max(b2, o2));
        b1 = max(b1, o1);
    };
    if constexpr (LG >= 2) join(dpp_mov<0xB1>(b1), dpp_mov<0xB1>(b2));
    if constexpr (LG >= 4) join(dpp_mov<0x4E>(b1), dpp_mov<0x4E>(b2));
    if constexpr (LG >= 8) join(dpp_mov<0x141>(b1), dpp_mov<0x141>(b2));
    if constexpr (LG >= 16) join(dpp_mov<0x140>(b1), dpp_mov<0x140>(b2));
    if constexpr (LG >= 32) join(__shfl_xor(b1, 16), __shfl_xor(b2, 16));
}

// Keys sorted downwards with their places, equal ones in their order.
template <int V>
__device__ __forceinline__ void sort_down(uint32_t (&key)[V], int (&place)[V])
{
#pragma unroll
    for (int end = V - 1; end > 0; end--)
#pragma unroll
        for (int i = 0; i < end; i++) {
            const bool swap = key[i + 1] > key[i];
            const uint32_t hi = max(key[i], key[i + 1]), lo = min(key[i], key[i + 1]);
            const int p = swap ? place[i + 1] : place[i], q = swap ? place[i] : place[i + 1];
            key[i] = hi;
            key[i + 1] = lo;
            place[i] = p;
            place[i + 1] = q;
        }
}

// Four experts a lane are sorted once, and a pick takes the lane's first; more
// are searched at each pick.  A pick's score comes back from LDS at the end.
// Bound by its instructions, about 580 a token of 256 experts and eight picks
// (16,391 of them in 8 groups: 17 us; 262,144 tokens of 8 experts, 32 to a wave:
// 7 us).  Two such tokens a wave, eight experts a lane, took 21 us: the sort grows
// faster than the picks shrink.
template <int V, int LPT>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(RouteArgs a)
{
    constexpr int kTokens = kRouteThreads / LPT;
    constexpr int kPicked = V == 4 ? 1024 : kTokens * 32;  // at most min(LPT V, 32) slots a token
    __shared__ int picked[kPicked];                        // lane of the token * V + its place, or -1
    __shared__ __attribute__((aligned(16))) float score[kRouteThreads * V];
    __shared__ uint32_t group_key[kRouteThreads];
    const int lane = threadIdx.x & 63, sub = threadIdx.x & (LPT - 1), local = threadIdx.x / LPT;
    const int token = a.token0 + (int)blockIdx.x * kTokens + local;
    const int lg = a.lanes_group, lg_bits = a.lanes_group_bits;
    const int group = sub >> lg_bits, in_group = (sub & (lg - 1)) * V;
    const int first = group * a.group_size + in_group;
    const int n = token < a.tokens && group < a.groups ? min(V, a.group_size - in_group) : 0;
    float z[V], s[V];
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = 0.0f;
    uint32_t live = load_logits(z, a, token, first, n);
    float bias[V];
#pragma unroll
    for (int i = 0; i < V; i++) bias[i] = a.bias && i < n ? a.bias[first + i] : 0.0f;
    scores_of<V, LPT>(s, z, live, a.sigmoid);
    uint32_t key[V];
    int place[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float c = s[i] + bias[i];
        key[i] = (live >> i & 1) && c > -INFINITY ? key_of(c) : 0u;
        place[i] = i;
        score[threadIdx.x * V + i] = s[i];
    }
    if (V == 4) sort_down(key, place);
    if (a.groups > 1) {
        uint32_t b1 = key[0], b2 = key[1];  // keys of the best two
        if (V != 4) {
            b2 = min(key[0], key[1]);
            b1 = max(key[0], key[1]);
#pragma unroll
            for (int i = 2; i < V; i++) {
                b2 = max(b2, min(b1, key[i]));
                b1 = max(b1, key[i]);
            }
        }
        switch (lg) {
            case 1: break;
            case 2: best_two<2>(b1, b2); break;
            case 4: best_two<4>(b1, b2); break;
            case 8: best_two<8>(b1, b2); break;
            case 16: best_two<16>(b1, b2); break;
            default: best_two<32>(b1, b2); break;
        }
        uint32_t g = b1;
        if (a.group_best == 2 && b2 != 0) g = key_of(of_key(b1) + of_key(b2));
        if ((sub & (lg - 1)) == 0) group_key[local * LPT + group] = g;
        __syncthreads();
        int ahead = 0;
        for (int o = 0; o < a.groups; o++) {
            const uint32_t k = group_key[local * LPT + o];
            ahead += k > g || (k == g && o < group);
        }
        if (ahead >= a.kept) {
#pragma unroll
            for (int i = 0; i < V; i++) key[i] = 0;
        }
    }
    int* const mine_picked = picked + local * a.topk;
    for (int j = 0; j < a.topk; j++) {
        uint32_t best = key[0];
        if (V != 4) {
#pragma unroll
            for (int i = 1; i < V; i++) best = max(best, key[i]);
        }
        const uint32_t top = largest<LPT>(best);
        const bool mine = best == top && top != 0;
        if (mine && lowest_of<LPT>(__ballot(mine), lane)) {
            int at = place[0];
            if (V == 4) {
#pragma unroll
                for (int i = 0; i + 1 < V; i++) key[i] = key[i + 1], place[i] = place[i + 1];
                key[V - 1] = 0;
            } else {
                at = 0;
#pragma unroll
                for (int i = V - 1; i >= 0; i--) at = key[i] == top ? i : at;
#pragma unroll
                for (int i = 0; i < V; i++) key[i] = i == at ? 0u : key[i];
            }
            mine_picked[j] = sub * V + at;
        } else if (top == 0 && sub == 0) {
            mine_picked[j] = -1;
        }
    }
    __syncthreads();
    float sum = 0.0f;
    for (int j = sub; j < a.topk; j += LPT) {
        const int p = mine_picked[j];
        sum += p >= 0 ? score[local * LPT * V + p] : 0.0f;
    }
    if (a.renorm) sum = lanes_sum<LPT>(sum);
    const float factor = a.renorm ? a.scale / (sum + 1e-20f) : a.scale;
    if (token >= a.tokens) return;
    for (int j = sub; j < a.topk; j += LPT) {
        const int p = mine_picked[j], l = p / V;
        const long long at = (long long)token * a.topk + j;
        a.indices[at] = p >= 0 ? (l >> lg_bits) * a.group_size + (l & (lg - 1)) * V + p % V : -1;
        a.weights[at] = p >= 0 ? score[local * LPT * V + p] * factor : 0.0f;
    }
}

// ds of the selected experts from dw, then the score function's derivative:
//   renorm: ds_i = scale (g_i - sum_j g_j s_j / S) / S, S = sum_j s_j + 1e-20
//   softmax dz = s (ds - sum s ds), sigmoid dz = ds s (1 - s)
// 65,536 x 64 fp32: 11 us, 3.3 TB/s; the scores' exponentials and the three sums
// take as long as the memory.
template <int V, int LPT>
__global__ __launch_bounds__(kRouteThreads) void route_backward_kernel(RouteArgs a)
{
    constexpr int kTokens = kRouteThreads / LPT;
    // The tokens' gradients at their experts' places; kNone (a NaN that no
    // gradient is written as) at those that were not selected.
    constexpr uint32_t kNone = 0xffffffffu;
    __shared__ __attribute__((aligned(16))) uint32_t dense[kRouteThreads * V];
    const int sub = threadIdx.x & (LPT - 1), token0 = a.token0 + (int)blockIdx.x * kTokens, token = token0 + (int)threadIdx.x / LPT;
    const int first = sub * V;
    const int n = token < a.tokens ? max(0, min(V, a.experts - first)) : 0;
#pragma unroll
    for (int i = 0; i < V; i++) dense[threadIdx.x * V + i] = kNone;
    float z[V], s[V], g[V];
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = 0.0f;
    const uint32_t live = load_logits(z, a, token, first, n);
    __syncthreads();
    const long long slot0 = (long long)token0 * a.topk;
    const int slots = min(kTokens, a.tokens - token0) * a.topk;
    for (int i = threadIdx.x; i < slots; i += kRouteThreads) {
        const int e = a.indices[slot0 + i];
        const uint32_t d = __builtin_bit_cast(uint32_t, a.dweights[slot0 + i]);
        if ((unsigned)e < (unsigned)a.experts) dense[i / a.topk * (LPT * V) + e] = d == kNone ? 0x7fc00000u : d;
    }
    __syncthreads();
    scores_of<V, LPT>(s, z, live, a.sigmoid);
    uint32_t chosen = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t d = dense[threadIdx.x * V + i];
        chosen |= d != kNone ? 1u << i : 0u;
        g[i] = __builtin_bit_cast(float, d);
    }
    float total = 0.0f, shift = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) total += chosen >> i & 1 ? s[i] : 0.0f;
    total = lanes_sum<LPT>(total) + 1e-20f;
    const float r = a.renorm ? 1.0f / total : 1.0f;
    if (a.renorm) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            // s / total to the last bit: one expert's weight is 1, its gradient 0
            const float w = s[i] * r;
            shift += chosen >> i & 1 ? g[i] * fmaf(fmaf(-w, total, s[i]), r, w) : 0.0f;
        }
        shift = lanes_sum<LPT>(shift);
    }
    float back = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
        g[i] = chosen >> i & 1 ? a.scale * (g[i] - shift) * r : 0.0f;
        back = fmaf(g[i], s[i], back);
    }
    back = lanes_sum<LPT>(back);
#pragma unroll
    for (int i = 0; i < V; i++) {
        float q = g[i] - back;
        if (a.sigmoid) {
            const float t = exp_neg(-fabsf(z[i]));  // 1 - s without cancellation
            const float rest = __builtin_amdgcn_rcpf(1.0f + t);
            q = g[i] * (z[i] >= 0.0f ? t * rest : rest);
        }
        g[i] = live >> i & 1 ? q * s[i] : 0.0f;
    }
    if (n <= 0) return;
    const long long at = (long long)token * a.dstride + first;
    auto store = [&](auto zero) {
        using T = decltype(zero);
        T* p = (T*)a.dlogits + at;
        if (a.vec) {
            constexpr int N = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;
#pragma unroll
            for (int i = 0; i < V; i += N) {
                Vec<T, N> v;
#pragma unroll
                for (int j = 0; j < N; j++) v[j] = (T)g[i + j];
                *reinterpret_cast<Vec<T, N>*>(p + i) = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < n) p[i] = (T)g[i];
        }
    };
    if (a.type == DATA_F32) store(float{});
    else if (a.type == DATA_F16) store((_Float16)0);
    else store((__bf16)0.0f);
}

int pow2_from(int n)
{
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

// Four experts a lane as long as a wave holds the token, then 8, 16 or 32.
template <class F>
void with_layout(int lanes, int per_lane, F&& f)
{
    using std::integral_constant;
    if (per_lane <= 4) {
        switch (lanes) {
            case 1: f(integral_constant<int, 4>{}, integral_constant<int, 1>{}); break;
            case 2: f(integral_constant<int, 4>{}, integral_constant<int, 2>{}); break;
            case 4: f(integral_constant<int, 4>{}, integral_constant<int, 4>{}); break;
            case 8: f(integral_constant<int, 4>{}, integral_constant<int, 8>{}); break;
            case 16: f(integral_constant<int, 4>{}, integral_constant<int, 16>{}); break;
            case 32: f(integral_constant<int, 4>{}, integral_constant<int, 32>{}); break;
            default: f(integral_constant<int, 4>{}, integral_constant<int, 64>{}); break;
        }
    } else if (per_lane <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 64>{});
    else if (per_lane <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 64>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 64>{});
}

void check_route(const RouteOption& o, const void* logits, long long stride, int tokens)
{
    check_route_option(o);
    require(tokens >= 0 && tokens <= kMaxRows, "numTokens must be 0..2^30");
    require(stride >= o.numExperts, "logitsStride must be at least numExperts");
    require(tokens == 0 || logits, "null argument");
}

RouteArgs route_args(const RouteOption& o, const void* logits, long long stride, int tokens)
{
    RouteArgs a{};
    a.logits = logits;
    a.stride = stride;
    a.tokens = tokens;
    a.experts = o.numExperts;
    a.topk = o.topK;
    a.type = o.logitsType;
    a.sigmoid = o.scoreType == ROUTE_SIGMOID;
    a.renorm = o.renormalize != 0;
    a.scale = o.scale;
    return a;
}

// Whole lanes of V from addresses that their vector loads take.
bool can_vec(const void* p, long long stride, int per_group, int V, int type)
{
    const int bytes = std::min(16, V * data_bytes(type));
    return per_group % V == 0 && (uintptr_t)p % bytes == 0 && stride * data_bytes(type) % bytes == 0;
}

}  // namespace

void check_route_option(const RouteOption& o)
{
    require(o.numExperts >= 1 && o.numExperts <= kMaxExperts, "numExperts must be 1..1024");
    require(o.topK >= 1 && o.topK <= 32 && o.topK <= o.numExperts, "topK must be 1..32 and at most numExperts");
    require(o.scoreType == ROUTE_SOFTMAX || o.scoreType == ROUTE_SIGMOID, "unknown scoreType");
    require(o.numGroups >= 1 && o.numGroups <= 64 && o.numExperts % o.numGroups == 0,
            "numGroups must be 1..64 and divide numExperts");
    require(o.topGroups >= 1 && o.topGroups <= o.numGroups, "topGroups must be 1..numGroups");
    require(o.numGroups == 1 || o.groupScore == 1 || o.groupScore == 2, "groupScore must be 1 or 2");
    require(std::isfinite(o.scale), "scale must be finite");
    require_type(o.logitsType);
}

void route_experts(const RouteOption& o, const void* logits, long long stride, const float* bias, int* indices,
                   float* weights, int tokens, hipStream_t s)
{
    check_route(o, logits, stride, tokens);
    if (tokens == 0) return;
    require(indices && weights, "null argument");
    RouteArgs a = route_args(o, logits, stride, tokens);
    a.bias = bias;
    a.indices = indices;
    a.weights = weights;
    a.groups = o.numGroups;
    a.kept = o.topGroups;
    a.group_size = o.numExperts / o.numGroups;
    a.group_best = o.groupScore;
    const int slots = pow2_from(o.numGroups);
    a.lanes_group = std::min(64 / slots, pow2_from((a.group_size + 3) / 4));
    while ((1 << a.lanes_group_bits) < a.lanes_group) a.lanes_group_bits++;
    const int lanes = slots * a.lanes_group, per_lane = (a.group_size + a.lanes_group - 1) / a.lanes_group;
    with_layout(lanes, per_lane, [&](auto V, auto LPT) {
        a.vec = can_vec(logits, stride, a.group_size, V, a.type);
        constexpr int kPerWg = kRouteThreads / decltype(LPT)::value;
        in_launches((tokens + kPerWg - 1) / kPerWg, kRouteThreads, [&](long long first, unsigned wgs) {
            a.token0 = (int)(first * kPerWg);
            route_kernel<decltype(V)::value, decltype(LPT)::value><<<wgs, kRouteThreads, 0, s>>>(a);
        });
    });
}

void route_experts_backward(const RouteOption& o, const void* logits, long long stride, const int* indices,
                            const float* dweights, void* dlogits, long long dstride, int tokens, hipStream_t s)
{
    check_route(o, logits, stride, tokens);
    require(dstride >= o.numExperts, "dlogitsStride must be at least numExperts");
    if (tokens == 0) return;
    require(indices && dweights && dlogits, "null argument");
    RouteArgs a = route_args(o, logits, stride, tokens);
    a.indices = const_cast<int*>(indices);
    a.dweights = dweights;
    a.dlogits = dlogits;
    a.dstride = dstride;
    const int lanes = std::min(64, pow2_from((o.numExperts + 3) / 4)), per_lane = (o.numExperts + lanes - 1) / lanes;
    with_layout(lanes, per_lane, [&](auto V, auto LPT) {
        a.vec = can_vec(logits, stride, o.numExperts, V, a.type) && can_vec(dlogits, dstride, o.numExperts, V, a.type);
        constexpr int kPerWg = kRouteThreads / decltype(LPT)::value;
        in_launches((tokens + kPerWg - 1) / kPerWg, kRouteThreads, [&](long long first, unsigned wgs) {
            a.token0 = (int)(first * kPerWg);
            route_backward_kernel<decltype(V)::value, decltype(LPT)::value><<<wgs, kRouteThreads, 0, s>>>(a);
        });
    });
}

// ---------------------------------------------------------------------------
// the plan: a stable counting sort of the slots by expert
// ---------------------------------------------------------------------------

namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPlanSmall = 4096;  // slots that one workgroup places alone
constexpr int kPlanRounds = 4, kPlanChunk = kPlanRounds * kPlanThreads;  // of a workgroup otherwise

struct PlanArgs {
    const int* indices;
    int slots, experts, align, capacity, blocks;
    int* offsets;
    int* order;
    int* position;
    int* counts;  // [blocks][experts]: a block's slots of an expert; scanned: those in front of them
    int* totals;  // [experts]: an expert's slots (scanned)
    bool scanned;
};

// A wave's slots of a workgroup's, up to R rounds of 64: their experts (-1: none),
// all loaded before the first is used.
template <int R>
struct PlanSlots {
    int first, rounds;
    int expert[R];

    __device__ __forceinline__ PlanSlots(const PlanArgs& a, int begin, int rounds) : rounds(rounds)
    {
        first = begin + (threadIdx.x >> 6) * (rounds * 64);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int i = first + r * 64 + (threadIdx.x & 63);
            expert[r] = r < rounds && i < a.slots ? a.indices[i] : -1;
        }
#pragma unroll
        for (int r = 0; r < R; r++) expert[r] = (unsigned)expert[r] < (unsigned)a.experts ? expert[r] : -1;
    }
};

// hist [waves][experts]: each wave's slots of an expert.
template <int R>
__device__ __forceinline__ void plan_count(const PlanArgs& a, int* hist, const PlanSlots<R>& slots)
{
    for (int i = threadIdx.x; i < kPlanWaves * a.experts; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    int* const mine = hist + (threadIdx.x >> 6) * a.experts;
#pragma unroll
    for (int r = 0; r < R; r++)
        if (slots.expert[r] >= 0) atomicAdd(&mine[slots.expert[r]], 1);
    __syncthreads();
}

// The wave's slots in order, from next [waves][experts]: rank among the round's
// slots of the same expert from one ballot per bit of the expert's number.
template <int R>
__device__ __forceinline__ void plan_place(const PlanArgs& a, int* next, const PlanSlots<R>& slots, int bits)
{
    const int lane = threadIdx.x & 63;
    int* const mine = next + (threadIdx.x >> 6) * a.experts;
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r >= slots.rounds) continue;
        const int i = slots.first + r * 64 + lane, e = slots.expert[r];
        uint64_t same = __ballot(e >= 0);
        for (int b = 0; b < bits; b++) {
            const uint64_t m = __ballot(e >> b & 1);
            same &= (e >> b & 1) ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        int row = -1;
        if (e >= 0) {
            row = mine[e] + rank;
            a.order[row] = i;
        }
        if (i < a.slots) a.position[i] = row;
        __builtin_amdgcn_wave_barrier();
        if (e >= 0 && rank == 0) mine[e] += __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(PlanArgs a)
{
    extern __shared__ int hist[];
    plan_count(a, hist, PlanSlots<kPlanRounds>(a, blockIdx.x * kPlanChunk, kPlanRounds));
    for (int e = threadIdx.x; e < a.experts; e += kPlanThreads) {
        int n = 0;
        for (int w = 0; w < kPlanWaves; w++) n += hist[w * a.experts + e];
        a.counts[(size_t)blockIdx.x * a.experts + e] = n;
    }
}

// A workgroup: each expert's segment from its slots in LDS (total, overwritten
// with the segment's first row, total[experts] with the rows of all; ends with the
// row behind its last slot), by the first wave.
__device__ __forceinline__ void plan_offsets(const PlanArgs& a, int* total, int* ends, int lane, int wave)
{
    if (wave == 0) {
        int base = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int e = e0 + lane;
            const int own = e < a.experts ? total[e] : 0, n = (own + a.align - 1) / a.align * a.align;
            const int up = lanes_scan(n);
            if (e < a.experts) {
                total[e] = base + up - n;
                ends[e] = base + up - n + own;
            }
            base += __shfl(up, 63);
        }
        if (lane == 0) total[a.experts] = base;
    }
    __syncthreads();
}

// Counts of many blocks, a wave an expert: the slots of the blocks in front of
// each, and of all.
__global__ __launch_bounds__(64) void plan_scan_kernel(PlanArgs a)
{
    const int lane = threadIdx.x;
    int* c = a.counts + blockIdx.x;
    const int per = (a.blocks + 63) / 64, b0 = min(a.blocks, lane * per), b1 = min(a.blocks, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; b++) sum += c[(size_t)b * a.experts];
    const int up = lanes_scan(sum);
    int at = up - sum;
    for (int b = b0; b < b1; b++) {
        const int n = c[(size_t)b * a.experts];
        c[(size_t)b * a.experts] = at;
        at += n;
    }
    if (lane == 63) a.totals[blockIdx.x] = up;
}

// All experts' slots (total) and those in front of `block` (before), by a
// workgroup: from the scan, or added up here.
__device__ __forceinline__ void plan_totals(const PlanArgs& a, int block, int* total, int* before)
{
    for (int e = threadIdx.x; e < a.experts; e += kPlanThreads) {
        total[e] = a.scanned ? a.totals[e] : 0;
        before[e] = a.scanned && block < a.blocks ? a.counts[(size_t)block * a.experts + e] : 0;
    }
    __syncthreads();
    if (a.scanned) return;
    const int shares = max(1, kPlanThreads / a.experts);  // of the blocks, where threads outnumber the experts
    for (int u = threadIdx.x; u < shares * a.experts; u += kPlanThreads) {
        const int e = u % a.experts;
        int all = 0, front = 0;
#pragma unroll 4
        for (int b = u / a.experts; b < a.blocks; b += shares) {
            const int n = a.counts[(size_t)b * a.experts + e];
            all += n;
            front += b < block ? n : 0;
        }
        atomicAdd(&total[e], all);  // whole numbers: any order
        atomicAdd(&before[e], front);
    }
    __syncthreads();
}

// Rows that no slot has: behind the segments' last slots and behind all
// segments, by workgroup `fill` of `fills`.
__device__ __forceinline__ void plan_fill(const PlanArgs& a, const int* starts, const int* ends, int fill, int fills)
{
    if (a.align > 1) {
        constexpr int kWaves = kPlanThreads / 64;
        for (int e = fill * kWaves + threadIdx.x / 64; e < a.experts; e += fills * kWaves)
            for (int r = ends[e] + (threadIdx.x & 63); r < starts[e + 1]; r += 64) a.order[r] = -1;
    }
    for (long long r = starts[a.experts] + (long long)fill * kPlanThreads + threadIdx.x; r < a.capacity;
         r += (long long)fills * kPlanThreads)
        a.order[r] = -1;
}

// The waves' first rows of each expert from their counts; add: what lies in
// front of the workgroup's.
template <class F>
__device__ __forceinline__ void plan_waves(const PlanArgs& a, int* next, F add)
{
    for (int e = threadIdx.x; e < a.experts; e += kPlanThreads) {
        int at = add(e);
        for (int w = 0; w < kPlanWaves; w++) {
            const int n = next[w * a.experts + e];
            next[w * a.experts + e] = at;
            at += n;
        }
    }
    __syncthreads();
}

// Blocks 0 .. blocks - 1 place their slots; those behind them fill the other
// rows.  Every one forms the offsets for itself.  Latency: four rounds of 64
// slots a wave behind the offsets, whose loads are issued ahead of them (5.4 us
// for 131,128 slots of 256 experts, 7.2 with a load in each round; chunks of
// 4,096 slots instead of 1,024 took 15).
__global__ __launch_bounds__(kPlanThreads) void plan_place_kernel(PlanArgs a, int bits)
{
    extern __shared__ int lds[];
    int* next = lds;                            // [waves][experts]
    int* starts = next + kPlanWaves * a.experts;  // [experts + 1]
    int* ends = starts + a.experts + 1;         // [experts]
    int* before = ends + a.experts;             // [experts]
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const PlanSlots<kPlanRounds> slots(a, blockIdx.x * kPlanChunk, kPlanRounds);
    plan_totals(a, blockIdx.x, starts, before);
    plan_offsets(a, starts, ends, lane, wave);
    if ((int)blockIdx.x >= a.blocks) {
        const int fill = blockIdx.x - a.blocks;
        if (fill == 0)
            for (int e = threadIdx.x; e <= a.experts; e += kPlanThreads) a.offsets[e] = starts[e];
        plan_fill(a, starts, ends, fill, gridDim.x - a.blocks);
        return;
    }
    plan_count(a, next, slots);
    plan_waves(a, next, [&](int e) { return starts[e] + before[e]; });
    plan_place(a, next, slots, bits);
}

// Few slots, up to 256 R: one workgroup does all of it.
template <int R>
__global__ __launch_bounds__(kPlanThreads) void plan_small_kernel(PlanArgs a, int bits)
{
    extern __shared__ int lds[];
    int* next = lds;
    int* starts = next + kPlanWaves * a.experts;
    int* ends = starts + a.experts + 1;
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const PlanSlots<R> slots(a, 0, (a.slots + kPlanThreads - 1) / kPlanThreads);
    plan_count(a, next, slots);
    for (int e = threadIdx.x; e < a.experts; e += kPlanThreads) {
        int n = 0;
        for (int w = 0; w < kPlanWaves; w++) n += next[w * a.experts + e];
        starts[e] = n;
    }
    __syncthreads();
    plan_offsets(a, starts, ends, lane, wave);
    for (int e = threadIdx.x; e <= a.experts; e += kPlanThreads) a.offsets[e] = starts[e];
    plan_fill(a, starts, ends, 0, 1);
    plan_waves(a, next, [&](int e) { return starts[e]; });
    plan_place(a, next, slots, bits);
}

}  // namespace

long long route_plan_capacity(int tokens, int topK, int experts, int align)
{
    if (tokens < 0 || tokens > kMaxRows || topK < 1 || topK > 32 || experts < 1 || experts > kMaxExperts || align < 1 || align > 128) return -1;
    const long long slots = (long long)tokens * topK;
    const long long rows = slots + std::min<long long>(experts, slots) * (align - 1);
    const long long capacity = round_up<long long>(rows, align);
    return capacity <= kMaxRows ? capacity : -1;
}

void route_plan(const int* indices, int tokens, int topK, int experts, int align, int capacity, int* offsets, int* order,
                int* position, hipStream_t s)
{
    const long long need = route_plan_capacity(tokens, topK, experts, align);
    require(need >= 0, "numTokens must be >= 0, topK 1..32, numExperts 1..1024, align 1..128, and the rows at most 2^30");
    require(capacity >= need, "capacity is less than routePlanCapacity()");
    require(offsets && (capacity == 0 || order) && (tokens == 0 || (indices && position)), "null argument");
    PlanArgs a{};
    a.indices = indices;
    a.slots = tokens * topK;
    a.experts = experts;
    a.align = align;
    a.capacity = capacity;
    a.offsets = offsets;
    a.order = order;
    a.position = position;
    int bits = 0;
    while ((1 << bits) < experts) bits++;
    const size_t lds = ((kPlanWaves + 3) * experts + 1) * sizeof(int);
    if (a.slots <= kPlanSmall) {
        if (a.slots <= 4 * kPlanThreads) plan_small_kernel<4><<<1, kPlanThreads, lds, s>>>(a, bits);
        else plan_small_kernel<kPlanSmall / kPlanThreads><<<1, kPlanThreads, lds, s>>>(a, bits);
        GRAFT_LAUNCH_CHECK();
        return;
    }
    a.blocks = (a.slots + kPlanChunk - 1) / kPlanChunk;
    Workspace& ws = stream_workspace(s);
    a.counts = (int*)ws.get(((size_t)a.blocks + 1) * experts * sizeof(int));
    a.totals = a.counts + (size_t)a.blocks * experts;
    plan_count_kernel<<<a.blocks, kPlanThreads, kPlanWaves * experts * sizeof(int), s>>>(a);
    GRAFT_LAUNCH_CHECK();
    // Every placing workgroup adds up the counts while they are few, which saves a
    // launch (512 blocks of 8 experts: 11.5 us in two, 13.4 in three; 129 of 256
    // experts: 20 and 14).
    a.scanned = (long long)a.blocks * experts > 1 << 13;
    if (a.scanned) {
        plan_scan_kernel<<<experts, 64, 0, s>>>(a);
        GRAFT_LAUNCH_CHECK();
    }
    plan_place_kernel<<<a.blocks + 64, kPlanThreads, lds, s>>>(a, bits);
    GRAFT_LAUNCH_CHECK();
}

}  // namespace graft
