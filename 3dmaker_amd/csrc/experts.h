// Internal interface of the mixture-of-experts operators (route.hip,
// fp8_quant.hip, fp8_product.hip, fp4_quant.hip, fp4_product.hip,
// expert_rows.hip, expert_layer.hip, norm_gate.hip); the options are those of
// experts_abi.h.  Every function checks its arguments before its first device call
// and throws std::runtime_error.
#pragma once

#include "common.h"
#include "experts_abi.h"

#include <algorithm>

namespace graft {

template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

// Tokens and rows of a call: 32-bit indices have room for a workgroup's rows
// behind the last.
constexpr int kMaxRows = 1 << 30;

inline int data_bytes(int type) { return type == DATA_F32 ? 4 : 2; }

inline void require(bool ok, const char* what)
{
    if (!ok) throw std::runtime_error(what);
}

inline void require_type(int type)
{
    require(type == DATA_F32 || type == DATA_F16 || type == DATA_BF16, "unknown data type");
}

// f(T{}) with the C++ type of a DATA_* type.
template <class F>
void with_type(int type, F&& f)
{
    if (type == DATA_F32) f(float{});
    else if (type == DATA_F16) f((_Float16)0);
    else f((__bf16)0.0f);
}

// f(first, number) over `wgs` workgroups in launches of less than 2^32 threads,
// which is what a grid can have: a larger one wraps without an error.
template <class F>
void in_launches(long long wgs, int threads, F&& f)
{
    const long long most = 0xffffffffll / threads;
    for (long long first = 0; first < wgs; first += most) {
        f(first, (unsigned)std::min(most, wgs - first));
        GRAFT_LAUNCH_CHECK();
    }
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <class I>
constexpr I round_up(I n, I m)
{
    return (n + m - 1) / m * m;
}

// Pitches of an 8-bit matrix of `cols` columns: bytes of a row, scales of a row.
constexpr int fp8_pitch(int cols) { return round_up(cols, 128); }
constexpr int fp8_scale_pitch(int cols) { return round_up(fp8_pitch(cols) / 128, 4); }

// The same of a 4-bit matrix.
constexpr int fp4_pitch(int cols) { return round_up(cols, 128) / 2; }
constexpr int fp4_scale_pitch(int cols) { return round_up(cols, 128) / 32; }

// What route_experts requires of its option.
void check_route_option(const RouteOption& o);
void route_experts(const RouteOption& o, const void* logits, long long stride, const float* bias, int* indices,
                   float* weights, int tokens, hipStream_t s);
void route_experts_backward(const RouteOption& o, const void* logits, long long stride, const int* indices,
                            const float* dweights, void* dlogits, long long dstride, int tokens, hipStream_t s);
long long route_plan_capacity(int tokens, int topK, int experts, int align);
void route_plan(const int* indices, int tokens, int topK, int experts, int align, int capacity, int* offsets, int* order,
                int* position, hipStream_t s);

void fp8_quantize(const Fp8QuantOption& o, const void* src, const int* order, const float* weights, const void* gate,
                  uint8_t* q, uint8_t* scales, uint8_t* qt, uint8_t* scalesT, hipStream_t s);
void fp8_product(const Fp8ProductOption& o, const uint8_t* a, const uint8_t* a_scales, const uint8_t* b,
                 const uint8_t* b_scales, const int* offsets, void* out, hipStream_t s);

void fp4_quantize(const Fp4QuantOption& o, const void* src, const int* order, uint8_t* q, uint8_t* scales, hipStream_t s);
void fp4_product(const Fp4ProductOption& o, const uint8_t* a, const uint8_t* a_scales, const uint8_t* b,
                 const uint8_t* b_scales, const int* offsets, void* out, hipStream_t s);

void expert_combine(int dim, int type, const void* rows, int num_rows, long long row_stride, const int* position,
                    const float* weights, void* out, long long out_stride, int tokens, int topK, hipStream_t s);
void expert_combine_backward(int dim, int type, const void* rows, int num_rows, long long row_stride, const int* position,
                             const void* dout, long long dout_stride, float* dweights, int tokens, int topK,
                             hipStream_t s);

struct ExpertLayerTensors {
    const void *x, *router;
    const float* bias;
    const uint8_t *w1, *w1_scales, *w2, *w2_scales;
};
void expert_layer(const ExpertLayerOption& o, const ExpertLayerTensors& t, void* out, int tokens, hipStream_t s);

struct NormGateTensors {
    const void *x, *f, *gate;
    const float *post_w, *post_b, *pre_w, *pre_b;
};
void norm_gate(const NormGateOption& o, const NormGateTensors& t, void* y, void* h, int rows, hipStream_t s);

struct NormGateGrads {
    void *dx, *df, *dgate;
    float *dpost_w, *dpost_b, *dpre_w, *dpre_b;
};
void norm_gate_backward(const NormGateOption& o, const NormGateTensors& t, const void* dy, const void* dh,
                        const NormGateGrads& g, int rows, hipStream_t s);

}  // namespace graft
