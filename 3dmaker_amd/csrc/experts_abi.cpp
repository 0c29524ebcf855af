// extern "C" surface of the mixture-of-experts operators (experts_abi.h).
#include "experts_abi.h"

#include "abi_error.h"
#include "experts.h"

using graft::guarded;
using graft::require;

extern "C" {

void launchRouteExperts(const RouteOption* opt, const void* d_logits, long long logitsStride, const float* d_bias,
                        int* d_indices, float* d_weights, int numTokens, hipStream_t stream)
{
    guarded("launchRouteExperts", [&] {
        require(opt, "null option");
        graft::route_experts(*opt, d_logits, logitsStride, d_bias, d_indices, d_weights, numTokens, stream);
    });
}

void launchRouteExpertsBackward(const RouteOption* opt, const void* d_logits, long long logitsStride,
                                const int* d_indices, const float* d_dweights, void* d_dlogits, long long dlogitsStride,
                                int numTokens, hipStream_t stream)
{
    guarded("launchRouteExpertsBackward", [&] {
        require(opt, "null option");
        graft::route_experts_backward(*opt, d_logits, logitsStride, d_indices, d_dweights, d_dlogits, dlogitsStride,
                                      numTokens, stream);
    });
}

long long routePlanCapacity(int numTokens, int topK, int numExperts, int align)
{
    return graft::route_plan_capacity(numTokens, topK, numExperts, align);
}

void launchRoutePlan(const int* d_indices, int numTokens, int topK, int numExperts, int align, int capacity,
                     int* d_offsets, int* d_order, int* d_position, hipStream_t stream)
{
    guarded("launchRoutePlan", [&] {
        graft::route_plan(d_indices, numTokens, topK, numExperts, align, capacity, d_offsets, d_order, d_position,
                          stream);
    });
}

void launchFp8Quantize(const Fp8QuantOption* opt, const void* d_src, const int* d_order, const float* d_weights,
                       const void* d_gate, uint8_t* d_q, uint8_t* d_scales, uint8_t* d_qt, uint8_t* d_scalesT,
                       hipStream_t stream)
{
    guarded("launchFp8Quantize", [&] {
        require(opt, "null option");
        graft::fp8_quantize(*opt, d_src, d_order, d_weights, d_gate, d_q, d_scales, d_qt, d_scalesT, stream);
    });
}

void launchFp8Product(const Fp8ProductOption* opt, const uint8_t* d_a, const uint8_t* d_aScales, const uint8_t* d_b,
                      const uint8_t* d_bScales, const int* d_offsets, void* d_out, hipStream_t stream)
{
    guarded("launchFp8Product", [&] {
        require(opt, "null option");
        graft::fp8_product(*opt, d_a, d_aScales, d_b, d_bScales, d_offsets, d_out, stream);
    });
}

void launchFp4Quantize(const Fp4QuantOption* opt, const void* d_src, const int* d_order, uint8_t* d_q, uint8_t* d_scales,
                       hipStream_t stream)
{
    guarded("launchFp4Quantize", [&] {
        require(opt, "null option");
        graft::fp4_quantize(*opt, d_src, d_order, d_q, d_scales, stream);
    });
}

void launchFp4Product(const Fp4ProductOption* opt, const uint8_t* d_a, const uint8_t* d_aScales, const uint8_t* d_b,
                      const uint8_t* d_bScales, const int* d_offsets, void* d_out, hipStream_t stream)
{
    guarded("launchFp4Product", [&] {
        require(opt, "null option");
        graft::fp4_product(*opt, d_a, d_aScales, d_b, d_bScales, d_offsets, d_out, stream);
    });
}

void launchExpertLayer(const ExpertLayerOption* opt, const void* d_x, const void* d_router, const float* d_bias,
                       const uint8_t* d_w1, const uint8_t* d_w1Scales, const uint8_t* d_w2, const uint8_t* d_w2Scales,
                       void* d_out, int numTokens, hipStream_t stream)
{
    guarded("launchExpertLayer", [&] {
        require(opt, "null option");
        graft::expert_layer(*opt, {d_x, d_router, d_bias, d_w1, d_w1Scales, d_w2, d_w2Scales}, d_out, numTokens, stream);
    });
}

void launchExpertCombine(int dim, int dataType, const void* d_rows, int numRows, long long rowStride,
                         const int* d_position, const float* d_weights, void* d_out, long long outStride, int numTokens,
                         int topK, hipStream_t stream)
{
    guarded("launchExpertCombine", [&] {
        graft::expert_combine(dim, dataType, d_rows, numRows, rowStride, d_position, d_weights, d_out, outStride,
                              numTokens, topK, stream);
    });
}

void launchExpertCombineBackward(int dim, int dataType, const void* d_rows, int numRows, long long rowStride,
                                 const int* d_position, const void* d_dout, long long doutStride, float* d_dweights,
                                 int numTokens, int topK, hipStream_t stream)
{
    guarded("launchExpertCombineBackward", [&] {
        graft::expert_combine_backward(dim, dataType, d_rows, numRows, rowStride, d_position, d_dout, doutStride,
                                       d_dweights, numTokens, topK, stream);
    });
}

void launchNormGateResidual(const NormGateOption* opt, const void* d_x, const void* d_f, const void* d_gate,
                            const float* d_postWeight, const float* d_postBias, const float* d_preWeight,
                            const float* d_preBias, void* d_y, void* d_h, int numRows, hipStream_t stream)
{
    guarded("launchNormGateResidual", [&] {
        require(opt, "null option");
        graft::norm_gate(*opt, {d_x, d_f, d_gate, d_postWeight, d_postBias, d_preWeight, d_preBias}, d_y, d_h, numRows,
                         stream);
    });
}

void launchNormGateResidualBackward(const NormGateOption* opt, const void* d_x, const void* d_f, const void* d_gate,
                                    const float* d_postWeight, const float* d_postBias, const float* d_preWeight,
                                    const float* d_preBias, const void* d_dy, const void* d_dh, void* d_dx, void* d_df,
                                    void* d_dgate, float* d_dPostWeight, float* d_dPostBias, float* d_dPreWeight,
                                    float* d_dPreBias, int numRows, hipStream_t stream)
{
    guarded("launchNormGateResidualBackward", [&] {
        require(opt, "null option");
        graft::norm_gate_backward(*opt, {d_x, d_f, d_gate, d_postWeight, d_postBias, d_preWeight, d_preBias}, d_dy, d_dh,
                                  {d_dx, d_df, d_dgate, d_dPostWeight, d_dPostBias, d_dPreWeight, d_dPreBias}, numRows,
                                  stream);
    });
}

}  // extern "C"
