// Internal interface of grad_norm.hip; the options are those of grad_abi.h.
#pragma once

#include "experts.h"
#include "grad_abi.h"

namespace graft {

void grad_norm(const GradTensor* tensors, int count, int norm, float scale, float* d_norm, hipStream_t s);
void grad_clip(const GradTensor* tensors, int count, float max_norm, int non_finite, const float* d_norm, hipStream_t s);
void grad_norm_clip(const GradTensor* tensors, int count, int norm, float scale, float max_norm, int non_finite,
                    float* d_norm, hipStream_t s);

}  // namespace graft
