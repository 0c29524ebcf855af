// extern "C" surface of the gradients' norm and its clipping (grad_abi.h).
#include "grad_abi.h"

#include "abi_error.h"
#include "grad_norm.h"

using graft::guarded;

extern "C" {

void launchGradNorm(const GradTensor* tensors, int count, int norm, float gradScale, float* d_norm, hipStream_t stream)
{
    guarded("launchGradNorm", [&] { graft::grad_norm(tensors, count, norm, gradScale, d_norm, stream); });
}

void launchGradClip(const GradTensor* tensors, int count, float maxNorm, int nonFinite, const float* d_norm,
                    hipStream_t stream)
{
    guarded("launchGradClip", [&] { graft::grad_clip(tensors, count, maxNorm, nonFinite, d_norm, stream); });
}

void launchGradNormClip(const GradTensor* tensors, int count, int norm, float gradScale, float maxNorm, int nonFinite,
                        float* d_norm, hipStream_t stream)
{
    guarded("launchGradNormClip",
            [&] { graft::grad_norm_clip(tensors, count, norm, gradScale, maxNorm, nonFinite, d_norm, stream); });
}

}  // extern "C"
