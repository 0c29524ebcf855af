/*
 * C-ABI of the gradients' global norm and its clipping on MI355X (gfx950), for
 * gradients that lie in arrays of the caller's: those of the backward launchers of
 * tinymlp_abi.h and experts_abi.h, and of the TinyMLP and TinyMLPHashGrid classes
 * (w_grad, b_grad and, where the table's gradient is an array, hashtable_grads).
 * A step runs it between the backward and the Adam launchers (tinymlp_abi.h), whose
 * lossScale is gradScale here.  The training steps of InstantNerf and NerfTrainer
 * do not clip: their binned scatter updates the table as its sums complete, without
 * an array of its gradients.  No counterpart exists in the reference, whose
 * optimizer takes the gradients as they are.
 *
 * Conventions are those of experts_abi.h: a trailing stream, errors through
 * tinymlp_last_error() before any device call, scratch by (device, stream), the
 * same bits from repeated calls.  The list of tensors is a host array, read
 * during the call and not kept; a call that is captured into a graph keeps its
 * contents.
 */
#ifndef GRAFT_GRAD_ABI_H
#define GRAFT_GRAD_ABI_H

#include "experts_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct GradTensor {
    const void* data;  /* device, n elements without gaps; may be NULL if n is 0 */
    void* out;         /* where the clipped elements go: NULL or data: in place */
    long long n;       /* 0..2^40 */
    int dataType;      /* DATA_* */
} GradTensor;

#define GRAD_NORM_2 0   /* sqrt(sum g^2) */
#define GRAD_NORM_MAX 1 /* max |g| */

#define GRAD_NONFINITE_KEEP 0 /* a norm that is infinite or NaN: the gradients are left (copied to out) as they are */
#define GRAD_NONFINITE_ZERO 1 /* they become zero */

/* *d_norm (fp32) = the norm over all elements of all tensors, divided by
 * gradScale; 0 of none.  Squares are summed in 64 bits, so that none overflows
 * or vanishes; infinities and NaN among the gradients give such a norm, and so
 * does a norm beyond fp32.  count 0..65536. */
void launchGradNorm(const GradTensor* tensors, int count, int norm, float gradScale, float* d_norm, hipStream_t stream);

/* g = g * min(1, maxNorm / *d_norm) in fp32, rounded to g's type.  d_norm
 * is launchGradNorm's, or what ranks that hold parts of the gradients have made of
 * theirs.  In place nothing is written where the factor is 1.  maxNorm >= 0.
 * A tensor that is written may not overlap another of the list, or d_norm. */
void launchGradClip(const GradTensor* tensors, int count, float maxNorm, int nonFinite, const float* d_norm,
                    hipStream_t stream);

/* Both in one call: *d_norm, which is no part of any tensor, is the norm before
 * clipping. */
void launchGradNormClip(const GradTensor* tensors, int count, int norm, float gradScale, float maxNorm, int nonFinite,
                        float* d_norm, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
