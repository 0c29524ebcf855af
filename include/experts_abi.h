/*
 * C-ABI of the operators of a mixture-of-experts residual block on MI355X
 * (gfx950): routing of tokens (samples) to experts, products of 8-bit
 * matrices with a scale for each block of 128, the gather and combine of the
 * experts' rows, and the norms, gate and residual around a block; forward and
 * backward.  No counterpart exists in the reference, whose heads are single
 * MLPs of at most 128 (modules/TinyMLP).
 *
 * Conventions are those of tinymlp_abi.h: device pointers unless stated, a
 * trailing stream, void launchers that report through tinymlp_last_error()
 * and tinymlp_last_error_message().  Every argument error is reported before any
 * device call.  A batch of zero tokens or rows is valid and does nothing (but a
 * plan of it is written, with no rows, and the norms' parameters' gradients, of
 * zeros).  Results do not depend on the order in which the GPU runs workgroups:
 * repeated calls give the same bits.  Strides count elements; tokens and rows of
 * a call are at most 2^30.  Scratch, where a call needs any, belongs to (device,
 * stream) as for the other launchers (hipStreamPerThread: to each thread's own),
 * so calls of several host threads on one stream have to be serialised by the
 * caller; it grows with hipMalloc on a larger call than before, so a call that is
 * captured into a graph has to be made once before.  The graph keeps that
 * scratch, which stays allocated however large later calls on the stream are; its
 * replays have to be ordered with the stream's other calls, as those are among
 * themselves.
 */
#ifndef GRAFT_EXPERTS_ABI_H
#define GRAFT_EXPERTS_ABI_H

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Types of the tensors passed as void*. */
#define DATA_F32 0
#define DATA_F16 1
#define DATA_BF16 2

/* ---- routing -------------------------------------------------------------- */

#define ROUTE_SOFTMAX 0
#define ROUTE_SIGMOID 1

typedef struct RouteOption {
    int numExperts;   /* E, 1..1024 */
    int topK;         /* k, 1..32, at most E */
    int scoreType;    /* ROUTE_SOFTMAX or ROUTE_SIGMOID */
    int numGroups;    /* G, 1..64, divides E; 1: no groups */
    int topGroups;    /* groups kept, 1..G */
    int groupScore;   /* a group's score: its best expert (1) or the sum of its best two (2) */
    int renormalize;  /* nonzero: weights are divided by their sum + 1e-20 */
    float scale;      /* the weights' factor */
    int logitsType;   /* DATA_* */
} RouteOption;

/* Scores s = softmax(logits) or sigmoid(logits) of each token; the topK experts
 * of the largest s + bias (bias fp32 [E], nullable: it selects, it does not
 * weigh) among the topGroups best groups, largest first, equal ones lowest
 * index first; weights from s.  d_indices, d_weights [numTokens x topK].
 * An expert whose logit is -infinity or NaN, or whose s + bias is, is not
 * available: it is never selected, and its score is 0 if its logit says so.  A
 * group's best two are of its available experts.  Where a token has fewer than
 * topK experts left, its last indices are -1 and their weights 0.  A logit of
 * +infinity counts as the largest finite number. */
void launchRouteExperts(const RouteOption* opt, const void* d_logits, long long logitsStride,
                        const float* d_bias, int* d_indices, float* d_weights, int numTokens,
                        hipStream_t stream);

/* dL/dlogits (type of the logits) from dL/dweights, for indices that
 * launchRouteExperts gave (distinct in a row; others than 0..E-1 are skipped).
 * The bias has no gradient.  d_dlogits may be d_logits, with the same stride. */
void launchRouteExpertsBackward(const RouteOption* opt, const void* d_logits, long long logitsStride,
                                const int* d_indices, const float* d_dweights, void* d_dlogits,
                                long long dlogitsStride, int numTokens, hipStream_t stream);

/* Rows that a plan of these sizes can need at most, a multiple of align
 * (host; -1 for sizes that a plan cannot have). */
long long routePlanCapacity(int numTokens, int topK, int numExperts, int align);

/* The experts' rows.  Slot t * topK + j (token t's j-th expert) gets a row in
 * the segment of its expert, in slot order; segments follow each other, each
 * from a multiple of `align` (1..128) rows on:
 *   d_offsets  [numExperts + 1]  first row of each expert's segment, and the end
 *   d_order    [capacity]        the slot of a row, -1 in rows that fill a segment up or follow the last
 *   d_position [numTokens x topK] the row of a slot, -1 for an index outside 0..E-1
 * capacity is at least routePlanCapacity(...). */
void launchRoutePlan(const int* d_indices, int numTokens, int topK, int numExperts, int align, int capacity,
                     int* d_offsets, int* d_order, int* d_position, hipStream_t stream);

/* ---- 8-bit matrices --------------------------------------------------------
 *
 * An 8-bit matrix [rows x cols] is held as OCP e4m3 bytes [rows x pitch], pitch
 * = cols rounded up to a multiple of 128, zero behind cols, and one scale byte
 * for each block of 128 columns (and of 1 or 128 rows), the power of two
 * 2^(byte - 127): [block rows x scale pitch], scale pitch = blocks rounded up
 * to a multiple of 4.  Both start at a multiple of 16 (bytes) and 4 (scales).
 * A scale is the smallest power of two that brings the block's finite values
 * within 448, at least 2^-126, so that quantising is exact but for one
 * rounding to e4m3 (to nearest, ties to even); infinities and NaN become NaN.
 */

typedef struct Fp8QuantOption {
    int rows, cols;            /* of one quantised matrix; cols 1..2^22 */
    int batch;                 /* matrices, 1..65535; with order or gate: 1 */
    int blockRows;             /* rows that share a scale: 1, or 128 (then transposed blocks are the same blocks) */
    int srcType;               /* DATA_* */
    int slotsPerRow;           /* with order: source row = slot / slotsPerRow */
    int srcRows;               /* rows of the source; slots beyond them read as zero */
    long long srcStride;       /* between source rows */
    long long srcBatchStride;  /* between source matrices */
    long long gateStride;      /* between the gate's rows */
} Fp8QuantOption;

/* Quantises x, or rows gathered from it: row r of the result is source row r,
 * or with d_order (nullable) source row d_order[r] / slotsPerRow, times
 * d_weights[d_order[r]] (nullable, fp32, with order), and zero where d_order[r]
 * is -1; with d_gate (nullable, type of the source, one row for each quantised
 * row) zero where the gate is not above 0 (the gradient behind a ReLU).
 * d_q, d_scales: the matrix [rows x cols]; d_qt, d_scalesT: its transpose
 * [cols x rows], quantised along the rows (blockRows 1: each column's block of
 * 128 rows has its scale; 128: the same blocks).  Either pair may be NULL. */
void launchFp8Quantize(const Fp8QuantOption* opt, const void* d_src, const int* d_order, const float* d_weights,
                       const void* d_gate, uint8_t* d_q, uint8_t* d_scales, uint8_t* d_qt, uint8_t* d_scalesT,
                       hipStream_t stream);

#define PRODUCT_DENSE 0 /* out [m x n] = A B^T */
#define PRODUCT_ROWS 1  /* A's rows [offsets[e], offsets[e+1]) times expert e's B */
#define PRODUCT_SUM 2   /* out of expert e: A's and B's columns [offsets[e], offsets[e+1]) */

typedef struct Fp8ProductOption {
    int m, n, k;          /* A [m x k], B [n x k] (DENSE, SUM) or [numExperts x n x k] (ROWS); n, k 1..2^22 (SUM: k from 0) */
    int numExperts;       /* 1..1024; DENSE: 1 */
    int grouping;         /* PRODUCT_* */
    int scaleRowsB;       /* rows of B that share a scale: 128 or 1 */
    int activation;       /* 0: none, 1: ReLU on the result */
    int outType;          /* DATA_*, with PRODUCT_EXACT or'ed to it on request */
    long long outStride;  /* between rows of out */
} Fp8ProductOption;

/* Results of any type from sums of exact products in fp32, whatever the sizes. */
#define PRODUCT_EXACT 0x100

/* out [m x n] (SUM: [numExperts x m x n], rows outStride apart, matrices m *
 * outStride) from 8-bit matrices, sums in fp32.  A has a scale for each row's
 * blocks.  d_offsets [numExperts + 1] ascending from launchRoutePlan (NULL for
 * DENSE); SUM needs them to be multiples of 128 (align 128), and gives an
 * expert without columns zeros.  ROWS leaves rows outside all segments as they
 * are.  NaN in a row's values makes that row's results NaN.
 *
 * fp32 results are sums of exact products in fp32, and so are all of SUM and all
 * with PRODUCT_EXACT, as far as the values are bf16 numbers: with scales of 2^-110
 * to 2^119 (bytes 17 to 246) they all are; of smaller scales' values what lies
 * below 2^-133 is lost, and values of 2^128 and more are infinite.  Other 16-bit
 * results may come from the matrix cores' 8-bit sums, 1.5 times as fast; which
 * calls take them goes by m, n and k.  Those add
 * eight products (of consecutive k) at a time and cut each towards zero to a
 * multiple of 2^-13 of the largest one's power of two, and add the eights in
 * fp32: a result is within 7 * 2^-13 of the sum of the eights' largest |a b|,
 * hence of the sum of all |a b|, besides fp32 rounding.  Where large products of
 * an eight cancel, that can be more than the result's own rounding, or all of it.
 * Of normal values it is 1.5e-5 of the results (2-norm), of non-negative ones
 * 3e-6, of values spread over all of e4m3 7e-5. */
void launchFp8Product(const Fp8ProductOption* opt, const uint8_t* d_a, const uint8_t* d_aScales, const uint8_t* d_b,
                      const uint8_t* d_bScales, const int* d_offsets, void* d_out, hipStream_t stream);

/* ---- the experts' rows back to tokens --------------------------------------- */

/* Or'ed to the dataType of the two launchers below: rows are fp32 whatever the
 * tokens' type, so that nothing is rounded between the experts' products
 * (outType DATA_F32) and the tokens. */
#define COMBINE_ROWS_F32 0x100

/* out[t] = sum_j weights[t, j] * rows[position[t, j]] in fp32, rounded once
 * (weights NULL: 1 each; a position outside 0..numRows-1 adds nothing).
 * rows [numRows x dim], out [numTokens x dim], both of dataType (rows fp32 with
 * COMBINE_ROWS_F32); dim 1..2^23, topK 1..32. */
void launchExpertCombine(int dim, int dataType, const void* d_rows, int numRows, long long rowStride,
                         const int* d_position, const float* d_weights, void* d_out, long long outStride,
                         int numTokens, int topK, hipStream_t stream);

/* dL/dweights [numTokens x topK] (fp32) = <dout[t], rows[position[t, j]]>, 0 for
 * positions outside; types as above, dout's as out's.  The rows' own gradient is weights * dout, which
 * launchFp8Quantize forms from dout, the order and the weights. */
void launchExpertCombineBackward(int dim, int dataType, const void* d_rows, int numRows, long long rowStride,
                                 const int* d_position, const void* d_dout, long long doutStride, float* d_dweights,
                                 int numTokens, int topK, hipStream_t stream);

/* ---- norms around a block, gate and residual --------------------------------- */

#define NORM_NONE 0
#define NORM_RMS 1
#define NORM_LAYER 2

typedef struct NormGateOption {
    int dim;              /* D, 1..8192 */
    int postNorm;         /* NORM_*: of the block's output f */
    int preNorm;          /* NORM_*: of the stream y, giving the next block's input h */
    int gateRows;         /* consecutive rows that share a row of the gate; 0: no gate */
    float residualScale;  /* alpha */
    float blockScale;     /* beta */
    float epsilon;
    int dataType;         /* DATA_*, of x, f, gate, y, h and their gradients */
    long long strideX, strideF, strideGate, strideY, strideH;  /* between rows; gradients have their tensor's (dy: y, dh: h) */
} NormGateOption;

/* y = alpha x + beta gate * postnorm(f),  h = prenorm(y):
 *   RMS    n = v / sqrt(mean(v^2) + eps) * weight + bias
 *   LAYER  the same of v - mean(v)
 * over each row, statistics in fp32, h from y before its rounding.  gate
 * [ceil(numRows / gateRows) x D].  Weights and biases fp32 [D]; a NULL weight is
 * 1, a NULL bias 0.  f NULL: y = alpha x (no gate, no post norm).  y or h may be
 * NULL, not both; a row of x is read before that of y is written, so y may be x,
 * with its stride.  y, h, x and f do not overlap otherwise. */
void launchNormGateResidual(const NormGateOption* opt, const void* d_x, const void* d_f, const void* d_gate,
                            const float* d_postWeight, const float* d_postBias, const float* d_preWeight,
                            const float* d_preBias, void* d_y, void* d_h, int numRows, hipStream_t stream);

/* Gradients of the same from dL/dy and dL/dh (either may be NULL: zero); x and f
 * are all that is kept of the forward.  dx (stride X), df (stride F), dgate and
 * the parameters' gradients (fp32 [D], summed over the rows in a fixed order)
 * are stored, not added; each may be NULL. */
void launchNormGateResidualBackward(const NormGateOption* opt, const void* d_x, const void* d_f, const void* d_gate,
                                    const float* d_postWeight, const float* d_postBias, const float* d_preWeight,
                                    const float* d_preBias, const void* d_dy, const void* d_dh, void* d_dx, void* d_df,
                                    void* d_dgate, float* d_dPostWeight, float* d_dPostBias, float* d_dPreWeight,
                                    float* d_dPreBias, int numRows, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
