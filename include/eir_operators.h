/*
 * eir_operators.h -- C-ABI of the row operators and the 8-bit contraction of
 * the einsum_ir B200 backend (sm_100a).
 *
 * The quantised layer around a contraction and what reads its result: the
 * root-mean-square norm with the residual's addition (and its backward pass),
 * the quantisation of rows to 8-bit integers with a scale a row, the
 * contraction of 8-bit integers with a scale for each token and channel, and
 * the log probabilities of given tokens with entropy and top alternatives (and
 * their backward pass). No counterpart in the reference.
 *
 * The conventions are those of eir_cuda.h: int status codes, no exceptions,
 * plans that are destroyed with eir_plan_destroy, device pointers owned by the
 * caller, calls asynchronous on `stream` (NULL = the legacy default stream).
 * A plan with a workspace (eir_plan_workspace_bytes() > 0) takes its memory on the first
 * call on a device that needs it, and keeps it until it is destroyed; such a call is
 * refused in a stream capture (EIR_INVALID_ARGUMENT). Calls that need it may come from
 * several streams and host threads: the next one waits for the last one's use. A
 * captured call cannot: the caller orders the replays of graphs that hold a plan's calls
 * against one another and against the plan's other calls, and they end before the plan
 * is destroyed.
 *
 * Matrices are row-major with unit column stride; a row stride is in elements.
 * An input's row stride may be any value >= 0 (0: every row is the same
 * one); an output's rows must not overlap (stride >= columns). Pointers need
 * the alignment of their element only: rows on 16-byte boundaries run faster.
 */
#ifndef EIR_OPERATORS_H
#define EIR_OPERATORS_H

#include "eir_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 8-bit integers (-127 .. 127 as written by the quantising operators; the
 * contraction takes -128 too) */
enum { EIR_INT8 = 3 };

/* --- root-mean-square norm with the residual's addition -------------------
 * h = x + residual; rstd = (mean(h^2) + eps)^(-1/2); y = h * rstd * weight.
 * Computed in FP32 from the inputs; h, y are rounded once when stored (y is
 * computed from the unrounded h). The sum of squares is FP32's too: above about
 * 1.8e19 an element's square is infinite, and rstd 0. With dtype_out EIR_INT8 a row of y is
 * stored as integers q and a scale s with y ~ q s: v = h * weight, m = max|v|,
 * q = round-to-even(v * (127 / m)), s = m * rstd / 127 (rstd cancels in q).
 * A row with m < 2^-100 gives q = 0, s = 0; a row with an infinity or NaN
 * gives q = 0, s = NaN. */
typedef struct {
  int64_t rows, cols;         /* cols >= 1 */
  int32_t dtype;              /* x, residual, sum, h: EIR_FP32 or EIR_BF16 */
  int32_t dtype_weight;       /* EIR_FP32 or EIR_BF16 */
  int32_t dtype_out;          /* EIR_FP32, EIR_BF16 or EIR_INT8 */
  int32_t dtype_grad;         /* dy, dsum, dx: EIR_FP32 or EIR_BF16 */
  double  eps;                /* >= 0 */
  int64_t stride_x, stride_residual, stride_sum, stride_out;
  int64_t stride_h, stride_dy, stride_dsum, stride_dx;
} eir_norm_desc;
int eir_norm_plan_create(eir_norm_desc const *desc, eir_plan **plan);
/* residual, weight (ones), sum (stores h) and rstd (FP32 [rows]) may be NULL;
 * scale (FP32 [rows]) is needed with EIR_INT8. sum may be x or residual itself
 * (same pointer and stride). */
int eir_norm(eir_plan *plan, void const *x, void const *residual, void const *weight, void *sum,
             void *out, float *scale, float *rstd, void *stream);
/* g = weight * dy; dx = rstd * (g - h * rstd^2 * mean(g * h)) + dsum, the
 * gradient of x and of residual alike; dweight = sum over rows of
 * dy * h * rstd (FP32 [cols], summed in a fixed order). h is the forward
 * call's sum (or its x where it had no residual), rstd the forward call's.
 * weight, dsum (the gradient that reaches h past the norm) and dweight may be
 * NULL; dx may be dy or dsum itself (same pointer and stride). */
int eir_norm_backward(eir_plan *plan, void const *dy, void const *h, void const *weight,
                      float const *rstd, void const *dsum, void *dx, float *dweight, void *stream);
/* the same with h's row stride given by the call (>= 0), not the plan: for a plan
 * whose backward pass reads x in one place and a sum with other rows in another */
int eir_norm_backward_strided(eir_plan *plan, void const *dy, void const *h, int64_t stride_h,
                              void const *weight, float const *rstd, void const *dsum, void *dx,
                              float *dweight, void *stream);

/* --- rows to 8-bit integers ---------------------------------------------------
 * m = max|x| of a row, q = round-to-even(x * (127 / m)), s = m / 127, with
 * the norm's rules for empty and non-finite rows. Weights [channels, k] take
 * one scale a channel the same way. */
typedef struct {
  int64_t rows, cols;         /* cols >= 1 */
  int32_t dtype;              /* EIR_FP32 or EIR_BF16 */
  int32_t pad_;
  int64_t stride_x, stride_out;
} eir_quantize_desc;
int eir_quantize_plan_create(eir_quantize_desc const *desc, eir_plan **plan);
int eir_quantize(eir_plan *plan, void const *x, void *q, float *scale, void *stream);

/* --- contraction of 8-bit integers with scales ------------------------------
 * acc[t, c] = sum over k of left[t, k] * right[c, k], exact in 32-bit integers
 * (k <= 131071); out[t, c] = act(acc * scale_left[t] * scale_right[c] + bias[c])
 * in FP32, rounded once when stored. EIR_ACT_GATED_SILU: the first n / 2
 * channels are gates, the others values; out has n / 2 columns,
 * out[t, c] = silu(z[t, c]) * z[t, c + n / 2], silu(z) = z / (1 + exp(-z)). */
enum { EIR_ACT_NONE = 0, EIR_ACT_RELU = 1, EIR_ACT_GATED_SILU = 2 };
typedef struct {
  int64_t m, n, k;            /* tokens, channels, summed dim */
  int32_t dtype_out;          /* EIR_FP32 or EIR_BF16 */
  int32_t activation;         /* EIR_ACT_* */
  int64_t stride_left, stride_right, stride_out;
} eir_contract_int8_desc;
int eir_contract_int8_plan_create(eir_contract_int8_desc const *desc, eir_plan **plan);
/* left [m, k], right [n, k] int8; scale_left FP32 [m], scale_right FP32 [n],
 * bias FP32 [n]: each of the three may be NULL (scales of one, no bias) */
int eir_contract_int8(eir_plan *plan, void const *left, void const *right, float const *scale_left,
                      float const *scale_right, float const *bias, void *out, void *stream);

/* --- log probabilities of given tokens -----------------------------------------
 * For a row x of `vocab` logits: lse = log(sum exp x), logprob = x[target] -
 * lse, entropy = -sum p log p with p = exp(x - lse), and the `top` largest
 * logits' indices and log probabilities, largest first, ties to the lowest
 * index. Logits of -infinity have probability 0 and add 0 to the entropy; a
 * row with nothing but -infinity gives lse = -infinity, logprob = -infinity
 * (top_logprob alike) and entropy 0; a NaN or +infinity makes the row's
 * values NaN. Finite logits may have any size, as masks too (a row whose
 * largest is beyond 2^20 in magnitude is read once more). A negative target is ignored (logprob 0); one >= vocab gives
 * NaN. */
typedef struct {
  int64_t rows, vocab;        /* 1 <= vocab < 2^31 */
  int32_t dtype;              /* logits, dlogits: EIR_FP32 or EIR_BF16 */
  int32_t top;                /* 0 .. min(32, vocab) */
  int64_t stride_logits, stride_dlogits;
} eir_logprob_desc;
int eir_logprob_plan_create(eir_logprob_desc const *desc, eir_plan **plan);
/* targets int64 [rows] and logprob FP32 [rows]: both or neither; entropy, lse
 * FP32 [rows] may be NULL; top_logprob FP32 and top_index int64, each
 * [rows, top], may be NULL */
int eir_logprob(eir_plan *plan, void const *logits, int64_t const *targets, float *logprob,
                float *entropy, float *lse, float *top_logprob, int64_t *top_index, void *stream);
/* dlogits = dlogprob * (onehot(target) - p) - dentropy * p * (x - lse +
 * entropy); lse and entropy are the forward call's. targets and dlogprob:
 * both or neither (neither: that term is 0); dentropy may be NULL (entropy is
 * read only with it); dlogits may be logits itself (same pointer and stride).
 * An ignored target takes no part; one >= vocab makes the row NaN; a row of
 * nothing but -infinity gets zeros. p is exp(x - lse) of the lse given, which
 * FP32 holds to 2^-24 of its size. The alternatives carry no gradient. */
int eir_logprob_backward(eir_plan *plan, void const *logits, int64_t const *targets,
                         float const *lse, float const *entropy, float const *dlogprob,
                         float const *dentropy, void *dlogits, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* EIR_OPERATORS_H */
