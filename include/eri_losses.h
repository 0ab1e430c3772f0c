/*
 * eri_losses -- C ABI of what stands between a model's logits and its gradients on MI355X (gfx950): log probabilities of
 * given tokens with entropy and top alternatives, and distillation from a teacher of which only the top tokens are kept, each
 * with the logits' gradient.
 *
 * Conventions are those of include/eri_layers.h: 0 on success, a positive hipError_t or a negative EriStatus,
 * eri_last_error() for the message, streams as void*, nothing synchronises, nothing is allocated, all pointers are device
 * memory of the current device, every call may be captured into a HIP graph.  Zero the argument structs first.  Rows of logits and of
 * out lie `*_stride` elements apart, those of a teacher's ids and values too, with 0 for rows without gaps; what has one value or a
 * few for each row has no gaps.  An address needs the alignment of its element only.  Outputs overlap neither each other nor an input, but
 * for the gradient's rows over the logits' (same address, stride and dtype).
 *
 * x is a row of `vocab` logits, T the temperature, m the largest logit and s the sum of exp((x - m) / T) over the row; p = exp((x - m) / T) / s.
 * Minus infinity is a token that cannot occur.  A row whose logits are all minus infinity leaves nothing: its log probabilities are minus infinity, its
 * entropy 0, its gradient 0.  A row that holds NaN or plus infinity has no softmax: what is computed from it is NaN.
 * A token id outside [0, vocab) names no token.  Sums are F32 or wider, in an order that the sizes
 * and the rows' distance from multiples of 128 bytes decide: the same call on the same inputs at the same addresses gives the same bits.
 */
#ifndef ERI_LOSSES_H
#define ERI_LOSSES_H

#include "eri_optim8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most alternatives of a row, and most tokens of a teacher. */
#define ERI_TOP_MOST 64

/* ---------------------------------------------------------------------------------------------
 * Scores of tokens:
 *     logprob = (x[id] - m) / T - ln s      0 where the id names no token
 *     entropy = ln s - (sum of p (x - m)) / T
 *     top: the top_n largest logits of the row as log probabilities, and their ids: in descending order, of equal logits the
 *          lowest id first.  In a row that holds NaN or plus infinity they are NaN, and the ids 0, 1, 2, ...
 *     stats = {m, ln s}, what the gradient takes; m / T + ln s is the log of the sum of exp(x / T).  {-inf, -inf} where nothing is left
 * The workspace that some rows need does for fewer rows of the same length and for fewer alternatives too.
 * ------------------------------------------------------------------------------------------- */
typedef struct EriTokenLogprobs {
    const void *logits; /* rows of vocab elements */
    const void *ids;    /* one per row; NULL: no logprob */
    float *logprob;     /* one per row */
    float *entropy;     /* NULL, or one per row */
    float *stats;       /* two per row */
    float *top;         /* top_n per row */
    int64_t *top_ids;   /* top_n per row */
    void *workspace;    /* 16-byte aligned, eri_token_logprobs_workspace() bytes */
    uint64_t workspace_bytes;
    uint64_t rows, vocab;
    uint64_t logits_stride;
    float temperature;  /* 1e-4 .. 1e4 */
    int32_t ids_64;     /* 0: 32-bit ids, 1: 64-bit ids */
    int32_t dtype_tag;  /* of logits: F32 or BF16 */
    int32_t top_n;      /* 0 .. ERI_TOP_MOST and vocab */
} EriTokenLogprobs;
int eri_token_logprobs_workspace(uint64_t rows, uint64_t vocab, int32_t top_n, uint64_t *bytes);
int eri_token_logprobs(const EriTokenLogprobs *args, void *stream);

/* The logits' gradient from grad = dL/dlogprob and grad_entropy = dL/dentropy:
 *     out[j] = (grad * ([j = id] - p[j]) - grad_entropy * p[j] * (ln p[j] + entropy)) / T
 * A row whose id names no token gets nothing from grad, and one that gets nothing from either is written with zeros and not read.  A token whose p
 * is 0 gets nothing but grad / T where it is the named one, as long as (grad + grad_entropy * entropy) / T and 256 grad_entropy / T are finite in F32; past that
 * a row may hold infinities and NaN. */
typedef struct EriTokenLogprobsGrad {
    const void *logits;
    const void *ids;
    const float *stats;
    const float *grad;         /* one per row; NULL with ids: nothing comes from the log probabilities */
    const float *grad_entropy; /* one per row; NULL: nothing comes from the entropies */
    const float *entropy;      /* with grad_entropy */
    void *out;                 /* rows of vocab elements */
    uint64_t rows, vocab;
    uint64_t logits_stride, out_stride;
    float temperature;
    int32_t ids_64;
    int32_t dtype_tag; /* of logits */
    int32_t out_dtype; /* F32 or BF16 */
} EriTokenLogprobsGrad;
int eri_token_logprobs_grad(const EriTokenLogprobsGrad *args, void *stream);

/* ---------------------------------------------------------------------------------------------
 * Distillation from a teacher's k top tokens: `teacher` holds their log probabilities at the temperature of the loss (the `top` of
 * eri_token_logprobs).  With S the set of the ids, entries whose id names no token left out:
 *     rest = 0    q = exp(teacher) / (sum of exp(teacher)): the teacher's values may be logits / T too
 *                 loss = sum of q (ln q - ln p[id])
 *     rest = 1    all other tokens are one more class: q = exp(teacher), divided by their sum where that is over 1,
 *                 qr = 1 - sum of q, pr = the sum of p outside of S
 *                 loss = sum of q (ln q - ln p[id]) + qr (ln qr - ln pr)
 * 0 ln 0 is 0.  rest = 1 is as rest = 0 in a row where no token outside of S is left, because all stand at minus infinity or there is none.
 * A row whose teacher leaves nothing (no id names a token, or all its values are minus infinity) has loss 0 and no gradient with rest = 0.
 *     stats = {m, ln s, m and ln s of the tokens outside of S, ln of what exp(teacher) is divided by, pr - qr}, what the gradient
 *             takes; {.., .., m, ln s, .., 1} where there is no rest, the last 0 where the teacher leaves nothing
 * ------------------------------------------------------------------------------------------- */
typedef struct EriDistillTop {
    const void *logits;  /* rows of vocab elements */
    const void *ids;     /* rows of k ids */
    const void *teacher; /* rows of k elements */
    float *loss;         /* one per row */
    float *stats;        /* six per row */
    void *workspace;     /* 16-byte aligned, eri_distill_top_workspace() bytes */
    uint64_t workspace_bytes;
    uint64_t rows, vocab;
    uint64_t logits_stride, ids_stride, teacher_stride;
    float temperature;
    int32_t ids_64;
    int32_t dtype_tag;     /* of logits: F32 or BF16 */
    int32_t teacher_dtype; /* F32 or BF16 */
    int32_t k;             /* 1 .. ERI_TOP_MOST */
    int32_t rest;          /* 0 or 1 */
} EriDistillTop;
int eri_distill_top_workspace(uint64_t rows, uint64_t vocab, uint64_t *bytes);
int eri_distill_top(const EriDistillTop *args, void *stream);

/* The logits' gradient from grad = dL/dloss:
 *     out[j] = grad * (p[j] - sum of q over the entries with id j) / T            for j in S
 *     out[j] = grad * (p[j] / pr) * (pr - qr) / T, or grad * p[j] / T without rest  for the others
 * A row whose grad is 0 is written with zeros and not read. */
typedef struct EriDistillTopGrad {
    const void *logits;
    const void *ids;
    const void *teacher;
    const float *stats;
    const float *grad; /* one per row */
    void *out;         /* rows of vocab elements */
    uint64_t rows, vocab;
    uint64_t logits_stride, ids_stride, teacher_stride, out_stride;
    float temperature;
    int32_t ids_64;
    int32_t dtype_tag;
    int32_t teacher_dtype;
    int32_t out_dtype; /* F32 or BF16 */
    int32_t k;
} EriDistillTopGrad;
int eri_distill_top_grad(const EriDistillTopGrad *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ERI_LOSSES_H */
