/*
 * eri_layers -- C ABI of the layers at a transformer's entry on MI355X (gfx950): embedding lookup with scaling and its
 * gradient, dropout from a counter-based generator, and the residual's addition with root-mean-square norm, forward
 * and backward.  They produce gradients in the forms that the step of include/eri_optim8.h reads (the parameter's
 * dtype, or F32 beside BF16 parameters).
 *
 * Conventions are those of include/eri_optim8.h: 0 on success, a positive hipError_t or a negative EriStatus,
 * eri_last_error() for the message, streams as void* with NULL the default stream, nothing synchronises, and nothing
 * is allocated: workspaces are the caller's.  All pointers are device memory of the current device; ordinary host memory in a
 * kernel faults the device and is not looked for here.  Every call may be captured into a HIP graph.
 *
 * The argument structs are plain data: zero them first, so that fields added later read as "not used".  Rows lie
 * `*_stride` elements apart, with 0 for rows without gaps; the elements of a row are adjacent.  An address needs
 * the alignment of its element only; rows that begin at 16-byte addresses are read in whole words and run fastest.
 * Outputs overlap neither each other nor an input, but for rows written over rows of the same address, stride and dtype:
 *     eri_dropout        y over x
 *     eri_rms_norm       y and h, each over x or residual
 *     eri_rms_norm_grad  grad_x and grad_residual, each over grad, h or grad_h;  grad_weight over weight
 */
#ifndef ERI_LAYERS_H
#define ERI_LAYERS_H

#include "eri_optim8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A further dtype tag, for the norm's output only: 8-bit floats of 4 exponent and 3 mantissa bits, largest value 448, no infinities. */
#define ERI_DTYPE_F8E4M3 16

/* ---------------------------------------------------------------------------------------------
 * Lookup: out[t] = scale * table[ids[t]], rounded once.  An id outside [0, vocab) gives a row of zeros.
 * ------------------------------------------------------------------------------------------- */
typedef struct EriEmbedding {
    const void *ids;   /* tokens ids */
    const void *table; /* vocab rows of dim elements */
    void *out;         /* tokens rows of dim elements, dtype of the table */
    uint64_t tokens, vocab, dim;
    uint64_t table_stride, out_stride;
    int32_t ids_64;    /* 0: 32-bit ids, 1: 64-bit ids */
    int32_t dtype_tag; /* of table and out: F32 or BF16 */
    float scale;
    int32_t reserved;  /* 0 */
} EriEmbedding;
int eri_embedding(const EriEmbedding *args, void *stream);

/* ---------------------------------------------------------------------------------------------
 * The table's gradient: out[v] = scale * (sum of grad[t] over the tokens t with ids[t] = v), all rows of out written,
 * rows that no token names with zeros.  accumulate: the sum is added to what out holds, and rows without a token are
 * not touched.  Tokens whose id is padding_id or lies outside [0, vocab) add nothing.  The workspace that some tokens need does
 * for fewer tokens of the same table too.  Sums are F32 in an order that
 * the sizes and accumulate decide: the same call on the same inputs gives the same bits.
 * ------------------------------------------------------------------------------------------- */
typedef struct EriEmbeddingGrad {
    const void *ids;
    const void *grad; /* tokens rows of dim elements */
    void *out;        /* vocab rows of dim elements */
    void *workspace;  /* 16-byte aligned, eri_embedding_grad_workspace() bytes; few tokens need none */
    uint64_t workspace_bytes;
    uint64_t tokens, vocab, dim;
    uint64_t grad_stride, out_stride;
    int64_t padding_id; /* negative: none */
    int32_t ids_64;
    int32_t grad_dtype; /* F32 or BF16 */
    int32_t out_dtype;  /* F32 or BF16 */
    int32_t accumulate;
    float scale;
    int32_t reserved;   /* 0 */
} EriEmbeddingGrad;
int eri_embedding_grad_workspace(uint64_t tokens, uint64_t vocab, uint64_t dim, uint64_t *bytes);
int eri_embedding_grad(const EriEmbeddingGrad *args, void *stream);

/* ---------------------------------------------------------------------------------------------
 * Dropout.  Element i (counted through the rows as if they had no gaps) draws the 16 bits
 *     word (i mod 8) / 2, half i mod 2 (low half first)
 * of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter
 * {i / 8, offset} under key seed, each 64 bits, low word first.  It is kept where they are not below
 * floor(65536 p + 1/2), and then divided by the share of the 65536 values that is kept, so that the mean is kept
 * exactly; a dropped element is 0 whatever it was.  The backward pass is the same call on the gradient: the mask is
 * computed again and never stored.  Calls that shall be independent differ in seed or offset.
 * ------------------------------------------------------------------------------------------- */
typedef struct EriDropoutKey {
    uint64_t seed;
    uint64_t offset;
    const uint64_t *offset_ptr; /* NULL, or 8 bytes on the device that are added to offset when the kernel runs: a captured
                                   graph draws anew where something advances them between its replays */
    double p;                   /* share that is dropped, 0 .. 1; 0: nothing is drawn */
} EriDropoutKey;

typedef struct EriDropout {
    const void *x;
    void *y;
    uint64_t rows, cols;
    uint64_t x_stride, y_stride;
    EriDropoutKey key;
    int32_t dtype_tag; /* F32 or BF16 */
    int32_t reserved;  /* 0 */
} EriDropout;
int eri_dropout(const EriDropout *args, void *stream);

/* ---------------------------------------------------------------------------------------------
 * Residual addition and root-mean-square norm:
 *     h = residual + dropout(x)           rstd = 1 / sqrt(mean of h^2 over the row + eps)
 *     y = h * rstd * weight               (from h before it is rounded to its dtype)
 * with y in F32, BF16, or F8E4M3 with scales: for each row (scale_group 0) or each 128 columns of a row (scale_group
 * 128, the last group of a row may be shorter) scale = max|y| / 448, or 1 where max|y| is below 2^-100.  The 8-bit value
 * is y * (448 / max|y|) (y itself where the scale is 1 for that reason), computed in F32 and rounded to nearest even: where y / scale
 * lies within F32's rounding of the middle between two 8-bit values it may be either.  NaN is left out of max|y| and
 * stays NaN.
 * ------------------------------------------------------------------------------------------- */
typedef struct EriRmsNorm {
    const void *x;        /* rows of cols elements */
    const void *residual; /* NULL: nothing is added */
    const void *weight;   /* cols elements, NULL: ones */
    void *y;
    void *h;              /* NULL: not stored; dtype of the residual, of x without one */
    float *rstd;          /* NULL: not stored; one per row */
    float *scales;        /* with F8E4M3: rows x (1 or ceil(cols / 128)), without gaps */
    uint64_t rows, cols;
    uint64_t x_stride, residual_stride, y_stride, h_stride;
    EriDropoutKey key;
    float eps;
    int32_t x_dtype, residual_dtype, weight_dtype; /* F32 or BF16 */
    int32_t y_dtype;                               /* F32, BF16 or F8E4M3 */
    int32_t scale_group;                           /* 0 or 128 */
} EriRmsNorm;
int eri_rms_norm(const EriRmsNorm *args, void *stream);

/* Its gradient, from grad = dL/dy and grad_h = dL/dh (what reaches h besides the norm; NULL: nothing):
 *     dh = grad_h + rstd * (grad * weight) - h * rstd^3 * mean(grad * weight * h)
 *     grad_residual = dh     grad_x = dropout(dh)     grad_weight = sum over rows of grad * h * rstd
 * Any of the three outputs may be NULL.  Sums are F32; grad_weight's order is decided by the sizes, the device's
 * number of compute units and whether an output lies over grad, h or weight: the same call on the same inputs gives the
 * same bits.  The workspace that some rows need does for fewer rows of the same length too. */
typedef struct EriRmsNormGrad {
    const void *grad;
    const void *h;
    const float *rstd;
    const void *weight;  /* NULL: ones */
    const void *grad_h;
    void *grad_x;
    void *grad_residual;
    void *grad_weight;   /* cols elements */
    void *workspace;     /* 16-byte aligned, eri_rms_norm_grad_workspace() bytes; not read without grad_weight */
    uint64_t workspace_bytes;
    uint64_t rows, cols;
    uint64_t grad_stride, h_stride, grad_h_stride, grad_x_stride, grad_residual_stride;
    EriDropoutKey key;
    int32_t grad_dtype;  /* of grad: F32 or BF16 */
    int32_t h_dtype;     /* of h, grad_h and grad_residual */
    int32_t x_dtype;     /* of grad_x */
    int32_t weight_dtype, grad_weight_dtype;
    int32_t reserved;    /* 0 */
} EriRmsNormGrad;
int eri_rms_norm_grad_workspace(uint64_t rows, uint64_t cols, uint64_t *bytes);
int eri_rms_norm_grad(const EriRmsNormGrad *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ERI_LAYERS_H */
