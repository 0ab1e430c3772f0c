/*
 * Host side of include/eri_losses.h: checks the arguments, then launches.  Nothing is allocated and nothing waits.
 */
#include "eri_layers_host.h"
#include "eri_losses_device.h"

namespace {

constexpr float kColdest = 1e-4f, kHottest = 1e4f;

/* What every call has. */
int logits_ok(uint64_t rows, uint64_t vocab, uint64_t *logits_stride, int dtype_tag, float temperature, const char *kCall) {
    ERI_NEED(floating(dtype_tag), ERI_ERR_DTYPE, "unsupported dtype tag of the logits (F32=0 and BF16=2 are supported)");
    ERI_NEED(vocab != 0, ERI_ERR_EMPTY, "rows without elements");
    ERI_NEED(rows <= kCountMost && vocab <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
    ERI_NEED(stride(logits_stride, vocab), ERI_ERR_ARG, "a stride shorter than a row");
    ERI_NEED(temperature >= kColdest && temperature <= kHottest, ERI_ERR_ARG, "the temperature is not between 1e-4 and 1e4");
    return 0;
}
int ids_ok(const void *ids, int ids_64, const char *kCall) {
    ERI_NEED(ids_64 == 0 || ids_64 == 1, ERI_ERR_DTYPE, "ids_64 is neither 0 nor 1");
    ERI_NEED(aligned(ids, ids_64 ? 8 : 4), ERI_ERR_ALIGN, "ids are not aligned to their size");
    return 0;
}
int teacher_ok(const void *teacher, int dtype, uint64_t k, uint64_t *ids_stride, uint64_t *teacher_stride, const char *kCall) {
    ERI_NEED(k >= 1 && k <= ERI_TOP_MOST, ERI_ERR_ARG, "k is not between 1 and 64");
    ERI_NEED(floating(dtype), ERI_ERR_DTYPE, "unsupported dtype tag of the teacher (F32=0 and BF16=2 are supported)");
    ERI_NEED(aligned(teacher, size_of(dtype)), ERI_ERR_ALIGN, "teacher is not aligned to its elements");
    ERI_NEED(stride(ids_stride, k) && stride(teacher_stride, k), ERI_ERR_ARG, "a stride shorter than a row");
    return 0;
}
int workspace_ok(const void *workspace, uint64_t bytes, uint64_t need, const char *kCall) {
    ERI_NEED(workspace || need == 0, ERI_ERR_NULL, "workspace is NULL");
    ERI_NEED(aligned(workspace, 16), ERI_ERR_ALIGN, "workspace is not 16-byte aligned");
    ERI_NEED(bytes >= need, ERI_ERR_ARG, "workspace is too small");
    return 0;
}
#define ERI_PASS(check)              \
    do {                             \
        if (int rc = check) return rc; \
    } while (0)

bool top_ok(int32_t top_n, uint64_t vocab) { return top_n >= 0 && top_n <= ERI_TOP_MOST && (uint64_t)top_n <= vocab; }

} // namespace

extern "C" {

int eri_token_logprobs_workspace(uint64_t rows, uint64_t vocab, int32_t top_n, uint64_t *bytes) {
    constexpr const char *kCall = "eri_token_logprobs_workspace";
    ERI_NEED(bytes, ERI_ERR_NULL, "bytes is NULL");
    ERI_NEED(vocab != 0, ERI_ERR_EMPTY, "rows without elements");
    ERI_NEED(rows <= kCountMost && vocab <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
    ERI_NEED(top_ok(top_n, vocab), ERI_ERR_ARG, "top_n is not between 0 and 64, or over vocab");
    *bytes = rows ? eri_losses::token_logprobs_workspace(rows, vocab, (uint32_t)top_n) : 0;
    return 0;
}

int eri_token_logprobs(const EriTokenLogprobs *args, void *stream) {
    constexpr const char *kCall = "eri_token_logprobs";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriTokenLogprobs a = *args;
    ERI_PASS(logits_ok(a.rows, a.vocab, &a.logits_stride, a.dtype_tag, a.temperature, kCall));
    ERI_PASS(ids_ok(a.ids, a.ids_64, kCall));
    ERI_NEED(top_ok(a.top_n, a.vocab), ERI_ERR_ARG, "top_n is not between 0 and 64, or over vocab");
    if (a.rows == 0) return 0;
    ERI_NEED(a.logits && a.stats, ERI_ERR_NULL, "logits or stats is NULL");
    ERI_NEED((a.ids != nullptr) == (a.logprob != nullptr), ERI_ERR_NULL, "one of ids and logprob is NULL");
    ERI_NEED(a.top_n == 0 || (a.top && a.top_ids), ERI_ERR_NULL, "top or top_ids is NULL");
    ERI_NEED(aligned(a.logits, size_of(a.dtype_tag)) && aligned(a.logprob, 4) && aligned(a.entropy, 4) && aligned(a.stats, 4) && aligned(a.top, 4) && aligned(a.top_ids, 8),
             ERI_ERR_ALIGN, "an address is not aligned to its elements");
    ERI_PASS(workspace_ok(a.workspace, a.workspace_bytes, eri_losses::token_logprobs_workspace(a.rows, a.vocab, (uint32_t)a.top_n), kCall));
    return done(eri_losses::launch_token_logprobs(a, stream), kCall);
}

int eri_token_logprobs_grad(const EriTokenLogprobsGrad *args, void *stream) {
    constexpr const char *kCall = "eri_token_logprobs_grad";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriTokenLogprobsGrad a = *args;
    ERI_PASS(logits_ok(a.rows, a.vocab, &a.logits_stride, a.dtype_tag, a.temperature, kCall));
    ERI_PASS(ids_ok(a.ids, a.ids_64, kCall));
    ERI_NEED(floating(a.out_dtype), ERI_ERR_DTYPE, "unsupported dtype tag of out (F32=0 and BF16=2 are supported)");
    ERI_NEED(stride(&a.out_stride, a.vocab), ERI_ERR_ARG, "a stride shorter than a row");
    if (a.rows == 0) return 0;
    ERI_NEED(a.logits && a.stats && a.out, ERI_ERR_NULL, "logits, stats or out is NULL");
    ERI_NEED((a.ids != nullptr) == (a.grad != nullptr), ERI_ERR_NULL, "one of ids and grad is NULL");
    ERI_NEED((a.grad_entropy != nullptr) == (a.entropy != nullptr), ERI_ERR_NULL, "one of grad_entropy and entropy is NULL");
    ERI_NEED(a.grad || a.grad_entropy, ERI_ERR_NULL, "grad and grad_entropy are NULL");
    ERI_NEED(aligned(a.logits, size_of(a.dtype_tag)) && aligned(a.out, size_of(a.out_dtype)) && aligned(a.stats, 4) && aligned(a.grad, 4) && aligned(a.grad_entropy, 4) &&
                 aligned(a.entropy, 4),
             ERI_ERR_ALIGN, "an address is not aligned to its elements");
    return done(eri_losses::launch_token_logprobs_grad(a, stream), kCall);
}

int eri_distill_top_workspace(uint64_t rows, uint64_t vocab, uint64_t *bytes) {
    constexpr const char *kCall = "eri_distill_top_workspace";
    ERI_NEED(bytes, ERI_ERR_NULL, "bytes is NULL");
    ERI_NEED(vocab != 0, ERI_ERR_EMPTY, "rows without elements");
    ERI_NEED(rows <= kCountMost && vocab <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
    *bytes = rows ? eri_losses::distill_top_workspace(rows, vocab) : 0;
    return 0;
}

int eri_distill_top(const EriDistillTop *args, void *stream) {
    constexpr const char *kCall = "eri_distill_top";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriDistillTop a = *args;
    ERI_PASS(logits_ok(a.rows, a.vocab, &a.logits_stride, a.dtype_tag, a.temperature, kCall));
    ERI_PASS(ids_ok(a.ids, a.ids_64, kCall));
    ERI_PASS(teacher_ok(a.teacher, a.teacher_dtype, (uint64_t)(int64_t)a.k, &a.ids_stride, &a.teacher_stride, kCall));
    ERI_NEED(a.rest == 0 || a.rest == 1, ERI_ERR_ARG, "rest is neither 0 nor 1");
    if (a.rows == 0) return 0;
    ERI_NEED(a.logits && a.ids && a.teacher && a.loss && a.stats, ERI_ERR_NULL, "logits, ids, teacher, loss or stats is NULL");
    ERI_NEED(aligned(a.logits, size_of(a.dtype_tag)) && aligned(a.loss, 4) && aligned(a.stats, 4), ERI_ERR_ALIGN, "an address is not aligned to its elements");
    ERI_PASS(workspace_ok(a.workspace, a.workspace_bytes, eri_losses::distill_top_workspace(a.rows, a.vocab), kCall));
    return done(eri_losses::launch_distill_top(a, stream), kCall);
}

int eri_distill_top_grad(const EriDistillTopGrad *args, void *stream) {
    constexpr const char *kCall = "eri_distill_top_grad";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriDistillTopGrad a = *args;
    ERI_PASS(logits_ok(a.rows, a.vocab, &a.logits_stride, a.dtype_tag, a.temperature, kCall));
    ERI_PASS(ids_ok(a.ids, a.ids_64, kCall));
    ERI_PASS(teacher_ok(a.teacher, a.teacher_dtype, (uint64_t)(int64_t)a.k, &a.ids_stride, &a.teacher_stride, kCall));
    ERI_NEED(floating(a.out_dtype), ERI_ERR_DTYPE, "unsupported dtype tag of out (F32=0 and BF16=2 are supported)");
    ERI_NEED(stride(&a.out_stride, a.vocab), ERI_ERR_ARG, "a stride shorter than a row");
    if (a.rows == 0) return 0;
    ERI_NEED(a.logits && a.ids && a.teacher && a.stats && a.grad && a.out, ERI_ERR_NULL, "logits, ids, teacher, stats, grad or out is NULL");
    ERI_NEED(aligned(a.logits, size_of(a.dtype_tag)) && aligned(a.out, size_of(a.out_dtype)) && aligned(a.stats, 4) && aligned(a.grad, 4), ERI_ERR_ALIGN,
             "an address is not aligned to its elements");
    return done(eri_losses::launch_distill_top_grad(a, stream), kCall);
}

} // extern "C"
