/*
 * Host side of include/eri_layers.h: checks the arguments, then launches.  Nothing is allocated and nothing waits.
 */
#include <atomic>
#include <cmath>

#include "eri_layers_device.h"
#include "eri_layers_host.h"

namespace {

using eri_layers::Drop;

/* Compute units of the current device, asked for once. */
int compute_units(uint32_t *out, const char *call) {
    constexpr int kMost = 64;
    static std::atomic<uint32_t> known[kMost];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    uint32_t n = e == hipSuccess && dev >= 0 && dev < kMost ? known[dev].load(std::memory_order_relaxed) : 0;
    if (e == hipSuccess && n == 0) {
        int cus = 0;
        e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
        n = (uint32_t)cus;
        if (e == hipSuccess && dev >= 0 && dev < kMost) known[dev].store(n, std::memory_order_relaxed);
    }
    if (e != hipSuccess) {
        (void)hipGetLastError(); // reported here
        return done((int)e, call);
    }
    *out = n;
    return 0;
}

int key_of(const EriDropoutKey &k, Drop *d, const char *call) {
    if (!(k.p >= 0.0 && k.p <= 1.0)) return fail(ERI_ERR_ARG, call, "p is not between 0 and 1");
    if (!aligned(k.offset_ptr, 8)) return fail(ERI_ERR_ALIGN, call, "offset_ptr is not 8-byte aligned");
    d->seed = k.seed;
    d->offset = k.offset;
    d->offset_ptr = k.offset_ptr;
    d->below = (uint32_t)std::floor(k.p * 65536.0 + 0.5);
    d->scale = d->below < 65536 ? (float)(65536.0 / (65536.0 - d->below)) : 0.0f;
    return 0;
}

int ids_ok(const void *ids, int ids_64, uint64_t tokens, uint64_t vocab, uint64_t dim, const char *kCall) {
    ERI_NEED(ids || tokens == 0, ERI_ERR_NULL, "ids is NULL");
    ERI_NEED(ids_64 == 0 || ids_64 == 1, ERI_ERR_DTYPE, "ids_64 is neither 0 nor 1");
    ERI_NEED(aligned(ids, ids_64 ? 8 : 4), ERI_ERR_ALIGN, "ids are not aligned to their size");
    ERI_NEED(vocab != 0 && dim != 0, ERI_ERR_EMPTY, "a table without rows or columns");
    ERI_NEED(tokens <= kCountMost && vocab <= kCountMost && dim <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 tokens, rows or columns");
    return 0;
}

} // namespace

extern "C" {

int eri_embedding(const EriEmbedding *args, void *stream) {
    constexpr const char *kCall = "eri_embedding";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriEmbedding a = *args;
    if (int rc = ids_ok(a.ids, a.ids_64, a.tokens, a.vocab, a.dim, kCall)) return rc;
    ERI_NEED(floating(a.dtype_tag), ERI_ERR_DTYPE, "unsupported dtype tag (F32=0 and BF16=2 are supported)");
    ERI_NEED(stride(&a.table_stride, a.dim) && stride(&a.out_stride, a.dim), ERI_ERR_ARG, "a stride shorter than a row");
    if (a.tokens == 0) return 0;
    ERI_NEED(a.table && a.out, ERI_ERR_NULL, "table or out is NULL");
    ERI_NEED(aligned(a.table, size_of(a.dtype_tag)) && aligned(a.out, size_of(a.dtype_tag)), ERI_ERR_ALIGN, "table or out is not aligned to its elements");
    uint32_t cus;
    if (int rc = compute_units(&cus, kCall)) return rc;
    return done(eri_layers::launch_embedding(a, cus, stream), kCall);
}

int eri_embedding_grad_workspace(uint64_t tokens, uint64_t vocab, uint64_t dim, uint64_t *bytes) {
    constexpr const char *kCall = "eri_embedding_grad_workspace";
    ERI_NEED(bytes, ERI_ERR_NULL, "bytes is NULL");
    if (int rc = ids_ok(nullptr, 0, 0, vocab, dim, kCall)) return rc;
    ERI_NEED(tokens <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 tokens");
    *bytes = eri_layers::embedding_grad_workspace(tokens, vocab, dim);
    return 0;
}

int eri_embedding_grad(const EriEmbeddingGrad *args, void *stream) {
    constexpr const char *kCall = "eri_embedding_grad";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriEmbeddingGrad a = *args;
    if (int rc = ids_ok(a.ids, a.ids_64, a.tokens, a.vocab, a.dim, kCall)) return rc;
    ERI_NEED(floating(a.grad_dtype) && floating(a.out_dtype), ERI_ERR_DTYPE, "unsupported dtype tag (F32=0 and BF16=2 are supported)");
    ERI_NEED(stride(&a.grad_stride, a.dim) && stride(&a.out_stride, a.dim), ERI_ERR_ARG, "a stride shorter than a row");
    const uint64_t need = eri_layers::embedding_grad_workspace(a.tokens, a.vocab, a.dim);
    ERI_NEED((a.grad || a.tokens == 0) && a.out && (a.workspace || need == 0), ERI_ERR_NULL, "grad, out or workspace is NULL");
    ERI_NEED(aligned(a.grad, size_of(a.grad_dtype)) && aligned(a.out, size_of(a.out_dtype)), ERI_ERR_ALIGN, "grad or out is not aligned to its elements");
    ERI_NEED(aligned(a.workspace, 16), ERI_ERR_ALIGN, "workspace is not 16-byte aligned");
    ERI_NEED(a.workspace_bytes >= need, ERI_ERR_ARG, "workspace is too small");
    return done(eri_layers::launch_embedding_grad(a, stream), kCall);
}

int eri_dropout(const EriDropout *args, void *stream) {
    constexpr const char *kCall = "eri_dropout";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriDropout a = *args;
    Drop d;
    if (int rc = key_of(a.key, &d, kCall)) return rc;
    ERI_NEED(floating(a.dtype_tag), ERI_ERR_DTYPE, "unsupported dtype tag (F32=0 and BF16=2 are supported)");
    ERI_NEED(a.rows <= kCountMost && a.cols <= kStrideMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or 2^40 columns");
    ERI_NEED(stride(&a.x_stride, a.cols) && stride(&a.y_stride, a.cols), ERI_ERR_ARG, "a stride shorter than a row");
    if (a.rows == 0 || a.cols == 0) return 0;
    ERI_NEED(a.x && a.y, ERI_ERR_NULL, "x or y is NULL");
    ERI_NEED(aligned(a.x, size_of(a.dtype_tag)) && aligned(a.y, size_of(a.dtype_tag)), ERI_ERR_ALIGN, "x or y is not aligned to its elements");
    uint32_t cus;
    if (int rc = compute_units(&cus, kCall)) return rc;
    return done(eri_layers::launch_dropout(a, d, cus, stream), kCall);
}

int eri_rms_norm(const EriRmsNorm *args, void *stream) {
    constexpr const char *kCall = "eri_rms_norm";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriRmsNorm a = *args;
    Drop d;
    if (int rc = key_of(a.key, &d, kCall)) return rc;
    ERI_NEED(floating(a.x_dtype) && (!a.residual || floating(a.residual_dtype)) && (!a.weight || floating(a.weight_dtype)), ERI_ERR_DTYPE,
             "unsupported dtype tag (F32=0 and BF16=2 are supported)");
    ERI_NEED(floating(a.y_dtype) || a.y_dtype == ERI_DTYPE_F8E4M3, ERI_ERR_DTYPE, "unsupported dtype tag of y (F32=0, BF16=2 and F8E4M3=16 are supported)");
    ERI_NEED(a.scale_group == 0 || (a.scale_group == 128 && a.y_dtype == ERI_DTYPE_F8E4M3), ERI_ERR_ARG, "scale_group is 0, or 128 with an 8-bit output");
    ERI_NEED(a.eps >= 0.0f, ERI_ERR_ARG, "eps is negative or not a number");
    ERI_NEED(a.rows <= kCountMost && a.cols <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
    ERI_NEED(a.cols != 0, ERI_ERR_EMPTY, "rows without elements");
    ERI_NEED(stride(&a.x_stride, a.cols) && stride(&a.residual_stride, a.cols) && stride(&a.y_stride, a.cols) && stride(&a.h_stride, a.cols), ERI_ERR_ARG,
             "a stride shorter than a row");
    if (a.rows == 0) return 0;
    ERI_NEED(a.x && a.y, ERI_ERR_NULL, "x or y is NULL");
    ERI_NEED(a.scales || a.y_dtype != ERI_DTYPE_F8E4M3, ERI_ERR_NULL, "scales is NULL with an 8-bit output");
    const int h_dtype = a.residual ? a.residual_dtype : a.x_dtype;
    ERI_NEED(aligned(a.x, size_of(a.x_dtype)) && aligned(a.y, size_of(a.y_dtype)) && aligned(a.h, size_of(h_dtype)) && aligned(a.rstd, 4) && aligned(a.scales, 4) &&
                 (!a.residual || aligned(a.residual, size_of(a.residual_dtype))) && (!a.weight || aligned(a.weight, size_of(a.weight_dtype))),
             ERI_ERR_ALIGN, "an address is not aligned to its elements");
    return done(eri_layers::launch_rms_norm(a, d, stream), kCall);
}

int eri_rms_norm_grad_workspace(uint64_t rows, uint64_t cols, uint64_t *bytes) {
    constexpr const char *kCall = "eri_rms_norm_grad_workspace";
    ERI_NEED(bytes, ERI_ERR_NULL, "bytes is NULL");
    ERI_NEED(rows <= kCountMost && cols <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
    ERI_NEED(cols != 0, ERI_ERR_EMPTY, "rows without elements");
    uint32_t cus;
    if (int rc = compute_units(&cus, kCall)) return rc;
    *bytes = eri_layers::rms_norm_grad_workspace(rows, cols, cus);
    return 0;
}

int eri_rms_norm_grad(const EriRmsNormGrad *args, void *stream) {
    constexpr const char *kCall = "eri_rms_norm_grad";
    ERI_NEED(args, ERI_ERR_NULL, "args is NULL");
    EriRmsNormGrad a = *args;
    Drop d;
    if (int rc = key_of(a.key, &d, kCall)) return rc;
    ERI_NEED(floating(a.grad_dtype) && floating(a.h_dtype) && (!a.grad_x || floating(a.x_dtype)) && (!a.weight || floating(a.weight_dtype)) &&
                 (!a.grad_weight || floating(a.grad_weight_dtype)),
             ERI_ERR_DTYPE, "unsupported dtype tag (F32=0 and BF16=2 are supported)");
    ERI_NEED(a.rows <= kCountMost && a.cols <= kCountMost, ERI_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
    ERI_NEED(a.cols != 0, ERI_ERR_EMPTY, "rows without elements");
    ERI_NEED(stride(&a.grad_stride, a.cols) && stride(&a.h_stride, a.cols) && stride(&a.grad_h_stride, a.cols) && stride(&a.grad_x_stride, a.cols) &&
                 stride(&a.grad_residual_stride, a.cols),
             ERI_ERR_ARG, "a stride shorter than a row");
    ERI_NEED(a.rows == 0 || (a.grad && a.h && a.rstd), ERI_ERR_NULL, "grad, h or rstd is NULL");
    ERI_NEED(aligned(a.grad, size_of(a.grad_dtype)) && aligned(a.h, size_of(a.h_dtype)) && aligned(a.rstd, 4) && aligned(a.grad_h, size_of(a.h_dtype)) &&
                 aligned(a.grad_residual, size_of(a.h_dtype)) && (!a.grad_x || aligned(a.grad_x, size_of(a.x_dtype))) &&
                 (!a.weight || aligned(a.weight, size_of(a.weight_dtype))) && (!a.grad_weight || aligned(a.grad_weight, size_of(a.grad_weight_dtype))),
             ERI_ERR_ALIGN, "an address is not aligned to its elements");
    uint32_t cus;
    if (int rc = compute_units(&cus, kCall)) return rc;
    if (a.grad_weight) {
        const uint64_t need = eri_layers::rms_norm_grad_workspace(a.rows, a.cols, cus);
        ERI_NEED(a.workspace || need == 0, ERI_ERR_NULL, "workspace is NULL");
        ERI_NEED(aligned(a.workspace, 16), ERI_ERR_ALIGN, "workspace is not 16-byte aligned");
        ERI_NEED(a.workspace_bytes >= need, ERI_ERR_ARG, "workspace is too small");
    }
    if ((a.rows == 0 || (!a.grad_x && !a.grad_residual)) && !a.grad_weight) return 0;
    return done(eri_layers::launch_rms_norm_grad(a, d, cus, stream), kCall);
}

} // extern "C"
