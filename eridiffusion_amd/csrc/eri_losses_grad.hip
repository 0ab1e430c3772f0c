/*
 * The logits' gradients of include/eri_losses.h: one pass that reads a row and writes a row.
 *
 *     scores        (g ([j = id] - p) - h p (ln p + H)) / T = p (u + w log2 p) + [j = id] g / T,  u = -(g + h H) / T,  w = -h ln 2 / T
 *     distillation  p_j / p_r (p_r - q_r) g / T for the tokens that the teacher does not name, written everywhere; the named ones,
 *                   (p_j - q_j) g / T, are computed by one wave before and put in their places afterwards
 * with log2 p = (x - m) log2(e) / T - log2 s in one fused product: one exponential an element, which is a quarter of the arithmetic.
 */
#include "eri_losses_device.h"

namespace eri_losses {
namespace {

struct GradArgs {
    const void *logits, *ids;
    const float *stats, *grad, *grad_entropy, *entropy;
    const void *teacher;
    void *out;
    uint64_t stride, out_stride, ids_stride, teacher_stride;
    uint32_t first, rows;
    uint32_t vocab, slices, per;
    uint32_t k, ids_64, teacher_f32;
    float c, inv_t;
};

template <typename T, typename O, int TPR, typename Of> __device__ __forceinline__ void each(const T *row, O *out, uint32_t first, uint32_t end, uint32_t vocab, uint32_t t, Of of) {
    const uint32_t whole = vocab / 8, last = end < whole ? end : whole;
    walk<TPR>(row, first, last, t, [&](auto &v, uint32_t at, bool full) {
        constexpr uint32_t C = sizeof v / sizeof v[0];
#pragma unroll
        for (uint32_t k = 0; k < C; ++k) {
            const uint32_t vec = at + k * TPR + t;
            of(v[k], vec * 8);
            if (full || k < C - 1 || vec < last) store_n(out + (uint64_t)vec * 8, 8, v[k]);
        }
    });
    if (end > whole && t == (whole - first) % TPR) {
        float v[8];
        load_last(v, row + (uint64_t)whole * 8, vocab % 8);
        of(v, whole * 8);
        store_n(out + (uint64_t)whole * 8, vocab % 8, v);
    }
}
template <typename O, int TPR> __device__ __forceinline__ void zeros(O *out, uint32_t first, uint32_t end, uint32_t vocab, uint32_t t) {
    const float v[8] = {};
    const uint32_t whole = vocab / 8, last = end < whole ? end : whole;
    for (uint32_t at = first + t; at < last; at += TPR) store_n(out + (uint64_t)at * 8, 8, v);
    if (end > whole && t == (whole - first) % TPR) store_n(out + (uint64_t)whole * 8, vocab % 8, v);
}

/* log2 p of an element, from {m, ln s}: nothing is left of a row where ln s is minus infinity. */
struct LogP {
    float m, log2_s, c;
    __device__ __forceinline__ LogP(const float *stats, float c_) : m(stats[0]), c(c_) {
        log2_s = stats[1] == -kInf ? kInf : stats[1] * (float)kLog2e;
        if (stats[1] == -kInf) m = 0.0f;
    }
    __device__ __forceinline__ float operator()(float x) const { return fmaf(x - m, c, -log2_s); }
};

template <typename T, typename O, int TPR, bool ENT> __global__ __launch_bounds__(256) void token_grad_kernel(const GradArgs a) {
    constexpr uint32_t ROWS = 256 / TPR;
    const uint32_t t = threadIdx.x % TPR, slice = blockIdx.x % a.slices;
    const uint64_t index = a.first + (uint64_t)(blockIdx.x / a.slices) * ROWS + threadIdx.x / TPR;
    if (index >= a.rows) return;
    const uint32_t all = (a.vocab + 7) / 8, first = slice * a.per, end = all - first > a.per ? first + a.per : all;
    O *out = (O *)a.out + index * a.out_stride;
    int64_t id = -1;
    float g = 0.0f, h = 0.0f;
    if (a.grad) {
        id = id_at(a.ids, a.ids_64, index);
        if (id >= 0 && id < (int64_t)a.vocab) g = a.grad[index];
        else id = -1;
    }
    if (ENT) h = a.grad_entropy[index];
    if (g == 0.0f && h == 0.0f) return zeros<O, TPR>(out, first, end, a.vocab, t);
    const LogP log2p(a.stats + index * 2, a.c);
    const uint32_t named = g == 0.0f || log2p.log2_s == kInf ? ~0u : (uint32_t)id;
    const float u = -(ENT ? fmaf(h, log2p.log2_s == kInf ? 0.0f : a.entropy[index], g) : g) * a.inv_t, w = -h * kLn2 * a.inv_t, more = g * a.inv_t;
    each<T, O, TPR>((const T *)a.logits + index * a.stride, out, first, end, a.vocab, t, [&](float(&v)[8], uint32_t col) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const float l = log2p(v[e]), p = exp2_of(l);
            v[e] = p * (ENT ? fmaf(w, fmaxf(l, kFloor), u) : u);
        }
        const uint32_t there = named - col;
        if (there < 8)
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (e == there) v[e] += more;
    });
}

template <typename T, typename O, int TPR> __global__ __launch_bounds__(TPR) void distill_grad_kernel(const GradArgs a) {
    const uint32_t t = threadIdx.x, slice = blockIdx.x % a.slices;
    const uint64_t index = a.first + blockIdx.x / a.slices;
    const uint32_t all = (a.vocab + 7) / 8, first = slice * a.per, end = all - first > a.per ? first + a.per : all;
    const T *row = (const T *)a.logits + index * a.stride;
    O *out = (O *)a.out + index * a.out_stride;
    const float g = a.grad[index] * a.inv_t, *st = a.stats + index * 6;
    if (a.grad[index] == 0.0f || st[1] == -kInf) return zeros<O, TPR>(out, first, end, a.vocab, t);
    int32_t id = -1;
    float value = 0.0f;
    if (t < kWave) {
        float q = 0.0f;
        if (t < a.k) {
            const int64_t given = id_at(a.ids, a.ids_64, index * a.ids_stride + t);
            if (given >= 0 && given < (int64_t)a.vocab) id = (int32_t)given;
            if (id >= 0 && st[4] != -kInf) q = exp2_of((bf16_or_f32{a.teacher, a.teacher_f32 != 0}[index * a.teacher_stride + t] - st[4]) * (float)kLog2e);
        }
        float sum = 0.0f; // over the entries of the same token
        for (uint32_t j = 0; j < a.k; ++j)
            if (__builtin_amdgcn_readlane(id, (int)j) == id) sum += lane_of(q, (int)j);
        const bool here = id >= 0 && (uint32_t)id / 8 >= first && (uint32_t)id / 8 < end;
        if (here) {
            const LogP log2p(st, a.c);
            const float p = st[4] == -kInf ? 0.0f : exp2_of(log2p(at(row + id)));
            value = (p - sum) * g;
        } else id = -1;
    }
    __syncthreads(); // the named logits have been read, before out may be written over them
    const LogP log2r(st + 2, a.c);
    const float over = st[5] * g;
    each<T, O, TPR>(row, out, first, end, a.vocab, t, [&](float(&v)[8], uint32_t) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = exp2_of(log2r(v[e])) * over;
    });
    __syncthreads();
    if (id >= 0) {
        const float v[8] = {value};
        store_n(out + id, 1, v);
    }
}

constexpr uint32_t kBlocks = 1u << 23; // of a launch

/* Launches over parts of the rows, so that a launch can count its threads. */
template <typename F> int in_parts(GradArgs &a, uint64_t rows, uint32_t rows_of_block, F launch) {
    const uint64_t most = (uint64_t)(kBlocks / a.slices) * rows_of_block;
    for (uint64_t first = 0; first < rows; first += most) {
        a.first = (uint32_t)first;
        a.rows = (uint32_t)(rows - first < most ? rows : first + most);
        launch((uint32_t)((a.rows - a.first + rows_of_block - 1) / rows_of_block) * a.slices);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

template <typename T, typename O> int token_grad(GradArgs &a, uint64_t rows, hipStream_t s) {
#define ERI_GRAD(TPR, ENT) in_parts(a, rows, 256 / TPR, [&](uint32_t n) { hipLaunchKernelGGL((token_grad_kernel<T, O, TPR, ENT>), dim3(n), dim3(256), 0, s, a); })
    if (a.vocab <= 2048) return a.grad_entropy ? ERI_GRAD(64, true) : ERI_GRAD(64, false);
    return a.grad_entropy ? ERI_GRAD(256, true) : ERI_GRAD(256, false);
#undef ERI_GRAD
}
template <typename T, typename O> int distill_grad(GradArgs &a, uint64_t rows, hipStream_t s) {
#define ERI_GRAD(TPR) in_parts(a, rows, 1, [&](uint32_t n) { hipLaunchKernelGGL((distill_grad_kernel<T, O, TPR>), dim3(n), dim3(TPR), 0, s, a); })
    return a.vocab <= 2048 ? ERI_GRAD(64) : ERI_GRAD(256);
#undef ERI_GRAD
}
void cut(GradArgs &a, uint64_t rows, uint32_t per) {
    const uint32_t n = (a.vocab + 7) / 8;
    a.per = rows >= 1024 ? n : per;
    if (a.per > n) a.per = n;
    a.slices = (n + a.per - 1) / a.per;
    if (a.slices > kBlocks) a.per = n, a.slices = 1;
}

} // namespace

int launch_token_logprobs_grad(const EriTokenLogprobsGrad &e, void *stream) {
    GradArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.stats = e.stats, a.grad = e.grad, a.grad_entropy = e.grad_entropy, a.entropy = e.entropy, a.out = e.out;
    a.stride = e.logits_stride, a.out_stride = e.out_stride, a.vocab = (uint32_t)e.vocab, a.ids_64 = (uint32_t)e.ids_64;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
    cut(a, e.rows, 1024);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = e.dtype_tag == ERI_DTYPE_F32, out_f32 = e.out_dtype == ERI_DTYPE_F32;
    if (f32) return out_f32 ? token_grad<float, float>(a, e.rows, s) : token_grad<float, bf16>(a, e.rows, s);
    return out_f32 ? token_grad<bf16, float>(a, e.rows, s) : token_grad<bf16, bf16>(a, e.rows, s);
}

int launch_distill_top_grad(const EriDistillTopGrad &e, void *stream) {
    GradArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.teacher = e.teacher, a.stats = e.stats, a.grad = e.grad, a.out = e.out;
    a.stride = e.logits_stride, a.out_stride = e.out_stride, a.ids_stride = e.ids_stride, a.teacher_stride = e.teacher_stride;
    a.vocab = (uint32_t)e.vocab, a.k = (uint32_t)e.k, a.ids_64 = (uint32_t)e.ids_64, a.teacher_f32 = e.teacher_dtype == ERI_DTYPE_F32;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
    cut(a, e.rows, 4096);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = e.dtype_tag == ERI_DTYPE_F32, out_f32 = e.out_dtype == ERI_DTYPE_F32;
    if (f32) return out_f32 ? distill_grad<float, float>(a, e.rows, s) : distill_grad<float, bf16>(a, e.rows, s);
    return out_f32 ? distill_grad<bf16, float>(a, e.rows, s) : distill_grad<bf16, bf16>(a, e.rows, s);
}

} // namespace eri_losses
