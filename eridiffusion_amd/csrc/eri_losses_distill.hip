/*
 * Distillation from a teacher's top tokens of include/eri_losses.h, forward: one pass over the row with a running softmax; where all other tokens are a
 * class of their own, it runs over these alone, and the teacher's few tokens are added at the end.
 *
 * What a class holds is never taken as a difference of two sums: with 64 tokens that hold all but 1e-6 the rest would keep one digit in
 * fp32, and its gradient too.  So the teacher's tokens are left out of the pass: each thread has a bit for each of its vectors that says
 * whether one of them is in it, and only then looks up, in a byte for each vector, which.  The few terms of the loss are joined in fp64 by one wave.
 */
#include "eri_losses_device.h"

namespace eri_losses {
namespace {

struct DistillArgs {
    const void *logits, *ids, *teacher;
    float *loss, *stats;
    Sums *parts;
    uint64_t stride, ids_stride, teacher_stride;
    uint32_t first, rows;
    uint32_t vocab, slices;
    uint32_t k, ids_64, teacher_f32;
    float c, inv_t;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < (int)kWave; d *= 2) v += __shfl_xor(v, d);
    return v;
}

/* The teacher's entry of a lane: its token, or -1 for none. */
__device__ __forceinline__ int32_t entry_of(const DistillArgs &a, uint64_t row, uint32_t lane) {
    if (lane >= a.k) return -1;
    const int64_t id = id_at(a.ids, a.ids_64, row * a.ids_stride + lane);
    return id >= 0 && id < (int64_t)a.vocab ? (int32_t)id : -1;
}

/* One wave: `o` are the sums over the row, or with REST over what the teacher does not name.  fp64 where two numbers that may all but cancel are
 * made: an exponential and a logarithm more or less for each row count where rows are short (16384 x 1000 with the rest 33.5 us with seven of them).  What the named
 * tokens hold and log1p of the two shares are single numbers, fp32: a unit or two in their last place. */
template <typename T, bool REST> __device__ __forceinline__ void finish(const DistillArgs &a, uint64_t row, Sums o, int32_t id, float x, float teacher, uint32_t lane) {
    const bool used = id >= 0;
    // the student: sums over the whole row, and what the named tokens hold of it, each token once
    Sums all = o;
    double held = 0.0;
    if (REST) {
        bool first = used;
        for (uint32_t j = 0; j + 1 < a.k; ++j)
            if (__builtin_amdgcn_readlane(id, (int)j) == id && j < lane) first = false;
        all.m = fmaxf(o.m, wave_most(used ? x : -kInf));
        const float share = first ? exp2_of((x - all.m) * a.c) : 0.0f, named = eri_layers::wave_sum(share);
        all.s = o.s * exp2_of((o.m - all.m) * a.c) + named;
        held = (double)named / (double)all.s;
    }
    const bool none = all.s == 0.0f, apart = REST && !(o.s == 0.0f);
    const double inv_t = a.inv_t, log_s = log((double)all.s);
    const double logp = !used || none ? -(double)kInf : ((double)x - all.m) * inv_t - log_s;
    // the teacher: its probabilities, their sum, and the log of what they are divided by
    const bool some = used && !(teacher == -kInf); // NaN too
    const bool has = __ballot(some) != 0;
    float most = wave_most(some ? teacher : -kInf);
    if (most == -kInf) most = 0.0f; // nothing, or nothing but NaN
    double q = some ? exp((double)teacher - most) : 0.0, total = wave_sum(q), norm = 0.0;
    const double size = apart ? exp((double)most) : 0.0;
    if (apart && total * size <= 1.0) q *= size, total *= size;
    else {
        norm = has ? (double)most + log(total) : -(double)kInf;
        if (some) q /= total;
        total = 1.0;
    }
    double loss = wave_sum(q == 0.0 ? 0.0 : q * ((double)teacher - norm - logp)), over = has ? norm == norm ? 1.0 : norm : 0.0, log_o = log_s;
    if (apart) {
        const double qr = 1.0 - total;
        log_o = log((double)o.s);
        // logs of what is left, from what is not where that is the smaller part
        const double log_r = held < 0.5 ? (double)log1pf((float)-held) : ((double)o.m - all.m) * inv_t + log_o - log_s;
        if (qr != 0.0) loss += qr * ((total < 0.5 ? (double)log1pf((float)-total) : log(qr)) - log_r);
        over = held < 0.5 ? total - held : exp(log_r) - qr;
        if (norm != norm) over = norm;
    } else o = all;
    if (lane != 0) return;
    a.loss[row] = (float)loss;
    float *st = a.stats + row * 6;
    st[0] = none ? -kInf : all.m;
    st[1] = (float)log_s;
    st[2] = none ? -kInf : o.m;
    st[3] = (float)log_o;
    st[4] = (float)norm;
    st[5] = (float)over;
}

constexpr uint32_t kSlice = kBatch * 256; // vectors

template <typename T, int TPR, bool REST, bool SPLIT, bool ONCE> __global__ __launch_bounds__(TPR) void distill_kernel(const DistillArgs a) {
    constexpr int WAVES = TPR / (int)kWave;
    constexpr uint32_t kTurns = TPR > 256 ? 32 : 64, kSegment = kTurns * TPR; // vectors whose bits a thread holds at a time
    __shared__ Sums slots[WAVES];
    __shared__ uint32_t named[REST ? kSegment / 4 : 1], hits[REST ? 2 * TPR : 1];
    const uint32_t t = threadIdx.x, slice = SPLIT ? blockIdx.x % a.slices : 0;
    const uint64_t index = a.first + (SPLIT ? blockIdx.x / a.slices : blockIdx.x);
    const Row<T> row((const T *)a.logits + index * a.stride, a.vocab);
    const uint32_t all = row.vectors(), first = SPLIT ? (slice * kSlice < all ? slice * kSlice : all) : 0, end = SPLIT && all - first > kSlice ? first + kSlice : all;
    int32_t id = -1;
    float x = -kInf, teacher = -kInf;
    if (t < kWave && (REST || !SPLIT)) {
        id = entry_of(a, index, t);
        if (!SPLIT && id >= 0) {
            x = at(row.from + row.skip + id);
            teacher = bf16_or_f32{a.teacher, a.teacher_f32 != 0}[index * a.teacher_stride + t];
        }
    }
    Sums r = {kLowest, 0.0f, 0.0f};
    for (uint32_t begin = first; begin < end; begin += REST ? kSegment : end - first) {
        const uint32_t stop = REST && end - begin > kSegment ? begin + kSegment : end;
        uint64_t mine = 0;
        if (REST) {
            const uint32_t place = row.skip + (uint32_t)id, vec = place / kEach<T> - begin; // of the segment
            const bool here = id >= 0 && place / kEach<T> >= begin && place / kEach<T> < stop;
            hits[t] = hits[TPR + t] = 0;
            if (here) ((uint8_t *)named)[vec] = 0;
            __syncthreads();
            if (here) {
                atomicOr(&named[vec / 4], 1u << (vec % 4 * 8 + place % kEach<T>));
                atomicOr(&hits[vec / TPR / 32 * TPR + vec % TPR], 1u << (vec / TPR % 32));
            }
            __syncthreads();
            mine = (uint64_t)hits[TPR + t] << 32 | hits[t];
        }
        walk<TPR, ONCE>(row, begin, stop, t, [&](auto &v, uint32_t at, bool) {
            if (REST) {
                const uint32_t bits = (uint32_t)(mine >> ((at - begin) / TPR));
#pragma unroll
                for (uint32_t k = 0; k < sizeof v / sizeof v[0]; ++k)
                    if (bits >> k & 1) {
                        const uint32_t which = ((const uint8_t *)named)[at - begin + k * TPR + t];
#pragma unroll
                        for (uint32_t e = 0; e < kEach<T>; ++e)
                            if (which >> e & 1) v[k][e] = -kInf;
                    }
            }
            add<false>(r, v, a.c);
        });
        if (REST) __syncthreads(); // the bytes have been read
    }
    group_join<false, WAVES>(r, a.c, slots);
    if (t >= kWave) return;
    if (SPLIT) {
        if (t == 0) a.parts[blockIdx.x] = r;
    } else finish<T, REST>(a, index, r, id, x, teacher, t);
}

/* Joins the slices of a row. */
template <typename T, bool REST> __global__ __launch_bounds__(64) void distill_join_kernel(const DistillArgs a) {
    const uint32_t lane = threadIdx.x;
    const uint64_t index = a.first + blockIdx.x;
    Sums r = {kLowest, 0.0f, 0.0f};
    if (lane < a.slices) r = a.parts[blockIdx.x * a.slices + lane];
    const int32_t id = entry_of(a, index, lane);
    float x = -kInf, teacher = -kInf;
    if (id >= 0) {
        x = at((const T *)a.logits + index * a.stride + id);
        teacher = bf16_or_f32{a.teacher, a.teacher_f32 != 0}[index * a.teacher_stride + lane];
    }
    wave_join<false>(r, a.c);
    finish<T, REST>(a, index, r, id, x, teacher, lane);
}

uint32_t slices_of(uint64_t vectors) { return (uint32_t)((vectors + kSlice - 1) / kSlice); }

/* Threads to a row.  us for a call with 20 tokens, without and with the rest as a class:
 *                        256 threads              1024                     slices, joined
 *     1 row  of  4000 vectors    6.3  8.6            5.9  7.6                 7.9  8.0
 *    64          6250            7.4 10.5            6.7  9.5                 7.7  9.2
 *    64         16000           14.7 19.2           10.3 13.7                 8.1 10.6
 *   128         16000           15.5 20.0           11.2 14.3                11.0 13.5
 *   256         32000           21.5 25.9           21.8 24.4                24.1 26.6
 *   400         16000           19.4 23.6           21.7 25.6                23.0 25.5
 * and a wave to a row, bf16:
 * 16384 rows of  375 vectors   33.6 63.7, not 26.4 41.4;   750   43.0 74.1, 41.9 56.4;   1500   65.3 93.7, 76.6 86.0
 *   200          375            6.1  6.7       6.0  7.8;   1500    5.8  7.5,  7.1 10.9 */
template <typename T, bool REST> void launch(DistillArgs &a, uint64_t all_rows, hipStream_t s) {
    const uint32_t rows = a.rows - a.first, n = vectors_most<T>(a.vocab);
    const bool large = all_rows * a.vocab * sizeof(T) > kCache;
#define ERI_DISTILL(TPR, ONCE) hipLaunchKernelGGL((distill_kernel<T, TPR, REST, false, ONCE>), dim3(rows), dim3(TPR), 0, s, a)
    a.slices = slices_of(n);
    if (n > kLong && all_rows <= kFew && a.slices <= kSlicesMost) {
        hipLaunchKernelGGL((distill_kernel<T, 256, REST, true, false>), dim3(rows * a.slices), dim3(256), 0, s, a);
        hipLaunchKernelGGL((distill_join_kernel<T, REST>), dim3(rows), dim3(64), 0, s, a);
    } else if (n <= 256 || (all_rows >= 1024 && n <= (REST ? 2048 : 1024))) {
        if (large) ERI_DISTILL(64, true);
        else ERI_DISTILL(64, false);
    } else if (n > 2048 && all_rows <= 256) ERI_DISTILL(1024, false);
    else if (large) ERI_DISTILL(256, true);
    else ERI_DISTILL(256, false);
#undef ERI_DISTILL
}

} // namespace

uint64_t distill_top_workspace(uint64_t rows, uint64_t vocab) {
    const uint64_t n = vectors_most<float>(vocab), most = kSlicesMost * kSlice;
    return n > kLong ? (rows < kFew ? rows : kFew) * slices_of(n < most ? n : most) * sizeof(Sums) : 0;
}

int launch_distill_top(const EriDistillTop &e, void *stream) {
    DistillArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.teacher = e.teacher, a.loss = e.loss, a.stats = e.stats, a.parts = (Sums *)e.workspace;
    a.stride = e.logits_stride, a.ids_stride = e.ids_stride, a.teacher_stride = e.teacher_stride;
    a.vocab = (uint32_t)e.vocab, a.k = (uint32_t)e.k, a.ids_64 = (uint32_t)e.ids_64, a.teacher_f32 = e.teacher_dtype == ERI_DTYPE_F32;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
    hipStream_t s = static_cast<hipStream_t>(stream);
    constexpr uint32_t kMost = 1u << 21; // rows of a launch
    for (uint64_t first = 0; first < e.rows; first += kMost) {
        a.first = (uint32_t)first;
        a.rows = (uint32_t)(e.rows - first < kMost ? e.rows : first + kMost);
        if (e.dtype_tag == ERI_DTYPE_F32) e.rest ? launch<float, true>(a, e.rows, s) : launch<float, false>(a, e.rows, s);
        else e.rest ? launch<bf16, true>(a, e.rows, s) : launch<bf16, false>(a, e.rows, s);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

} // namespace eri_losses
