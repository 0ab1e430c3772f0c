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
    uint32_t vocab, slices, per;
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

/* One wave: `o` are the sums over the row, or with REST over what the teacher does not name. */
template <typename T, bool REST> __device__ __forceinline__ void finish(const DistillArgs &a, uint64_t row, Sums o, int32_t id, float x, float teacher, uint32_t lane) {
    const bool used = id >= 0;
    // the teacher: the log of the sum of its probabilities
    const bool some = used && !(teacher == -kInf); // NaN too
    const bool has = __ballot(some) != 0;
    float most = some ? teacher : -kInf;
#pragma unroll
    for (int d = 1; d < (int)kWave; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    if (most == -kInf) most = 0.0f; // nothing, or nothing but NaN
    const double weight = wave_sum(some ? exp((double)teacher - most) : 0.0);
    double norm = has ? (double)most + log(weight) : -(double)kInf;
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
    if (apart && norm <= 0.0) norm = 0.0;
    const double q = !some ? 0.0 : exp((double)teacher - norm);
    double loss = wave_sum(q == 0.0 ? 0.0 : q * ((double)teacher - norm - logp)), over = has ? 1.0 : 0.0;
    if (norm != norm) over = norm;
    if (apart) {
        const double total = wave_sum(q), left = 1.0 - total, qr = left < 0.0 ? 0.0 : left;
        // the log of what is left, from what is held where that is the smaller part
        const double log_r = held < 0.5 ? log1p(-held) : ((double)o.m - all.m) * inv_t + log((double)o.s) - log_s;
        loss += qr == 0.0 ? 0.0 : qr * (log(qr) - log_r);
        over = held < 0.5 ? total - held : exp(log_r) - qr;
    } else o = all;
    if (lane != 0) return;
    a.loss[row] = (float)loss;
    float *st = a.stats + row * 6;
    st[0] = none ? -kInf : all.m;
    st[1] = (float)log_s;
    st[2] = none ? -kInf : o.m;
    st[3] = apart ? (float)log((double)o.s) : (float)log_s;
    st[4] = (float)norm;
    st[5] = (float)over;
}

template <typename T, int TPR, bool REST, bool SPLIT> __global__ __launch_bounds__(TPR) void distill_kernel(const DistillArgs a) {
    constexpr int WAVES = TPR / (int)kWave;
    constexpr uint32_t kTurns = TPR > 256 ? 32 : 64, kSegment = kTurns * TPR; // vectors whose bits a thread holds at a time
    __shared__ Sums slots[WAVES];
    __shared__ uint32_t named[REST ? kSegment / 4 : 1], hits[REST ? 2 * TPR : 1];
    const uint32_t t = threadIdx.x, slice = SPLIT ? blockIdx.x % a.slices : 0;
    const uint64_t index = a.first + (SPLIT ? blockIdx.x / a.slices : blockIdx.x);
    const T *row = (const T *)a.logits + index * a.stride;
    const uint32_t whole = a.vocab / 8, all = (a.vocab + 7) / 8;
    const uint32_t first = SPLIT ? slice * a.per : 0, end = SPLIT && all - first > a.per ? first + a.per : all;
    int32_t id = -1;
    float x = -kInf, teacher = -kInf;
    if (t < kWave && (REST || !SPLIT)) {
        id = entry_of(a, index, t);
        if (!SPLIT && id >= 0) {
            x = at(row + id);
            teacher = bf16_or_f32{a.teacher, a.teacher_f32 != 0}[index * a.teacher_stride + t];
        }
    }
    Sums r = {kLowest, 0.0f, 0.0f};
    for (uint32_t begin = first; begin < end; begin += REST ? kSegment : end - first) {
        const uint32_t stop = REST && end - begin > kSegment ? begin + kSegment : end, last = stop < whole ? stop : whole;
        uint64_t mine = 0;
        if (REST) {
            const uint32_t vec = (uint32_t)id / 8 - begin; // of the segment
            const bool here = id >= 0 && (uint32_t)id / 8 >= begin && (uint32_t)id / 8 < stop;
            hits[t] = hits[TPR + t] = 0;
            if (here) ((uint8_t *)named)[vec] = 0;
            __syncthreads();
            if (here) {
                atomicOr(&named[vec / 4], 1u << (vec % 4 * 8 + (uint32_t)id % 8));
                atomicOr(&hits[vec / TPR / 32 * TPR + vec % TPR], 1u << (vec / TPR % 32));
            }
            __syncthreads();
            mine = (uint64_t)hits[TPR + t] << 32 | hits[t];
        }
        auto leave_out = [&](float(&v)[8], uint32_t vec) { // vec of the segment
            const uint32_t which = ((const uint8_t *)named)[vec];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (which >> e & 1) v[e] = -kInf;
        };
        walk<TPR>(row, begin, last, t, [&](auto &v, uint32_t at, bool) {
            if (REST) {
                const uint32_t bits = (uint32_t)(mine >> ((at - begin) / TPR));
#pragma unroll
                for (uint32_t k = 0; k < sizeof v / sizeof v[0]; ++k)
                    if (bits >> k & 1) leave_out(v[k], at - begin + k * TPR + t); // the last, shorter vector has its turn below
            }
            add<false>(r, v, a.c);
        });
        if (stop > whole && t == (whole - begin) % TPR) { // the row's last vector, of less than eight elements
            float v[1][8];
            load_last(v[0], row + (uint64_t)whole * 8, a.vocab % 8);
            if (REST && (mine >> ((whole - begin) / TPR) & 1)) leave_out(v[0], whole - begin);
            add<false>(r, v, a.c);
        }
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

/* Slices of a row.  Rows that fill the chip by themselves are not cut. */
constexpr uint32_t kFill = 1024, kSlicesMost = 64;
uint32_t slices_most(uint64_t vocab) {
    const uint64_t n = (vocab + 7) / 8 / 512;
    return n < 1 ? 1 : n > kSlicesMost ? kSlicesMost : (uint32_t)n;
}
uint32_t slices_of(uint64_t rows, uint64_t vocab) {
    const uint64_t n = kFill / rows, most = slices_most(vocab);
    return n < 2 ? 1 : (uint32_t)(n < most ? n : most);
}

template <typename T, bool REST> void launch(const DistillArgs &a, hipStream_t s) {
    const uint32_t rows = a.rows - a.first;
    if (a.slices > 1) {
        hipLaunchKernelGGL((distill_kernel<T, 256, REST, true>), dim3(rows * a.slices), dim3(256), 0, s, a);
        hipLaunchKernelGGL((distill_join_kernel<T, REST>), dim3(rows), dim3(64), 0, s, a);
    } else if (a.vocab <= 2048) hipLaunchKernelGGL((distill_kernel<T, 64, REST, false>), dim3(rows), dim3(64), 0, s, a);
    else hipLaunchKernelGGL((distill_kernel<T, 256, REST, false>), dim3(rows), dim3(256), 0, s, a);
}

} // namespace

uint64_t distill_top_workspace(uint64_t rows, uint64_t vocab) {
    const uint64_t most = slices_most(vocab), parts = rows * most < kFill ? rows * most : kFill;
    return most > 1 ? parts * sizeof(Sums) : 0;
}

int launch_distill_top(const EriDistillTop &e, void *stream) {
    DistillArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.teacher = e.teacher, a.loss = e.loss, a.stats = e.stats, a.parts = (Sums *)e.workspace;
    a.stride = e.logits_stride, a.ids_stride = e.ids_stride, a.teacher_stride = e.teacher_stride;
    a.vocab = (uint32_t)e.vocab, a.k = (uint32_t)e.k, a.ids_64 = (uint32_t)e.ids_64, a.teacher_f32 = e.teacher_dtype == ERI_DTYPE_F32;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
    const uint32_t n = (a.vocab + 7) / 8, want = slices_of(e.rows, e.vocab);
    a.per = ((n + want - 1) / want + 255) / 256 * 256;
    a.slices = (n + a.per - 1) / a.per;
    hipStream_t s = static_cast<hipStream_t>(stream);
    constexpr uint32_t kMost = 1u << 21; // rows of a launch
    for (uint64_t first = 0; first < e.rows; first += kMost) {
        a.first = (uint32_t)first;
        a.rows = (uint32_t)(e.rows - first < kMost ? e.rows : first + kMost);
        if (e.dtype_tag == ERI_DTYPE_F32) e.rest ? launch<float, true>(a, s) : launch<float, false>(a, s);
        else e.rest ? launch<bf16, true>(a, s) : launch<bf16, false>(a, s);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

} // namespace eri_losses
