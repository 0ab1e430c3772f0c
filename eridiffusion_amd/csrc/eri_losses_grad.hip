/*
 * The logits' gradients of include/eri_losses.h: one pass that reads a row and writes a row.
 *
 *     scores        (g ([j = id] - p) - h p (ln p + H)) / T = p (u + w log2 p) + [j = id] g / T,  u = -(g + h H) / T,  w = -h ln 2 / T
 *     distillation  p_j / p_r (p_r - q_r) g / T for the tokens that the teacher does not name, (p_j - q_j) g / T for those it names, which each workgroup
 *                   marks in LDS before it begins: which elements of a vector, and by which entry, so that a token costs two looks at LDS and not one
 *                   at every entry (1025 x 10007 f32 with 64 tokens 25.1 us, so 17.1)
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

#define ERI_PUT(TYPE, P, ...) \
    do { \
        if (ONCE) __builtin_nontemporal_store(__VA_ARGS__, (TYPE *)(P)); \
        else *(TYPE *)(P) = __VA_ARGS__; \
    } while (0)
template <bool ONCE> __device__ __forceinline__ void store_whole(float *p, const float (&v)[4]) { ERI_PUT(u32x4_at4, p, u32x4{as_bits(v[0]), as_bits(v[1]), as_bits(v[2]), as_bits(v[3])}); }
template <bool ONCE> __device__ __forceinline__ void store_whole(float *p, const float (&v)[8]) {
    ERI_PUT(u32x4_at4, p, u32x4{as_bits(v[0]), as_bits(v[1]), as_bits(v[2]), as_bits(v[3])});
    ERI_PUT(u32x4_at4, p + 4, u32x4{as_bits(v[4]), as_bits(v[5]), as_bits(v[6]), as_bits(v[7])});
}
template <bool ONCE> __device__ __forceinline__ void store_whole(bf16 *p, const float (&v)[4]) { ERI_PUT(u32x2_at2, p, u32x2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])}); }
template <bool ONCE> __device__ __forceinline__ void store_whole(bf16 *p, const float (&v)[8]) {
    ERI_PUT(u32x4_at2, p, u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])});
}
#undef ERI_PUT
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16 *p, float v) { p->bits = (uint16_t)bf16_pair(v, 0.0f); }

/* A vector of the gradient, where the row's vector lies; `out` is its beginning, taken down as the row's. */
template <bool ONCE, typename T, typename O, int E> __device__ __forceinline__ void store_any(O *out, const Row<T> &row, uint32_t vec, uint32_t end, const float (&v)[E]) {
    if (vec >= end) return;
    if (vec >= row.whole_from() && vec < row.whole_to()) store_whole<ONCE>(out + (uint64_t)vec * E, v);
    else
#pragma unroll
        for (uint32_t e = 0; e < (uint32_t)E; ++e)
            if (row.has(vec, e)) store_one(out + (uint64_t)vec * E + e, v[e]);
}
enum Past { kNothing, kStores, kBoth }; // what passes the caches by

template <int TPR, Past PAST, typename T, typename O, typename Of> __device__ __forceinline__ void each(const Row<T> &row, O *out, uint32_t first, uint32_t end, uint32_t t, Of of) {
    walk<TPR, PAST == kBoth>(row, first, end, t, [&](auto &v, uint32_t at, bool full) {
#pragma unroll
        for (uint32_t k = 0; k < sizeof v / sizeof v[0]; ++k) {
            const uint32_t vec = at + k * TPR + t;
            of(v[k], vec * kEach<T>);
            if (full) store_whole<PAST != kNothing>(out + (uint64_t)vec * kEach<T>, v[k]);
            else store_any<PAST != kNothing>(out, row, vec, end, v[k]);
        }
    });
}
template <int TPR, bool ONCE, typename T, typename O> __device__ __forceinline__ void zeros(const Row<T> &row, O *out, uint32_t first, uint32_t end, uint32_t t) {
    const float v[kEach<T>] = {};
    for (uint32_t vec = first + t; vec < end; vec += TPR) store_any<ONCE>(out, row, vec, end, v);
}

/* Below any log2 p whose p is not 0: it keeps 0 * minus infinity out of p log2 p.  w kLeast is finite for all w below 2^120, where kFloor, which is for differences
 * of logits, made infinity of it, and NaN of a masked element, from |grad_entropy| / T of 4.9e10 on. */
constexpr float kLeast = -256.0f;

/* log2 p of an element, from {m, ln s}: nothing is left of a row where ln s is minus infinity. */
struct LogP {
    float m, log2_s, c;
    __device__ __forceinline__ LogP(const float *stats, float c_) : c(c_) {
        const float first = stats[0], log_s = stats[1];
        m = log_s == -kInf ? 0.0f : first;
        log2_s = log_s == -kInf ? kInf : log_s * (float)kLog2e;
    }
    __device__ __forceinline__ float operator()(float x) const { return fmaf(x - m, c, -log2_s); }
};

template <typename T, typename O, int TPR, bool ENT, Past PAST> __global__ __launch_bounds__(256) void token_grad_kernel(const GradArgs a) {
    constexpr uint32_t ROWS = 256 / TPR;
    const uint32_t t = threadIdx.x % TPR, slice = blockIdx.x % a.slices;
    const uint64_t index = a.first + (uint64_t)(blockIdx.x / a.slices) * ROWS + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / TPR));
    if (index >= a.rows) return;
    const Row<T> row((const T *)a.logits + index * a.stride, a.vocab);
    const uint32_t all = row.vectors(), first = slice * a.per < all ? slice * a.per : all, end = all - first > a.per ? first + a.per : all;
    O *out = (O *)a.out + index * a.out_stride - row.skip;
    // all that is known of the row is asked for at once, not one after the other
    const int64_t id = a.grad ? id_at(a.ids, a.ids_64, index) : -1;
    float g = a.grad ? a.grad[index] : 0.0f;
    const float h = ENT ? a.grad_entropy[index] : 0.0f, entropy = ENT ? a.entropy[index] : 0.0f;
    const LogP log2p(a.stats + index * 2, a.c);
    if (id < 0 || id >= (int64_t)a.vocab) g = 0.0f;
    if (g == 0.0f && h == 0.0f) return zeros<TPR, PAST != kNothing>(row, out, first, end, t);
    const uint32_t named = g == 0.0f || log2p.log2_s == kInf ? ~0u : row.skip + (uint32_t)id;
    const float u = -(ENT ? fmaf(h, log2p.log2_s == kInf ? 0.0f : entropy, g) : g) * a.inv_t, w = -h * kLn2 * a.inv_t, more = g * a.inv_t;
    each<TPR, PAST>(row, out, first, end, t, [&](float(&v)[kEach<T>], uint32_t place) {
#pragma unroll
        for (uint32_t e = 0; e < kEach<T>; ++e) {
            const float l = log2p(v[e]), p = exp2_of(l);
            v[e] = p * (ENT ? fmaf(w, fmaxf(l, kLeast), u) : u);
        }
        const uint32_t there = named - place;
        if (there < kEach<T>)
#pragma unroll
            for (uint32_t e = 0; e < kEach<T>; ++e)
                if (e == there) v[e] += more;
    });
}

constexpr uint32_t kDistillMost = 4096; // vectors of a row or slice

template <typename T, typename O, int TPR, Past PAST> __global__ __launch_bounds__(TPR) void distill_grad_kernel(const GradArgs a) {
    constexpr uint32_t MOST = TPR > (int)kWave ? kDistillMost : kDistillMost / 4;
    __shared__ uint32_t named[MOST / 4]; // a byte for each vector: which of its elements the teacher names
    __shared__ uint8_t entries[MOST];    // and one of the entries that name it
    __shared__ uint32_t places[kWave];
    __shared__ float shares[kWave]; // of a token: all its entries
    const uint32_t t = threadIdx.x, slice = blockIdx.x % a.slices;
    const uint64_t index = a.first + blockIdx.x / a.slices;
    const Row<T> row((const T *)a.logits + index * a.stride, a.vocab);
    const uint32_t all = row.vectors(), first = slice * a.per < all ? slice * a.per : all, end = all - first > a.per ? first + a.per : all;
    O *out = (O *)a.out + index * a.out_stride - row.skip;
    const float given = a.grad[index], g = given * a.inv_t, *st = a.stats + index * 6, norm = st[4], over = st[5] * g;
    int64_t id = -1;
    float q = 0.0f;
    if (t < a.k) {
        id = id_at(a.ids, a.ids_64, index * a.ids_stride + t);
        q = bf16_or_f32{a.teacher, a.teacher_f32 != 0}[index * a.teacher_stride + t];
    }
    const LogP log2p(st, a.c), log2r(st + 2, a.c);
    if (given == 0.0f || st[1] == -kInf) return zeros<TPR, PAST != kNothing>(row, out, first, end, t);
    for (uint32_t i = t; i < (end - first + 3) / 4; i += TPR) named[i] = 0;
    const uint32_t place = row.skip + (uint32_t)id, vec = place / kEach<T> - first;
    const bool here = id >= 0 && id < (int64_t)a.vocab && place / kEach<T> >= first && place / kEach<T> < end;
    __syncthreads();
    if (t < kWave) {
        q = here && norm != -kInf ? exp2_of((q - norm) * (float)kLog2e) : 0.0f;
        const uint32_t mine = here ? place : ~0u, bit = 1u << (vec % 4 * 8 + place % kEach<T>);
        float share = q;
        if (__ballot(here && (atomicOr(&named[vec / 4], bit) & bit)) != 0) { // a token twice
            share = 0.0f;
            for (uint32_t j = 0; j < a.k; ++j)
                if ((uint32_t)__builtin_amdgcn_readlane((int)mine, (int)j) == mine) share += lane_of(q, (int)j);
        }
        if (here) entries[vec] = (uint8_t)t;
        places[t] = mine;
        shares[t] = share;
    }
    __syncthreads();
    each<TPR, PAST>(row, out, first, end, t, [&](float(&v)[kEach<T>], uint32_t from) {
        float r[kEach<T>];
#pragma unroll
        for (uint32_t e = 0; e < kEach<T>; ++e) r[e] = exp2_of(log2r(v[e])) * over;
        uint32_t which = from / kEach<T> < end ? ((const uint8_t *)named)[from / kEach<T> - first] : 0;
        for (; which != 0; which &= which - 1) {
            const uint32_t e = (uint32_t)__builtin_ctz(which);
            uint32_t j = entries[from / kEach<T> - first];
            if (places[j] != from + e) // the vector holds another token of the teacher's too
                for (j = 0; j + 1 < kWave && places[j] != from + e;) ++j;
            const float share = shares[j];
            float x = v[0];
#pragma unroll
            for (uint32_t i = 1; i < kEach<T>; ++i) x = i == e ? v[i] : x;
            const float value = ((norm == -kInf ? 0.0f : exp2_of(log2p(x))) - share) * g;
#pragma unroll
            for (uint32_t i = 0; i < kEach<T>; ++i) r[i] = i == e ? value : r[i];
        }
#pragma unroll
        for (uint32_t e = 0; e < kEach<T>; ++e) v[e] = r[e];
    });
}

constexpr uint32_t kBlocks = 1u << 23; // of a launch

/* Cuts rows into slices; whether the logits are more than half of the last cache.  A small part of a row to each workgroup keeps the chip within one
 * window of the memory, and what is stored, and for float32 scores what is read too, passes the caches by.  us with 2048, 1024 and 512
 * vectors to a workgroup, both past the caches, and (the stores alone):
 *     scores        8192 x 128000 bf16     768 (785)  758 (749)  726 (892)      distillation  (775)      665 (647)  782 (899)
 *                  16384 x 32000           371 (383)  370 (330)  358 (425)                    (380)          (345)      (487)
 *                  16384 x 50257           624 (628)  538 (510)  599 (659)                    (646)          (545)      (778)
 *                   4096 x 128000 f32      763 (784)  708 (776)  684 (700)                752 (770)      697 (729)  760 (828)
 *                  16384 x 32000 f32                                                      758            700 (655)  815 (897)
 * before, with a row to a workgroup and all of it through the caches, 8192 x 128000 took 817 and 842.  A float32 gradient of bf16 logits goes through the
 * caches at any size: a lane's eight elements are two stores, which leave gaps for one another, and only the caches put them together.  4096 x 128000 595 us, past
 * them 804, distillation 540 and 833; 8192 x 50257 462 and 592, 416 and 429. */
template <typename T, typename O> bool cut(GradArgs &a, uint64_t rows, uint32_t per, uint32_t per_large) {
    const uint32_t n = vectors_most<T>(a.vocab);
    const bool large = sizeof(O) <= sizeof(T) && rows * a.vocab * sizeof(T) > kCache;
    a.per = large ? per_large : per;
    if (a.per > n) a.per = n;
    a.slices = (n + a.per - 1) / a.per;
    return large;
}

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

/* Whether a wave has a row: short ones, and longer ones where there are many: 16384 x 3000 bf16 35 us for 51, and 44 for 61 (scores, distillation), 6000 75
 * for 77, and 80 for 90; 200 x 6000 5.1 for 7.1. */
template <typename T> bool by_waves(uint64_t vocab, uint64_t rows, uint32_t many) {
    const uint32_t n = vectors_most<T>(vocab);
    return n <= 256 || (rows >= 1024 && n <= many);
}

/* LDS to ask for beyond what a workgroup of 256 uses, so that no more than `groups` of them fit a unit's 160 KB, or none.  Fewer rows' pieces under way at once
 * leave the memory's channels less to jump between, where rows are long, begin together on 128 bytes and are many.  By their registers the scores' kernels fit 4
 * workgroups to a unit (bf16 without entropy, 117 registers), 5 (with entropy, 82) and 8 (f32, 52), the distillation's 4 (f32, 106).  us with those and with
 * `groups`, for a gradient of its own and (over the logits):
 *     scores, bf16, entropy, 4     65536 x 8192    461 505 (467 511)   21845 x 24576   368 375 (360 368)   16777 x 32000   379 343 (406 342)
 *                                   8388 x 128000  779 741 (827 761)    5336 x 50304   174 170 (179 173)    2668 x 50304  78.3 76.6 (86.0 90.5)
 *     scores, bf16, 3               9362 x 57344   360 373 (346 362)    7281 x 73728   378 356 (390 372)    4194 x 128000  380 354 (399 348)
 *                                   8388 x 128000  756 694 (813 693)    2097 x 128000  183 182 (192 178)    1365 x 196608  176 188 (175 182)
 *     distillation, f32, 3          5041 x 106496  682 687 (728 706)    4369 x 122880  708 690 (743 703)    2097 x 128000  361 349 (395 357)
 *                                   4194 x 128000  739 692 (816 709)    1048 x 128000  179 180 (187 186)     819 x 163840  175 176 (175 181)
 * Not asked for by scores of f32, with 4 (53649 x 10007 692 819, 4194 x 128000 694 713, 4369 x 122880 723 708); bf16 gradients of f32, 4194 x 128000, the scores' with 4 (538 686) and the
 * distillation's with 3 (521 582); distillation of bf16, with 3 (8388 x 128000 670 727); rows that begin anywhere (8192 x 128001 bf16 753 795).  Where the gradient's
 * rows begin does not matter: 8 elements off, 8388 x 128000 bf16 803 704. */
constexpr uint32_t room_for(uint32_t groups, uint32_t used = 0) { return 160 * 1024 / (groups + 1) + 512 - used; }
template <typename T> bool long_and_even(const GradArgs &a, uint64_t rows, uint64_t cols, uint64_t bytes) {
    return a.vocab >= cols && rows * a.vocab * sizeof(T) >= bytes && ((uintptr_t)a.logits | a.stride * sizeof(T)) % 128 == 0;
}
template <typename T, typename O> int token_grad(GradArgs &a, uint64_t rows, hipStream_t s) {
#define ERI_GRAD(TPR, ENT, PAST) in_parts(a, rows, 256 / TPR, [&](uint32_t n) { hipLaunchKernelGGL((token_grad_kernel<T, O, TPR, ENT, PAST>), dim3(n), dim3(256), lds, s, a); })
    constexpr bool kWide = sizeof(T) == 4;
    uint32_t lds = 0;
    const bool large = cut<T, O>(a, rows, kBatch * 256, kWide ? 512 : kBatch * 256);
    if (by_waves<T>(a.vocab, rows, 512)) {
        a.per = vectors_most<T>(a.vocab), a.slices = 1;
        if (large) return a.grad_entropy ? ERI_GRAD(64, true, kStores) : ERI_GRAD(64, false, kStores);
        return a.grad_entropy ? ERI_GRAD(64, true, kNothing) : ERI_GRAD(64, false, kNothing);
    }
    if (large && !kWide) {
        if (a.grad_entropy && long_and_even<T>(a, rows, 31 << 10, 1ull << 29)) lds = room_for(4);
        if (!a.grad_entropy && long_and_even<T>(a, rows, 72 << 10, 1ull << 30)) lds = room_for(3);
    }
    if (!large) return a.grad_entropy ? ERI_GRAD(256, true, kNothing) : ERI_GRAD(256, false, kNothing);
    return a.grad_entropy ? ERI_GRAD(256, true, (kWide ? kBoth : kStores)) : ERI_GRAD(256, false, (kWide ? kBoth : kStores));
#undef ERI_GRAD
}
template <typename T, typename O> int distill_grad(GradArgs &a, uint64_t rows, hipStream_t s) {
#define ERI_GRAD(TPR, PAST) in_parts(a, rows, 1, [&](uint32_t n) { hipLaunchKernelGGL((distill_grad_kernel<T, O, TPR, PAST>), dim3(n), dim3(TPR), lds, s, a); })
    uint32_t lds = 0;
    // looking up the teacher's tokens costs each workgroup something: longer slices, unless the rows are few
    const bool large = cut<T, O>(a, rows, rows >= 1024 && vectors_most<T>(a.vocab) <= kDistillMost ? kDistillMost : kBatch * 256, kBatch * 256);
    if (by_waves<T>(a.vocab, rows, large ? kDistillMost * 3 / 16 : kDistillMost / 4)) { // large ones, 64 tokens: 65536 x 4000 bf16 202 us for 309, x 6000 300 for 343, but x 8000 412 for 379
        a.per = vectors_most<T>(a.vocab), a.slices = 1;
        return large ? ERI_GRAD(64, kStores) : ERI_GRAD(64, kNothing);
    }
    if (large && sizeof(T) == 4 && sizeof(O) == 4 && long_and_even<T>(a, rows, 120 << 10, 1ull << 30)) lds = room_for(3, kDistillMost * 2);
    return large ? ERI_GRAD(256, kStores) : ERI_GRAD(256, kNothing);
#undef ERI_GRAD
}
} // namespace

int launch_token_logprobs_grad(const EriTokenLogprobsGrad &e, void *stream) {
    GradArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.stats = e.stats, a.grad = e.grad, a.grad_entropy = e.grad_entropy, a.entropy = e.entropy, a.out = e.out;
    a.stride = e.logits_stride, a.out_stride = e.out_stride, a.vocab = (uint32_t)e.vocab, a.ids_64 = (uint32_t)e.ids_64;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = e.dtype_tag == ERI_DTYPE_F32, out_f32 = e.out_dtype == ERI_DTYPE_F32;
    if (f32) return out_f32 ? distill_grad<float, float>(a, e.rows, s) : distill_grad<float, bf16>(a, e.rows, s);
    return out_f32 ? distill_grad<bf16, float>(a, e.rows, s) : distill_grad<bf16, bf16>(a, e.rows, s);
}

} // namespace eri_losses
