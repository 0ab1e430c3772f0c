/*
 * What the kernels of include/eri_losses.h share: the running softmax of a row of logits, and the largest of its elements as
 * sorted 64-bit keys, one to a lane.
 */
#pragma once
#include "../../include/eri_losses.h"
#include "eri_layers_device.h"

namespace eri_losses {

using namespace eri_layers;

constexpr float kInf = __builtin_inff();
constexpr float kLowest = -3.40282347e38f; // the running maximum before the first element: finite, so that its distance to minus infinity is no NaN
constexpr float kFloor = -1e28f;           // below any distance that counts: 0 * kFloor is 0 where 0 * -infinity would be NaN, and 2^31 of them are finite
/* Rows of more than kLong vectors are cut where there are no more than kFew of them. */
constexpr uint32_t kLong = 8192, kFew = 64, kSlicesMost = 64;
constexpr uint64_t kCache = 128u << 20;        // bytes, half of the last cache: the gradient wants room there too
constexpr double kLog2e = 1.4426950408889634074;
constexpr float kLn2 = 0.693147181f;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); } // one instruction, one unit in the last place

/* A row of logits in vectors of 16 bytes that begin at multiples of 128 bytes: `from` is the row's beginning, taken down to one, `skip` the elements that
 * lie before it there, so that a row begins anywhere inside of its vectors and ends anywhere.  Rows that begin at any other place are slower to
 * read in vectors from where they begin: 5600 x 50001 bf16 113 us, 50000 91, 49984, whose rows are multiples of 128 bytes, 83; from a multiple, 84 for all of them.
 * Of a vector that is not whole, the row's elements are read one by one, and nothing else: it may be written over
 * while the rows beside it are still wanted. */
template <typename T> constexpr uint32_t kEach = 16 / sizeof(T); // elements of a vector
template <typename T> struct Row {
    const T *from;
    uint32_t skip, cols;
    __device__ __forceinline__ Row(const T *row, uint32_t cols_) : cols(cols_) {
        skip = (uint32_t)((uintptr_t)row % 128 / sizeof(T));
        from = row - skip;
    }
    __device__ __forceinline__ uint32_t whole_from() const { return (skip + kEach<T> - 1) / kEach<T>; }
    __device__ __forceinline__ uint32_t whole_to() const { return (uint32_t)(((uint64_t)skip + cols) / kEach<T>); }
    __device__ __forceinline__ uint32_t vectors() const { return (uint32_t)(((uint64_t)skip + cols + kEach<T> - 1) / kEach<T>); }
    __device__ __forceinline__ bool has(uint32_t vec, uint32_t e) const { return vec * kEach<T> + e - skip < cols; }
    __device__ __forceinline__ uint32_t col(uint32_t vec, uint32_t e) const { return vec * kEach<T> + e - skip; }
};
/* Most vectors of a row of that many columns, wherever it begins. */
template <typename T> uint32_t vectors_most(uint64_t cols) { return (uint32_t)((cols + 128 / sizeof(T) - 1 + kEach<T> - 1) / kEach<T>); }

template <bool ONCE, typename T> __device__ __forceinline__ u32x4 load_whole(const Row<T> &row, uint32_t vec) {
    const u32x4 *p = (const u32x4 *)(row.from + (uint64_t)vec * kEach<T>);
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}
__device__ __forceinline__ void values_of(float (&v)[8], const u32x4 &a) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = as_float(e & 1 ? a[e / 2] & 0xffff0000u : a[e / 2] << 16);
}
__device__ __forceinline__ void values_of(float (&v)[4], const u32x4 &a) {
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) v[e] = as_float(a[e]);
}
__device__ __forceinline__ uint32_t bits_at(const bf16 *p) { return p->bits; }
__device__ __forceinline__ uint32_t bits_at(const float *p) { return *(const uint32_t *)p; }
template <typename T> __device__ __forceinline__ float at(const T *p) { return as_float(bits_at(p) << (sizeof(T) == 2 ? 16 : 0)); }
/* Any vector, minus infinity where the row has nothing. */
template <bool ONCE, typename T> __device__ __forceinline__ u32x4 load_any(const Row<T> &row, uint32_t vec) {
    constexpr uint32_t least = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
    u32x4 a = {least, least, least, least};
    if (vec >= row.whole_from() && vec < row.whole_to()) a = load_whole<ONCE>(row, vec);
    else
#pragma unroll
        for (uint32_t e = 0; e < kEach<T>; ++e)
            if (row.has(vec, e)) {
                const uint32_t u = bits_at(row.from + (uint64_t)vec * kEach<T> + e);
                if (sizeof(T) == 4) a[e] = u;
                else a[e / 2] = e & 1 ? (a[e / 2] & 0xffffu) | u << 16 : (a[e / 2] & 0xffff0000u) | u;
            }
    return a;
}

/* Vectors first .. end-1 of a row, dealt to TPR threads in turn, four of each at a time: all loads of a batch are under way before the first is
 * wanted.  `use(values, at, full)` gets an array of C vectors, those that begin at vector at + k TPR + t; unless `full`, some of them may not be whole
 * ones.  The row's end is one smaller batch: vector by vector it took a trip to memory for each.
 * ONCE: the loads pass the caches by, which pays where the logits are more than half of the last cache (kCache): read at 6.3-6.9 TB/s in place of
 * 5.6-5.9.  us for scores and gradient right behind what wrote the logits, not so and so: 41 MB 23 and 26, 131 MB 77 and 70, 150 MB 72 and 75, 164 MB 76 and
 * 68, 250 MB 134 and 124. */
template <int TPR, bool ONCE, int C, bool FULL, typename T, typename Use> __device__ __forceinline__ void walk_batch(const Row<T> &row, uint32_t at, uint32_t end, uint32_t t, Use &use) {
    u32x4 raw[C];
    float v[C][kEach<T>];
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const uint32_t vec = at + k * TPR + t;
        raw[k] = FULL ? load_whole<ONCE>(row, vec) : load_any<ONCE>(row, vec < end ? vec : ~0u / kEach<T>);
    }
#pragma unroll
    for (int k = 0; k < C; ++k) values_of(v[k], raw[k]);
    use(v, at, FULL);
}
constexpr uint32_t kBatch = 4;
template <int TPR, bool ONCE, typename T, typename Use> __device__ __forceinline__ void walk(const Row<T> &row, uint32_t first, uint32_t end, uint32_t t, Use use) {
    const uint32_t from = row.whole_from(), to = row.whole_to();
    for (uint32_t at = first; at < end;) {
        for (; at >= from && at + kBatch * TPR <= to && at + kBatch * TPR <= end; at += kBatch * TPR) walk_batch<TPR, ONCE, kBatch, true>(row, at, end, t, use);
        if (at >= end) break;
        const uint32_t left = (end - at + TPR - 1) / TPR;
        if (left == 1) walk_batch<TPR, ONCE, 1, false>(row, at, end, t, use);
        else if (left == 2) walk_batch<TPR, ONCE, 2, false>(row, at, end, t, use);
        else if (left == 3) walk_batch<TPR, ONCE, 3, false>(row, at, end, t, use);
        else walk_batch<TPR, ONCE, 4, false>(row, at, end, t, use);
        at += kBatch * TPR;
    }
}

/* The running softmax: m the largest logit, s the sum of exp((x - m) / T), t the sum of exp((x - m) / T) (x - m), whose terms are all
 * of one sign, so that the entropy ln s - t / (s T) loses nothing.  c = log2(e) / T.  Differences are taken before they are scaled: x c - m c in
 * one fused product would overflow for the lowest values of a type, which stand for masks, and round m c on the way. */
struct Sums {
    float m, s, t;
};
/* A NaN is passed over or returned, and makes the sums NaN either way.  fmaxf would first quiet each element in an instruction of its own, as it
 * does not know that they come from memory as they are: one in twelve of the loop's cycles. */
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
template <int E> __device__ __forceinline__ float largest(const float (&v)[E], float m) {
#pragma unroll
    for (int e = 0; e < E; e += 2) m = max3(v[e], v[e + 1], m);
    return m;
}
template <bool ENT> __device__ __forceinline__ void scale_to(Sums &a, float m, float c) { // m >= a.m
    const float d = a.m - m, f = exp2_of(d * c);
    if (ENT) a.t = f * fmaf(a.s, fmaxf(d, kFloor), a.t);
    a.s *= f;
    a.m = m;
}
template <bool ENT, int N, int E> __device__ __forceinline__ void add(Sums &a, const float (&v)[N][E], float c) {
    float m = a.m;
#pragma unroll
    for (int k = 0; k < N; ++k) m = largest(v[k], m);
    scale_to<ENT>(a, m, c);
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = v[k][e] - m, x = exp2_of(d * c);
            s += x;
            if (ENT) t = fmaf(x, d, t);
        }
    if (ENT && t != t) { // minus infinity times 0, most likely: once more, without
        t = 0.0f;
        float at = m;
        asm volatile("" : "+v"(at)); // or this is computed beside the other, every time
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = v[k][e] - at;
                t = fmaf(exp2_of(d * c), fmaxf(d, kFloor), t);
            }
    }
    a.s += s;
    if (ENT) a.t += t;
}

__device__ __forceinline__ float wave_most(float v) {
    v = row16_max(v);
    return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}
/* Over the lanes of a wave, the same in all of them. */
template <bool ENT> __device__ __forceinline__ void wave_join(Sums &a, float c) {
    scale_to<ENT>(a, wave_most(a.m), c);
    a.s = wave_sum(a.s);
    if (ENT) a.t = wave_sum(a.t);
}
/* Over the waves of a workgroup, through a slot for each. */
template <bool ENT, int WAVES> __device__ __forceinline__ void group_join(Sums &a, float c, Sums *slots) {
    wave_join<ENT>(a, c);
    if (WAVES == 1) return;
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = a;
    __syncthreads();
    float m = slots[0].m;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, slots[w].m);
    Sums all = {m, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        Sums b = slots[w];
        scale_to<ENT>(b, m, c);
        all.s += b.s;
        all.t += b.t;
    }
    a = all;
}

/* Elements as 63-bit keys: ordered by value, of equal values the one that comes first is larger; 0 is no element.  But for NaN's they are the bits of
 * positive normal doubles, which one instruction compares and selects; as integers they took a comparison, its inversion in half of the lanes and two
 * selections one after the other, and a sort of a wave's keys 2060 cycles. */
typedef uint64_t Key;
__device__ __forceinline__ Key key_of(float v, uint32_t place) { // place below 2^31
    const uint32_t u = as_bits(v + 0.0f); // minus zero is zero
    return (Key)(u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) << 31 | (~place & 0x7fffffffu);
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t u = (uint32_t)(k >> 31);
    return as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t place_of(Key k) { return ~(uint32_t)k & 0x7fffffffu; }

template <int CTRL> __device__ __forceinline__ Key key_dpp(Key k) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)k, CTRL, 0xf, 0xf, true), hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(k >> 32), CTRL, 0xf, 0xf, true);
    return (Key)hi << 32 | lo;
}
__device__ __forceinline__ Key key_from(Key k, uint32_t lane) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(lane * 4), (int)(uint32_t)k), hi = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(lane * 4), (int)(uint32_t)(k >> 32));
    return (Key)hi << 32 | lo;
}
/* The key of lane ^ M. */
template <int M> __device__ __forceinline__ Key key_across(Key k, uint32_t lane) {
    if (M == 1) return key_dpp<0xb1>(k);
    if (M == 2) return key_dpp<0x4e>(k);
    if (M == 3) return key_dpp<0x1b>(k);
    if (M == 4) return key_dpp<0x141>(key_dpp<0x1b>(k)); // row_half_mirror is 7
    if (M == 7) return key_dpp<0x141>(k);
    if (M == 8) return key_dpp<0x128>(k); // row_ror:8
    if (M == 15) return key_dpp<0x140>(k);
    return key_from(k, lane ^ M);
}
__device__ __forceinline__ Key larger(Key a, Key b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(__builtin_bit_cast(double, a)), "v"(__builtin_bit_cast(double, b)));
    return __builtin_bit_cast(Key, r);
}
__device__ __forceinline__ Key smaller(Key a, Key b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(__builtin_bit_cast(double, a)), "v"(__builtin_bit_cast(double, b)));
    return __builtin_bit_cast(Key, r);
}
/* Of two lanes M apart the one whose bit HIGH is clear takes the larger key. */
template <int M, int HIGH> __device__ __forceinline__ void exchange(Key &k, uint32_t lane) {
    const Key o = key_across<M>(k, lane), up = larger(k, o), down = smaller(k, o);
    k = lane & HIGH ? down : up;
}
/* A wave's 64 keys in descending order, by Batcher's bitonic network. */
__device__ __forceinline__ void sort64(Key &k, uint32_t lane) {
    exchange<1, 1>(k, lane);
    exchange<3, 2>(k, lane), exchange<1, 1>(k, lane);
    exchange<7, 4>(k, lane), exchange<2, 2>(k, lane), exchange<1, 1>(k, lane);
    exchange<15, 8>(k, lane), exchange<4, 4>(k, lane), exchange<2, 2>(k, lane), exchange<1, 1>(k, lane);
    exchange<31, 16>(k, lane), exchange<8, 8>(k, lane), exchange<4, 4>(k, lane), exchange<2, 2>(k, lane), exchange<1, 1>(k, lane);
    exchange<63, 32>(k, lane), exchange<16, 16>(k, lane), exchange<8, 8>(k, lane), exchange<4, 4>(k, lane), exchange<2, 2>(k, lane), exchange<1, 1>(k, lane);
}
/* The 64 largest of a descending list and of another that is given in ascending order. */
__device__ __forceinline__ void merge64(Key &k, Key ascending, uint32_t lane) {
    k = larger(k, ascending); // goes to LDS next: a lane exchange right behind inline assembly would lack the wait that the compiler puts there else
    exchange<32, 32>(k, lane), exchange<16, 16>(k, lane), exchange<8, 8>(k, lane), exchange<4, 4>(k, lane), exchange<2, 2>(k, lane), exchange<1, 1>(k, lane);
}

__device__ __forceinline__ int64_t id_at(const void *ids, bool wide, uint64_t i) { return wide ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i]; }

struct bf16_or_f32 { // elements whose type is known at run time only
    const void *p;
    bool f32;
    __device__ __forceinline__ float operator[](uint64_t i) const { return f32 ? ((const float *)p)[i] : as_float((uint32_t)((const uint16_t *)p)[i] << 16); }
};
/* Launchers, one file for the scores, one for the distillation, one for the gradients; the arguments have been checked and are not empty. */
int launch_token_logprobs(const EriTokenLogprobs &a, void *stream);
uint64_t token_logprobs_workspace(uint64_t rows, uint64_t vocab, uint32_t top);
int launch_distill_top(const EriDistillTop &a, void *stream);
uint64_t distill_top_workspace(uint64_t rows, uint64_t vocab);
int launch_token_logprobs_grad(const EriTokenLogprobsGrad &a, void *stream);
int launch_distill_top_grad(const EriDistillTopGrad &a, void *stream);

} // namespace eri_losses
