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
constexpr float kFloor = -1e30f;           // below any distance that counts: 0 * kFloor is 0 where 0 * -infinity would be NaN
constexpr double kLog2e = 1.4426950408889634074;
constexpr float kLn2 = 0.693147181f;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); } // one instruction, one unit in the last place

/* Vectors of eight logits.  A row is cut into whole vectors and a last one of cols % 8 elements, which is read element by
 * element: nothing outside of a vector is read with it, so that a row may be written over while its other vectors are still wanted. */
__device__ __forceinline__ void all_least(Raw<bf16> &r) { r.a = u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
__device__ __forceinline__ void all_least(Raw<float> &r) { r.a = r.b = u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}; }
template <typename T> __device__ __forceinline__ void values_of(float (&v)[8], const Raw<T> &r) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = r.get(e);
}
template <typename T> __device__ __forceinline__ void load_last(float (&v)[8], const T *p, uint32_t n) { // 0 < n < 8 elements, minus infinity behind them
    Raw<T> r;
    r.load_some(p, n);
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = e < n ? r.get(e) : -kInf;
}

/* Vectors first .. last-1 of a row, dealt to TPR threads in turn, N of each at a time: all loads of a batch are under way before the first is
 * wanted.  `use(values, at, full)` gets an array of C vectors, those that begin at vector at + k TPR + t; in the last of them there is nothing but
 * minus infinity for threads past the end, unless `full`.  The rest of the row is one smaller batch: vector by vector it took a trip to memory for each. */
template <int TPR, int C, bool FULL, typename T, typename Use> __device__ __forceinline__ void walk_batch(const T *row, uint32_t at, uint32_t last, uint32_t t, Use &use) {
    Raw<T> raw[C];
    float v[C][8];
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const uint32_t vec = at + k * TPR + t;
        if (FULL || k < C - 1) raw[k].load(row + (uint64_t)vec * 8);
        else {
            all_least(raw[k]);
            if (vec < last) raw[k].load(row + (uint64_t)vec * 8);
        }
    }
#pragma unroll
    for (int k = 0; k < C; ++k) values_of(v[k], raw[k]);
    use(v, at, FULL);
}
template <int TPR, typename T, typename Use> __device__ __forceinline__ void walk(const T *row, uint32_t first, uint32_t last, uint32_t t, Use use) {
    constexpr int N = sizeof(T) == 2 ? 4 : 2; // 64 bytes of a row for each thread
    uint32_t at = first;
    for (; at + N * TPR <= last; at += N * TPR) walk_batch<TPR, N, true>(row, at, last, t, use);
    if (at >= last) return;
    const uint32_t left = (last - at + TPR - 1) / TPR;
    if (left == 1) walk_batch<TPR, 1, false>(row, at, last, t, use);
    else if (N == 2 || left == 2) walk_batch<TPR, 2, false>(row, at, last, t, use);
    else if (left == 3) walk_batch<TPR, 3, false>(row, at, last, t, use);
    else walk_batch<TPR, 4, false>(row, at, last, t, use);
}

/* The running softmax: m the largest logit, s the sum of exp((x - m) / T), t the sum of exp((x - m) / T) (x - m), whose terms are all
 * of one sign, so that the entropy ln s - t / (s T) loses nothing.  c = log2(e) / T.  Differences are taken before they are scaled: x c - m c in
 * one fused product would overflow for the lowest values of a type, which stand for masks, and round m c on the way. */
struct Sums {
    float m, s, t;
};
__device__ __forceinline__ float largest(const float (&v)[8]) { // NaN is passed over
    return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}
template <bool ENT> __device__ __forceinline__ void scale_to(Sums &a, float m, float c) { // m >= a.m
    const float d = a.m - m, f = exp2_of(d * c);
    if (ENT) a.t = f * fmaf(a.s, fmaxf(d, kFloor), a.t);
    a.s *= f;
    a.m = m;
}
template <bool ENT, int N> __device__ __forceinline__ void add(Sums &a, float (&v)[N][8], float c) {
    float m = a.m;
#pragma unroll
    for (int k = 0; k < N; ++k) m = fmaxf(m, largest(v[k]));
    scale_to<ENT>(a, m, c);
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = v[k][e] - m, x = exp2_of(d * c);
            s += x;
            if (ENT) t = fmaf(x, fmaxf(d, kFloor), t);
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

/* Elements as 64-bit keys: ordered by value, of equal values the one that comes first is larger.  0 is no element. */
typedef uint64_t Key;
__device__ __forceinline__ Key key_of(float v, uint32_t place) {
    const uint32_t u = as_bits(v + 0.0f); // minus zero is zero
    return (Key)(u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) << 32 | (uint32_t)~place;
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t place_of(Key k) { return ~(uint32_t)k; }

template <int CTRL> __device__ __forceinline__ Key key_dpp(Key k) {
    const uint32_t lo = as_bits(dpp<CTRL, 0xf>(0.0f, as_float((uint32_t)k))), hi = as_bits(dpp<CTRL, 0xf>(0.0f, as_float((uint32_t)(k >> 32))));
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
/* Of two lanes M apart the one whose bit HIGH is clear takes the larger key. */
template <int M, int HIGH> __device__ __forceinline__ void exchange(Key &k, uint32_t lane) {
    const Key o = key_across<M>(k, lane);
    k = (o > k) == ((lane & HIGH) == 0) ? o : k; // equal keys are the same element
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
    if (ascending > k) k = ascending;
    exchange<32, 32>(k, lane), exchange<16, 16>(k, lane), exchange<8, 8>(k, lane), exchange<4, 4>(k, lane), exchange<2, 2>(k, lane), exchange<1, 1>(k, lane);
}

__device__ __forceinline__ int64_t id_at(const void *ids, bool wide, uint64_t i) { return wide ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i]; }

struct bf16_or_f32 { // elements whose type is known at run time only
    const void *p;
    bool f32;
    __device__ __forceinline__ float operator[](uint64_t i) const { return f32 ? ((const float *)p)[i] : as_float((uint32_t)((const uint16_t *)p)[i] << 16); }
};
template <typename T> __device__ __forceinline__ float at(const T *p) { return (float)*p; }
template <> __device__ __forceinline__ float at<bf16>(const bf16 *p) { return as_float((uint32_t)p->bits << 16); }

/* Launchers, one file for the scores, one for the distillation, one for the gradients; the arguments have been checked and are not empty. */
int launch_token_logprobs(const EriTokenLogprobs &a, void *stream);
uint64_t token_logprobs_workspace(uint64_t rows, uint64_t vocab, uint32_t top);
int launch_distill_top(const EriDistillTop &a, void *stream);
uint64_t distill_top_workspace(uint64_t rows, uint64_t vocab);
int launch_token_logprobs_grad(const EriTokenLogprobsGrad &a, void *stream);
int launch_distill_top_grad(const EriDistillTopGrad &a, void *stream);

} // namespace eri_losses
