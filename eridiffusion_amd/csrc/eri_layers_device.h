/*
 * What the kernels of include/eri_layers.h share: rows of F32 or BF16 elements in vectors of eight, sums over a
 * wave and a workgroup, and the generator behind dropout.
 */
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/eri_layers.h"

namespace eri_layers {

constexpr uint32_t kWave = 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2))); // rows of odd length: the hardware takes a 16-byte access at any address
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_at1 __attribute__((aligned(1)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
typedef u32x2 u32x2_at4 __attribute__((aligned(4)));
typedef uint32_t u32_at2 __attribute__((aligned(2)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));
typedef uint16_t u16_at1 __attribute__((aligned(1)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct bf16 { // an element's bits
    uint16_t bits;
};

__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

/* Two fp32 to one dword of two bf16, nearest even. */
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const f32x2 f = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

/* Eight adjacent elements as they lie in memory. */
template <typename T> struct Raw;
template <> struct Raw<bf16> {
    u32x4 a;
    __device__ __forceinline__ void clear() { a = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void load(const bf16 *p) { a = *(const u32x4_at2 *)p; }
    __device__ __forceinline__ void load_once(const bf16 *p) { a = __builtin_nontemporal_load((const u32x4_at2 *)p); }
    __device__ __forceinline__ void load_some(const bf16 *p, uint32_t n) { // n < 8 elements
        clear();
#pragma unroll
        for (uint32_t e = 0; e < 7; ++e)
            if (e < n) a[e / 2] |= (uint32_t)p[e].bits << (16 * (e & 1));
    }
    __device__ __forceinline__ void shift(uint32_t n) { // drops the first n elements, zeros come after the last
        if (n & 4) a = u32x4{a[2], a[3], 0, 0};
        if (n & 2) a = u32x4{a[1], a[2], a[3], 0};
        if (n & 1) a = u32x4{a[0] >> 16 | a[1] << 16, a[1] >> 16 | a[2] << 16, a[2] >> 16 | a[3] << 16, a[3] >> 16};
        if (n & 8) clear();
    }
    __device__ __forceinline__ float get(uint32_t e) const { return as_float(e & 1 ? a[e / 2] & 0xffff0000u : a[e / 2] << 16); }
};
template <> struct Raw<float> {
    u32x4 a, b;
    __device__ __forceinline__ void clear() { a = b = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void load(const float *p) {
        a = *(const u32x4_at4 *)p;
        b = *(const u32x4_at4 *)(p + 4);
    }
    __device__ __forceinline__ void load_once(const float *p) {
        a = __builtin_nontemporal_load((const u32x4_at4 *)p);
        b = __builtin_nontemporal_load((const u32x4_at4 *)(p + 4));
    }
    __device__ __forceinline__ void load_some(const float *p, uint32_t n) {
        clear();
#pragma unroll
        for (uint32_t e = 0; e < 7; ++e)
            if (e < n) set(e, p[e]);
    }
    __device__ __forceinline__ void shift(uint32_t n) {
        if (n & 4) a = b, b = u32x4{0, 0, 0, 0};
        if (n & 2) a = u32x4{a[2], a[3], b[0], b[1]}, b = u32x4{b[2], b[3], 0, 0};
        if (n & 1) a = u32x4{a[1], a[2], a[3], b[0]}, b = u32x4{b[1], b[2], b[3], 0};
        if (n & 8) clear();
    }
    __device__ __forceinline__ float get(uint32_t e) const { return as_float(e < 4 ? a[e] : b[e - 4]); }
    __device__ __forceinline__ void set(uint32_t e, float f) { if (e < 4) a[e] = as_bits(f); else b[e - 4] = as_bits(f); }
};

/* Elements col .. col+7 of a row of cols, with zeros past its end, in two steps: load8 starts the loads, and settle8 is called
 * when the values are wanted.  Where a row ends inside the vector, its last eight elements are loaded instead and shifted
 * into place later: all lanes take the same load, and nothing between two loads waits for the first.  With a branch for each
 * case in its place, the wave at the end of an odd row waited at every row (sums of a table's gradient of 1155 columns: 59 us, so 25).
 * SHORT is for rows of less than eight elements, which have kernels of their own; ONCE for rows that nobody reads again. */
template <typename I> __device__ __forceinline__ I from_of(I col, I cols) { return col + 8 <= cols ? col : cols - 8; }
template <bool SHORT, bool ONCE = false, typename T, typename I> __device__ __forceinline__ void load8(Raw<T> &r, const T *row, I col, I cols) {
    if (SHORT) r.load_some(row, col == 0 ? (uint32_t)cols : 0u);
    else if (ONCE) r.load_once(row + from_of(col, cols));
    else r.load(row + from_of(col, cols));
}
template <typename I> __device__ __forceinline__ uint32_t past_of(I col, I cols) { // elements of the vector that lie past the row's end
    return col >= cols ? 8u : (uint32_t)(col + 8 - cols);
}
template <bool SHORT, typename T, typename I> __device__ __forceinline__ void settle8(Raw<T> &r, I col, I cols) {
    if (!SHORT && col + 8 > cols) r.shift(past_of(col, cols));
}

/* n of eight elements: all, or the 4, 2 and 1 that n is made of. */
__device__ __forceinline__ void store_n(bf16 *p, uint32_t n, const float (&v)[8]) {
    u32x4 w = {bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
    if (n >= 8) {
        *(u32x4_at2 *)p = w;
        return;
    }
    if (n & 4) {
        *(u32x2_at2 *)p = u32x2{w[0], w[1]};
        p += 4, w[0] = w[2], w[1] = w[3];
    }
    if (n & 2) {
        *(u32_at2 *)p = w[0];
        p += 2, w[0] = w[1];
    }
    if (n & 1) p->bits = (uint16_t)w[0];
}
__device__ __forceinline__ void store_n(float *p, uint32_t n, const float (&v)[8]) {
    u32x4 a = {as_bits(v[0]), as_bits(v[1]), as_bits(v[2]), as_bits(v[3])}, b = {as_bits(v[4]), as_bits(v[5]), as_bits(v[6]), as_bits(v[7])};
    if (n >= 8) {
        *(u32x4_at4 *)p = a;
        *(u32x4_at4 *)(p + 4) = b;
        return;
    }
    if (n & 4) {
        *(u32x4_at4 *)p = a;
        p += 4, a = b;
    }
    if (n & 2) {
        *(u32x2_at4 *)p = u32x2{a[0], a[1]};
        p += 2, a[0] = a[2];
    }
    if (n & 1) *p = as_float(a[0]);
}
template <typename T, typename I> __device__ __forceinline__ void store8(T *row, I col, I cols, const float (&v)[8]) {
    if (col < cols) store_n(row + col, col + 8 <= cols ? 8u : (uint32_t)(cols - col), v);
}

/* The same with the element's type known at run time only (the same for all lanes). */
template <bool SHORT> __device__ __forceinline__ void load8_of(float (&v)[8], const void *row, bool f32, uint32_t col, uint32_t cols) {
    if (f32) {
        Raw<float> r;
        load8<SHORT>(r, (const float *)row, col, cols);
        settle8<SHORT>(r, col, cols);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = r.get(e);
    } else {
        Raw<bf16> r;
        load8<SHORT>(r, (const bf16 *)row, col, cols);
        settle8<SHORT>(r, col, cols);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = r.get(e);
    }
}

/* Sum and maximum over a wave in a fixed order, the same for all its lanes. */
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp(float old, float v) {
    return as_float(__builtin_amdgcn_update_dpp((int)as_bits(old), (int)as_bits(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp<0xb1, 0xf>(0.0f, v);  // quad_perm [1,0,3,2]
    v += dpp<0x4e, 0xf>(0.0f, v);  // quad_perm [2,3,0,1]
    v += dpp<0x141, 0xf>(0.0f, v); // row_half_mirror
    v += dpp<0x140, 0xf>(0.0f, v); // row_mirror: every lane has the sum of its 16
    return v;
}
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp<0xb1, 0xf>(0.0f, v));
    v = fmaxf(v, dpp<0x4e, 0xf>(0.0f, v));
    v = fmaxf(v, dpp<0x141, 0xf>(0.0f, v));
    v = fmaxf(v, dpp<0x140, 0xf>(0.0f, v));
    return v;
}
__device__ __forceinline__ float lane_of(float v, int lane) { return as_float((uint32_t)__builtin_amdgcn_readlane((int)as_bits(v), lane)); }
__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
__device__ __forceinline__ float wave_max(float v) { // of values >= 0
    v = row16_max(v);
    return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}

/* Over T threads that stand side by side: 16, 32, a wave, or the waves of a workgroup through `slots` (a float for each).  The caller
 * alternates between two arrays of slots from one call to the next: a wave that is a call ahead must not overwrite
 * what a slower one still reads. */
template <int T> constexpr int kSlots = T > (int)kWave ? T / (int)kWave : 1;
template <int T> __device__ __forceinline__ float sum_over(float v, float *slots) {
    if (T == 16) return row16_sum(v);
    if (T == 32) {
        v = row16_sum(v);
        return v + __shfl_xor(v, 16);
    }
    v = wave_sum(v);
    if (T == kWave) return v;
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = slots[0];
#pragma unroll
    for (int w = 1; w < kSlots<T>; ++w) s += slots[w];
    return s;
}
template <int T> __device__ __forceinline__ float max_over(float v, float *slots) { // of values >= 0
    if (T == 16) return row16_max(v);
    if (T == 32) {
        v = row16_max(v);
        return fmaxf(v, __shfl_xor(v, 16));
    }
    v = wave_max(v);
    if (T == kWave) return v;
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = slots[0];
#pragma unroll
    for (int w = 1; w < kSlots<T>; ++w) s = fmaxf(s, slots[w]);
    return s;
}

/* What a kernel needs of an EriDropoutKey. */
struct Drop {
    uint64_t seed, offset;
    const uint64_t *offset_ptr;
    uint32_t below; // kept where the 16 bits are not below this; 65536: nothing is kept
    float scale;    // 65536 / (65536 - below)
};

/* Philox4x32-10: the 128 bits at counter {group, offset}.  Twenty 32x32->64 products, which is what costs. */
__device__ __forceinline__ u32x4 philox(uint64_t group, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

/* The 16-bit draws of elements first .. first+7, two a word.  Where `first` is no multiple of eight (rows of odd length)
 * they straddle two counters. */
__device__ __forceinline__ u32x4 draw8(uint64_t first, const Drop &d, uint64_t offset) {
    const u32x4 w = philox(first >> 3, offset, d.seed);
    const uint32_t s = (uint32_t)first & 7u;
    if (s == 0) return w;
    const u32x4 n = philox((first >> 3) + 1, offset, d.seed);
    const bool by4 = s & 4, by2 = s & 2;
    const uint32_t b0 = by4 ? w[2] : w[0], b1 = by4 ? w[3] : w[1], b2 = by4 ? n[0] : w[2], b3 = by4 ? n[1] : w[3], b4 = by4 ? n[2] : n[0], b5 = by4 ? n[3] : n[1];
    const uint32_t c0 = by2 ? b1 : b0, c1 = by2 ? b2 : b1, c2 = by2 ? b3 : b2, c3 = by2 ? b4 : b3, c4 = by2 ? b5 : b4;
    if (!(s & 1)) return u32x4{c0, c1, c2, c3};
    return u32x4{c0 >> 16 | c1 << 16, c1 >> 16 | c2 << 16, c2 >> 16 | c3 << 16, c3 >> 16 | c4 << 16};
}

__device__ __forceinline__ uint64_t drop_offset(const Drop &d) { return d.offset + (d.offset_ptr ? *d.offset_ptr : 0); }

__device__ __forceinline__ float dropped(float v, const u32x4 &bits, uint32_t e, const Drop &d) {
    const uint32_t half = e & 1 ? bits[e / 2] >> 16 : bits[e / 2] & 0xffffu;
    return half >= d.below ? v * d.scale : 0.0f;
}

/* Launchers, one file for each; `stream` is a hipStream_t and the result a hipError_t.  The arguments have been checked:
 * strides are set, rows and cols are not 0 where it is not said. */
int launch_embedding(const EriEmbedding &a, uint32_t compute_units, void *stream);
int launch_embedding_grad(const EriEmbeddingGrad &a, void *stream);
uint64_t embedding_grad_workspace(uint64_t tokens, uint64_t vocab, uint64_t dim);
int launch_dropout(const EriDropout &a, const Drop &d, uint32_t compute_units, void *stream);
int launch_rms_norm(const EriRmsNorm &a, const Drop &d, void *stream);
int launch_rms_norm_grad(const EriRmsNormGrad &a, const Drop &d, uint32_t compute_units, void *stream); // rows may be 0
uint64_t rms_norm_grad_workspace(uint64_t rows, uint64_t cols, uint32_t compute_units);

} // namespace eri_layers
