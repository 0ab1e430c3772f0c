/*
 * Residual addition and root-mean-square norm of include/eri_layers.h, forward: h = r + drop(x), q = 1/sqrt(mean h^2 + eps),
 * y = h q w, in 8 bits scaled by each group's largest |y|.
 *
 * Bound by HBM: x and r are read once, h and y written once, and the row waits in registers for its sum.  16 threads to a row of up
 * to 128 columns (a group of the 8-bit output is 16 lanes then, as it is in every layout), 32 to 256, a wave to 1024 and no
 * barrier that far, then as many threads as the row has vectors of eight, to two or four each in the longest.  Narrow rows on
 * whole waves ran at a third: 100000 x 128 bf16 28 us, now 11.  Fewer threads with more of the row each, us for 8192 rows with a
 * residual:
 *   2048 bf16 64 threads 22.4, 256 21.2;   4096 bf16 64 50.9, 256 42.6, 512 42.2;   4096 fp32 64 109, 256 97.8, 512 93.4;
 *   6144 fp32 256 150, 512 144;   8192 bf16 256 96.7, 512 94.6, 1024 91.4;   1000 bf16 128 12.4, 64 11.9
 * Where a row moves fewer bytes, half the threads with twice the vectors win.  A
 * bf16 row of 4097 to 6144 columns: to 8 bits with a residual 256 threads 50.7, 512 57.5 (at 6144 columns 65.5 and 67.6), to bf16
 * with one 60.1 and 59.2 (2048 rows 14.1 and 15.5).  Without a residual, unless y is fp32:
 *   bf16 to 8 bits  2560 18.4, was 22.2;   4096 20.2, 23.1;   5120 30.0, 38.3;   8192 43.2, 51.9;   12288 64.1, 80.0
 *   bf16 to bf16    2560 16.4, was 19.6;   4096 21.5, 22.9;   5120 30.1, 35.6;   8192 44.7, 52.5;   12288 72.9, 80.4
 *   fp32 to bf16    2560 22.9, was 26.2;   4096 32.8, 32.5;   5120 41.6, 43.8;   8192 72.4, 76.2;   12288 105.9, 117.7
 *   bf16 to fp32    2560 22.2, not so 22.8; 4096 37.3, 35.3; 5120 45.3, 47.7; 8192 76.8, 75.6;   2048 19.5, 18.1: not worth it
 * and of 1025 to 2048 columns, 32768 rows: 128 threads with two vectors each, before them 256 with one:
 *   bf16 to 8 bits  1100 39.1, was 49.1;   1536 38.5, 48.7;   2048 40.4, 49.4
 *   bf16 to bf16    1100 38.3, was 45.9;   1536 37.9, 45.1;   2048 44.9, 48.3
 *   fp32 to bf16    1100 40.0, was 47.2;   1536 48.7, 52.9;   2048 68.1, 67.6
 * A row's layout, and so its rounding, does not depend on how many rows there are.
 * Dropout is drawn beside the loads and costs nothing: 16384 x 4096 bf16 with residual and dropout 91 us, 5.9 TB/s (a copy of that
 * size runs at 5.2); 8192 x 5120 to 8 bits 51-57 us, 5.2-5.8 TB/s; one row of 4096 2.2 us, a launch and two trips to memory.
 */
#include "eri_layers_device.h"

namespace eri_layers {
namespace {

constexpr float kF8Max = 448.0f;
constexpr float kLeast = 0x1p-100f; // a group whose largest |y| is below this is zeros: 448 / |y| would leave fp32 not far below
constexpr uint32_t rows_of(uint32_t tpr) { return tpr <= kWave ? 256 / tpr : 1; } // of a workgroup

struct NormArgs {
    const void *x, *residual, *weight;
    void *y, *h;
    float *rstd, *scales;
    uint32_t first, rows, cols; // rows first .. rows-1
    uint64_t x_stride, residual_stride, y_stride, h_stride;
    float eps;
    uint32_t weight_f32, y_dtype, group, groups;
    Drop drop;
};

__device__ __forceinline__ void store8_f8(uint8_t *row, uint32_t col, uint32_t cols, const float (&v)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
        w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], p, true);
    }
    if (col >= cols) return;
    row += col;
    const uint32_t n = cols - col;
    if (n >= 8) {
        *(u32x2_at1 *)row = u32x2{w[0], w[1]};
        return;
    }
    if (n & 4) {
        *(u32_at1 *)row = w[0];
        row += 4, w[0] = w[1];
    }
    if (n & 2) {
        *(u16_at1 *)row = (uint16_t)w[0];
        row += 2, w[0] >>= 16;
    }
    if (n & 1) *row = (uint8_t)w[0];
}

/* h of elements col .. col+7 of a row, zero past its end. */
template <bool SHORT, typename TX, typename TR, bool RES, bool DROP>
__device__ __forceinline__ void sum8(float (&h)[8], Raw<TX> &x, Raw<TR> &r, uint32_t row, uint32_t col, uint32_t cols, const Drop &d, uint64_t offset) {
    const uint64_t first = (uint64_t)row * cols + col;
    u32x4 bits = {0, 0, 0, 0};
    if (DROP) bits = draw8(first, d, offset);
    settle8<SHORT>(x, col, cols);
    if (RES) settle8<SHORT>(r, col, cols);
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        h[e] = x.get(e);
        if (DROP) h[e] = dropped(h[e], bits, e, d);
        if (RES) h[e] += r.get(e);
    }
}

template <typename TX, typename TR, bool RES> __device__ __forceinline__ void store_h(const NormArgs &a, uint32_t row, uint32_t col, const float (&h)[8]) {
    if (RES) store8((TR *)a.h + row * a.h_stride, col, a.cols, h);
    else store8((TX *)a.h + row * a.h_stride, col, a.cols, h);
}

template <bool SHORT> __device__ __forceinline__ void weigh(float (&v)[8], const NormArgs &a, uint32_t col, float rstd) {
    float w[8];
    if (a.weight) load8_of<SHORT>(w, a.weight, a.weight_f32, col, a.cols);
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = a.weight ? v[e] * rstd * w[e] : v[e] * rstd;
}

/* y / scale as 8-bit floats; `most` is the largest |y| of the group */
__device__ __forceinline__ void store_scaled(const NormArgs &a, uint32_t row, uint32_t col, const float (&v)[8], float most) {
    const float inv = most >= kLeast ? kF8Max / most : 1.0f;
    float q[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) q[e] = v[e] * inv;
    store8_f8((uint8_t *)a.y + row * a.y_stride, col, a.cols, q);
}
__device__ __forceinline__ float scale_of(float most) { return most >= kLeast ? most / kF8Max : 1.0f; }
__device__ __forceinline__ float most_of(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    return m;
}

/* A row to TPR threads, NV vectors of eight elements in the registers of each. */
template <typename TX, typename TR, bool RES, bool DROP, int TPR, int NV, bool SHORT>
__global__ __launch_bounds__(TPR * rows_of(TPR)) void rms_norm_kernel(const NormArgs a) {
    __shared__ float slots[2][kSlots<TPR>];
    const uint32_t row = a.first + blockIdx.x * rows_of(TPR) + threadIdx.x / TPR, t = threadIdx.x % TPR;
    if (row >= a.rows) return; // all threads of the row, and only where none of them waits for others
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    Raw<TX> x[NV];
    Raw<TR> r[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) load8<SHORT>(x[k], (const TX *)a.x + row * a.x_stride, (k * TPR + t) * 8, a.cols);
    if (RES)
#pragma unroll
        for (int k = 0; k < NV; ++k) load8<SHORT>(r[k], (const TR *)a.residual + row * a.residual_stride, (k * TPR + t) * 8, a.cols);
    float h[NV][8], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t col = (k * TPR + t) * 8;
        sum8<SHORT, TX, TR, RES, DROP>(h[k], x[k], r[k], row, col, a.cols, a.drop, offset);
        if (a.h) store_h<TX, TR, RES>(a, row, col, h[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(h[k][e], h[k][e], sum);
    }
    const float rstd = 1.0f / sqrtf(sum_over<TPR>(sum, slots[0]) / (float)a.cols + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = rstd;
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t col = (k * TPR + t) * 8;
        weigh<SHORT>(h[k], a, col, rstd);
        if (a.y_dtype == ERI_DTYPE_BF16) store8((bf16 *)a.y + row * a.y_stride, col, a.cols, h[k]);
        else if (a.y_dtype == ERI_DTYPE_F32) store8((float *)a.y + row * a.y_stride, col, a.cols, h[k]);
        else if (a.group) {
            const float m = row16_max(most_of(h[k])); // 16 lanes hold 128 columns
            store_scaled(a, row, col, h[k], m);
            if (t % 16 == 0 && col < a.cols) a.scales[(uint64_t)row * a.groups + col / 128] = scale_of(m);
        } else most = fmaxf(most, most_of(h[k]));
    }
    if (a.y_dtype == ERI_DTYPE_F8E4M3 && !a.group) {
        most = max_over<TPR>(most, slots[1]);
#pragma unroll
        for (int k = 0; k < NV; ++k) store_scaled(a, row, (k * TPR + t) * 8, h[k], most);
        if (t == 0) a.scales[row] = scale_of(most);
    }
}

/* Rows over 32768 columns, too long for registers: read again for each of the passes.  h and y are written in the last one only, each
 * element by the thread that has just read it, so that they may replace the residual and x. */
template <typename TX, typename TR, bool RES, bool DROP> __global__ __launch_bounds__(1024) void rms_norm_long_kernel(const NormArgs a) {
    __shared__ float slots[2][16];
    const uint32_t row = a.first + blockIdx.x;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    auto value = [&](float (&h)[8], uint32_t col) {
        Raw<TX> x;
        Raw<TR> r;
        load8<false>(x, (const TX *)a.x + row * a.x_stride, col, a.cols);
        if (RES) load8<false>(r, (const TR *)a.residual + row * a.residual_stride, col, a.cols);
        sum8<false, TX, TR, RES, DROP>(h, x, r, row, col, a.cols, a.drop, offset);
    };
    float sum = 0.0f;
    for (uint32_t col = threadIdx.x * 8; col < a.cols; col += 8192) {
        float h[8];
        value(h, col);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(h[e], h[e], sum);
    }
    const float rstd = 1.0f / sqrtf(sum_over<1024>(sum, slots[0]) / (float)a.cols + a.eps);
    float most = 0.0f;
    if (a.y_dtype == ERI_DTYPE_F8E4M3 && !a.group) {
        for (uint32_t col = threadIdx.x * 8; col < a.cols; col += 8192) {
            float h[8];
            value(h, col);
            weigh<false>(h, a, col, rstd);
            most = fmaxf(most, most_of(h));
        }
        most = max_over<1024>(most, slots[1]);
        if (threadIdx.x == 0) a.scales[row] = scale_of(most);
    }
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    // all lanes stay together to the last column: 16 of them share a group's maximum
    for (uint32_t at = 0; at < a.cols; at += 8192) {
        const uint32_t col = at + threadIdx.x * 8;
        float h[8];
        value(h, col);
        if (a.h) store_h<TX, TR, RES>(a, row, col, h);
        weigh<false>(h, a, col, rstd);
        if (a.y_dtype == ERI_DTYPE_BF16) store8((bf16 *)a.y + row * a.y_stride, col, a.cols, h);
        else if (a.y_dtype == ERI_DTYPE_F32) store8((float *)a.y + row * a.y_stride, col, a.cols, h);
        else if (a.group) {
            const float m = row16_max(most_of(h));
            store_scaled(a, row, col, h, m);
            if (threadIdx.x % 16 == 0 && col < a.cols) a.scales[(uint64_t)row * a.groups + col / 128] = scale_of(m);
        } else store_scaled(a, row, col, h, most);
    }
}

template <typename TX, typename TR, bool RES, bool DROP> void launch(const NormArgs &a, hipStream_t s) {
#define ERI_NORM(TPR, NV, SHORT) \
    hipLaunchKernelGGL((rms_norm_kernel<TX, TR, RES, DROP, TPR, NV, SHORT>), dim3((a.rows - a.first + rows_of(TPR) - 1) / rows_of(TPR)), dim3(TPR * rows_of(TPR)), 0, s, a)
// the layout of a row that moves few bytes, then the others'; only those that some call reaches are compiled
#define ERI_NORM_EITHER(TPR, NV, TPR2, NV2) \
    do { \
        if constexpr (!kMayBeLight) ERI_NORM(TPR2, NV2, false); \
        else if (a.y_dtype != ERI_DTYPE_F32) ERI_NORM(TPR, NV, false); \
        else ERI_NORM(TPR2, NV2, false); \
    } while (0)
    constexpr bool kMayBeLight = !RES; // and is unless y is fp32
    constexpr int kMiddle = RES && sizeof(TX) + sizeof(TR) == 4 ? 256 : 512; // threads to other rows of 4097 to 6144 columns
    if (a.cols < 8) ERI_NORM(16, 1, true);
    else if (a.cols <= 128) ERI_NORM(16, 1, false);
    else if (a.cols <= 256) ERI_NORM(32, 1, false);
    else if (a.cols <= 512) ERI_NORM(64, 1, false);
    else if (a.cols <= 1024) ERI_NORM(64, 2, false);
    else if (a.cols <= 2048) ERI_NORM_EITHER(128, 2, 256, 1);
    else if (a.cols <= 4096) ERI_NORM_EITHER(256, 2, 512, 1);
    else if (a.cols <= 6144) ERI_NORM_EITHER(256, 3, kMiddle, (kMiddle == 256 ? 3 : 2));
    else if (a.cols <= 8192) ERI_NORM_EITHER(256, 4, 1024, 1);
    else if (a.cols <= 12288) ERI_NORM_EITHER(512, 3, 1024, 2);
    else if (a.cols <= 16384) ERI_NORM(1024, 2, false);
    else if (a.cols <= 32768) ERI_NORM(1024, 4, false);
    else hipLaunchKernelGGL((rms_norm_long_kernel<TX, TR, RES, DROP>), dim3(a.rows - a.first), dim3(1024), 0, s, a);
#undef ERI_NORM_EITHER
#undef ERI_NORM
}

template <typename TX> void launch_of(const NormArgs &a, bool res, bool res_f32, hipStream_t s) {
    const bool drop = a.drop.below != 0;
    if (!res) drop ? launch<TX, TX, false, true>(a, s) : launch<TX, TX, false, false>(a, s);
    else if (res_f32) drop ? launch<TX, float, true, true>(a, s) : launch<TX, float, true, false>(a, s);
    else drop ? launch<TX, bf16, true, true>(a, s) : launch<TX, bf16, true, false>(a, s);
}

} // namespace

int launch_rms_norm(const EriRmsNorm &e, const Drop &d, void *stream) {
    NormArgs a = {e.x, e.residual, e.weight, e.y, e.h, e.rstd, e.scales, 0, 0, (uint32_t)e.cols,
                  e.x_stride, e.residual_stride, e.y_stride, e.h_stride, e.eps, e.weight_dtype == ERI_DTYPE_F32, (uint32_t)e.y_dtype,
                  (uint32_t)e.scale_group, e.scale_group ? (uint32_t)((e.cols + 127) / 128) : 1u, d};
    hipStream_t s = static_cast<hipStream_t>(stream);
    constexpr uint32_t kMost = 1u << 21; // rows of a launch
    for (a.first = 0; a.first < e.rows; a.first += kMost) {
        a.rows = e.rows - a.first < kMost ? (uint32_t)e.rows : a.first + kMost;
        if (e.x_dtype == ERI_DTYPE_F32) launch_of<float>(a, e.residual != nullptr, e.residual_dtype == ERI_DTYPE_F32, s);
        else launch_of<bf16>(a, e.residual != nullptr, e.residual_dtype == ERI_DTYPE_F32, s);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

} // namespace eri_layers
