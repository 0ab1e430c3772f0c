/*
 * Gradient of the residual addition and root-mean-square norm of include/eri_layers.h:
 *     dh = dr + q dy w - h q^3 mean(dy w h),  dx = drop(dh),  dw = sum over rows of dy h q
 * computed as c = q (q mean(dy w h)), dh = dr + q (dy w - h c): q^3 leaves fp32 for rows of 1e-13 and is lost for rows of 1e15, while
 * q mean(dy w h) and h c are of the order of dy w whatever the rows' size.
 *
 * Bound by HBM: dy, h and dr are read once, dh and dx written once; the row waits in registers for its sum, and each thread keeps
 * the weight and the sums of dw of its columns over all rows that its workgroup takes.  The workgroups' sums (two a compute
 * unit) are joined by a second kernel in their order, so that the same inputs give the same bits; few rows do without it.
 * 16384 x 4096 bf16 with dropout 131 us, 5.1 TB/s (a copy of that size runs at 5.2); 1025 x 1281 fp32 7.5 + 3.5 us.
 * Tried: the next row's loads before this row's sum (level or 1-25 % slower: the registers cost waves), four workgroups a unit.
 */
#include "eri_layers_device.h"

namespace eri_layers {
namespace {

struct NormGradArgs {
    const void *grad, *h, *weight, *grad_h;
    const float *rstd;
    void *grad_x, *grad_residual;
    float *partial;    // per workgroup a row of grad_weight's sums, padded floats apart; NULL: not wanted
    void *grad_weight; // few rows: written by the workgroups behind the first row_groups; NULL otherwise
    uint32_t rows, cols, padded, row_groups, grad_weight_f32;
    uint64_t grad_stride, h_stride, grad_h_stride, grad_x_stride, grad_residual_stride;
    uint32_t weight_f32, x_f32;
    Drop drop;
};

constexpr uint32_t kRowsOf(int tpr) { return tpr < 256 ? 256 / tpr : 1; }

template <typename TR, bool DROP>
__device__ __forceinline__ void store_grads(const NormGradArgs &a, uint32_t row, uint32_t col, float (&dh)[8], uint64_t offset) {
    if (a.grad_residual) store8((TR *)a.grad_residual + row * a.grad_residual_stride, col, a.cols, dh);
    if (!a.grad_x) return;
    if (DROP) {
        const u32x4 bits = draw8((uint64_t)row * a.cols + col, a.drop, offset);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) dh[e] = dropped(dh[e], bits, e, a.drop);
    }
    if (a.x_f32) store8((float *)a.grad_x + row * a.grad_x_stride, col, a.cols, dh);
    else store8((bf16 *)a.grad_x + row * a.grad_x_stride, col, a.cols, dh);
}

/* grad_weight of 32 columns over all rows: four lanes to a row's part of them, the rest of the workgroup side by side, and their
 * sums joined in their order. */
template <typename TG, typename TR, bool SHORT, int THREADS> __device__ __forceinline__ void weight_of_columns(const NormGradArgs &a, uint32_t tile) {
    __shared__ float sums[THREADS / 4][32];
    const uint32_t part = threadIdx.x / 4, in = threadIdx.x % 4 * 8, col = tile * 32 + in;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t row = part; row < a.rows; row += THREADS / 4) {
        Raw<TG> g;
        Raw<TR> h;
        load8<SHORT>(g, (const TG *)a.grad + row * a.grad_stride, col, a.cols);
        load8<SHORT>(h, (const TR *)a.h + row * a.h_stride, col, a.cols);
        const float rstd = a.rstd[row];
        settle8<SHORT>(g, col, a.cols);
        settle8<SHORT>(h, col, a.cols);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = fmaf(g.get(e) * h.get(e), rstd, v[e]);
    }
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) sums[part][in + e] = v[e];
    __syncthreads();
    const uint32_t c = tile * 32 + threadIdx.x;
    if (threadIdx.x >= 32 || c >= a.cols) return;
    float total = 0.0f;
    for (uint32_t p = 0; p < THREADS / 4; ++p) total += sums[p][threadIdx.x];
    if (a.grad_weight_f32) ((float *)a.grad_weight)[c] = total;
    else ((bf16 *)a.grad_weight)[c].bits = (uint16_t)bf16_pair(total, 0.0f);
}

/* A row at a time to TPR threads, which keep the weight and their columns' sums of grad_weight in registers. */
template <typename TG, typename TR, bool DROP, int TPR, int NV, bool SHORT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_grad_kernel(const NormGradArgs a) {
    __shared__ float slots[2][kSlots<TPR>];
    __shared__ float joined[TPR < 256 ? TPR * NV * 8 : 1];
    if (blockIdx.x >= a.row_groups) return weight_of_columns<TG, TR, SHORT, TPR < 256 ? 256 : TPR>(a, blockIdx.x - a.row_groups);
    const uint32_t t = threadIdx.x % TPR;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    float w[NV][8], acc[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (a.weight) load8_of<SHORT>(w[k], a.weight, a.weight_f32, (k * TPR + t) * 8, a.cols);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            acc[k][e] = 0.0f;
            if (!a.weight) w[k][e] = 1.0f;
        }
    }
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x * kRowsOf(TPR) + threadIdx.x / TPR; row < a.rows; row += a.row_groups * kRowsOf(TPR), turn ^= 1) {
        Raw<TG> g[NV];
        Raw<TR> h[NV], r[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            load8<SHORT>(g[k], (const TG *)a.grad + row * a.grad_stride, (k * TPR + t) * 8, a.cols);
            load8<SHORT>(h[k], (const TR *)a.h + row * a.h_stride, (k * TPR + t) * 8, a.cols);
        }
        if (a.grad_h)
#pragma unroll
            for (int k = 0; k < NV; ++k) load8<SHORT>(r[k], (const TR *)a.grad_h + row * a.grad_h_stride, (k * TPR + t) * 8, a.cols);
        else
#pragma unroll
            for (int k = 0; k < NV; ++k) r[k].clear();
        const float rstd = a.rstd[row];
        float c = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            settle8<SHORT>(g[k], (k * TPR + t) * 8, a.cols);
            settle8<SHORT>(h[k], (k * TPR + t) * 8, a.cols);
            settle8<SHORT>(r[k], (k * TPR + t) * 8, a.cols);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const float gh = g[k].get(e) * h[k].get(e);
                c = fmaf(gh, w[k][e], c);
                acc[k][e] = fmaf(gh, rstd, acc[k][e]);
            }
        }
        c = sum_over<TPR>(c, slots[turn]) * rstd / (float)a.cols * rstd;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float dh[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) dh[e] = fmaf(fmaf(-h[k].get(e), c, g[k].get(e) * w[k][e]), rstd, r[k].get(e));
            store_grads<TR, DROP>(a, row, (k * TPR + t) * 8, dh, offset);
        }
    }
    if (!a.partial) return;
    if (TPR < 256) { // the waves' sums, one after the other
        for (uint32_t turn = 0; turn < kRowsOf(TPR); ++turn) {
            if (threadIdx.x / TPR == turn)
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float *j = joined + (k * 8 + e) * TPR + t;
                        *j = acc[k][e] += turn ? *j : 0.0f;
                    }
            __syncthreads();
        }
        if (threadIdx.x / TPR != kRowsOf(TPR) - 1) return;
    }
    float *out = a.partial + (uint64_t)blockIdx.x * a.padded;
#pragma unroll
    for (int k = 0; k < NV; ++k) store8(out, (k * TPR + t) * 8, a.padded, acc[k]);
}

/* Rows too long for registers (with 32 elements of four rows in each of 1024 threads the compiler spills 200 of them, and 4096 x 20000
 * bf16 took 535 us; this takes 254; with 16 elements, up to 16384 columns, it spills two, in fp32 only): read twice, and the sums of grad_weight kept in the workgroup's row of partial. */
template <typename TG, typename TR, bool DROP> __global__ __launch_bounds__(1024) void rms_norm_grad_long_kernel(const NormGradArgs a) {
    __shared__ float slots[2][16];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    float *out = a.partial ? a.partial + (uint64_t)blockIdx.x * a.padded : nullptr;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const float rstd = a.rstd[row];
        float c = 0.0f;
        for (uint32_t col = threadIdx.x * 8; col < a.cols; col += 8192) {
            Raw<TG> g;
            Raw<TR> h;
            float w[8], gh[8];
            load8<false>(g, (const TG *)a.grad + row * a.grad_stride, col, a.cols);
            load8<false>(h, (const TR *)a.h + row * a.h_stride, col, a.cols);
            if (a.weight) load8_of<false>(w, a.weight, a.weight_f32, col, a.cols);
            settle8<false>(g, col, a.cols);
            settle8<false>(h, col, a.cols);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                gh[e] = g.get(e) * h.get(e);
                c = fmaf(gh[e], a.weight ? w[e] : 1.0f, c);
            }
            if (out) {
                float old[8];
                load8_of<false>(old, out, true, col, a.padded);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) old[e] = row == blockIdx.x ? gh[e] * rstd : fmaf(gh[e], rstd, old[e]);
                store8(out, col, a.padded, old);
            }
        }
        c = sum_over<1024>(c, slots[turn]) * rstd / (float)a.cols * rstd;
        for (uint32_t col = threadIdx.x * 8; col < a.cols; col += 8192) {
            Raw<TG> g;
            Raw<TR> h, r;
            float w[8], dh[8];
            load8<false>(g, (const TG *)a.grad + row * a.grad_stride, col, a.cols);
            load8<false>(h, (const TR *)a.h + row * a.h_stride, col, a.cols);
            if (a.grad_h) load8<false>(r, (const TR *)a.grad_h + row * a.grad_h_stride, col, a.cols);
            else r.clear();
            if (a.weight) load8_of<false>(w, a.weight, a.weight_f32, col, a.cols);
            settle8<false>(g, col, a.cols);
            settle8<false>(h, col, a.cols);
            settle8<false>(r, col, a.cols);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) dh[e] = fmaf(fmaf(-h.get(e), c, a.weight ? g.get(e) * w[e] : g.get(e)), rstd, r.get(e));
            store_grads<TR, DROP>(a, row, col, dh, offset);
        }
    }
}

/* grad_weight out of the workgroups' sums: 64 columns to a workgroup, 64 groups of rows, joined in their order. */
__global__ __launch_bounds__(1024) void rms_norm_grad_weight_kernel(const float *partial, uint32_t n, uint32_t padded, void *out, uint32_t cols, uint32_t out_f32) {
    __shared__ float sums[64][64];
    const uint32_t quad = threadIdx.x % 16, part = threadIdx.x / 16, col = blockIdx.x * 64 + quad * 4;
    float s[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t r = part; r < n; r += 64) {
        const float4 v = *(const float4 *)(partial + (uint64_t)r * padded + col);
        s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[part][quad * 4 + e] = s[e];
    __syncthreads();
    const uint32_t c = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x >= 64 || c >= cols) return;
    float total = 0.0f;
    for (uint32_t p = 0; p < 64; ++p) total += sums[p][threadIdx.x];
    if (out_f32) ((float *)out)[c] = total;
    else ((bf16 *)out)[c].bits = (uint16_t)bf16_pair(total, 0.0f);
}

/* Few rows: grad_weight comes out of the same launch, from workgroups that read grad and h once more, instead of a second one
 * over the sums that the rows' workgroups leave.  One line for all widths over 512 columns lies between those where one launch
 * wins for longer (4096 bf16) and those where it stops winning earlier (8192 fp32), 2 us to either side.  us, one launch | two, at so
 * many rows:
 *   rows            128          512          768          1024         1536
 *   256 bf16     5.8 | 9.0    5.8 | 9.1    6.0 | 9.0    5.9 | 9.1    6.1 | 9.3
 *   1024 fp32    5.8 | 8.9    5.6 | 8.9    6.6 | 8.8    8.7 | 9.2   11.3 | 10.4
 *   1281 bf16    5.5 | 9.0    6.1 | 8.9    8.4 | 9.4   10.5 | 9.6   14.7 | 10.6
 *   4096 bf16    5.4 | 8.8    6.7 | 12.5   9.3 | 13.6  11.8 | 13.8  16.6 | 15.5
 *   8192 fp32    5.8 | 10.5  17.6 | 20.1  28.6 | 26.1  34.0 | 31.4  48.3 | 42.2 */
bool is_few(uint64_t rows, uint64_t cols) { return rows <= (cols <= 512 ? 1536 : 768); }

/* Threads to a row, and how many workgroups the rows are dealt to.  512 threads to a row of 2049 to 8192 columns: with 256 and twice
 * as much of it each, 2048 x 4096 bf16 took 18.2 us for 17.1, 2048 x 8192 30.1 for 28.0, 256 x 8192 7.6 for 6.8; with 1024 to a row of
 * 8192 26.5, but 256 rows 9.4. */
struct Shape {
    int tpr, nv; // nv 0: rows too long for registers
    uint32_t groups;
};
Shape shape_of(uint64_t rows, uint64_t cols, uint32_t compute_units) {
    Shape s = cols <= 128 ? Shape{16, 1, 0} : cols <= 256 ? Shape{32, 1, 0} : cols <= 512 ? Shape{64, 1, 0} : cols <= 1024 ? Shape{64, 2, 0} : cols <= 2048 ? Shape{256, 1, 0} : cols <= 4096 ? Shape{512, 1, 0} :
              cols <= 8192 ? Shape{512, 2, 0} : cols <= 16384 ? Shape{1024, 2, 0} : Shape{1024, 0, 0};
    const uint64_t all = (rows + kRowsOf(s.tpr) - 1) / kRowsOf(s.tpr), most = (uint64_t)compute_units * (s.tpr == 1024 ? 1 : 2); // more of them leave more sums to read again: with 4, 3-15 % slower
    s.groups = (uint32_t)(all < most ? all : most);
    return s;
}
uint64_t padded_of(uint64_t cols) { return (cols + 63) / 64 * 64; }

template <typename TG, typename TR, bool DROP> void launch(const NormGradArgs &a, const Shape &shape, hipStream_t s) {
    const uint32_t groups = shape.groups + (a.grad_weight ? a.padded / 32 : 0);
#define ERI_NORM_GRAD(TPR, NV, SHORT) \
    if (shape.tpr == TPR && shape.nv == NV && SHORT == (a.cols < 8)) \
    hipLaunchKernelGGL((rms_norm_grad_kernel<TG, TR, DROP, TPR, NV, SHORT>), dim3(groups), dim3(TPR < 256 ? 256 : TPR), 0, s, a)
    ERI_NORM_GRAD(16, 1, true);
    ERI_NORM_GRAD(16, 1, false);
    ERI_NORM_GRAD(32, 1, false);
    ERI_NORM_GRAD(64, 1, false);
    ERI_NORM_GRAD(64, 2, false);
    ERI_NORM_GRAD(256, 1, false);
    ERI_NORM_GRAD(512, 1, false);
    ERI_NORM_GRAD(512, 2, false);
    ERI_NORM_GRAD(1024, 2, false);
#undef ERI_NORM_GRAD
    if (shape.nv == 0) hipLaunchKernelGGL((rms_norm_grad_long_kernel<TG, TR, DROP>), dim3(shape.groups), dim3(1024), 0, s, a);
}

template <typename TG> void launch_of(const NormGradArgs &a, bool h_f32, const Shape &shape, hipStream_t s) {
    if (h_f32) a.drop.below ? launch<TG, float, true>(a, shape, s) : launch<TG, float, false>(a, shape, s);
    else a.drop.below ? launch<TG, bf16, true>(a, shape, s) : launch<TG, bf16, false>(a, shape, s);
}

} // namespace

uint64_t rms_norm_grad_workspace(uint64_t rows, uint64_t cols, uint32_t compute_units) {
    return shape_of(rows, cols, compute_units).groups * padded_of(cols) * sizeof(float);
}

int launch_rms_norm_grad(const EriRmsNormGrad &e, const Drop &d, uint32_t compute_units, void *stream) {
    const Shape shape = shape_of(e.rows, e.cols, compute_units);
    const uint32_t padded = (uint32_t)padded_of(e.cols);
    // Where that saves the second launch, grad and h are read by other workgroups too, and grad_weight is written while weight is
    // still read: not when one of them is being replaced.
    auto over = [&](const void *out, const void *in) { return out && out == in; };
    const bool replaces = over(e.grad_x, e.grad) || over(e.grad_x, e.h) || over(e.grad_residual, e.grad) || over(e.grad_residual, e.h) || over(e.grad_weight, e.weight);
    const bool few = e.grad_weight && e.rows && is_few(e.rows, e.cols) && shape.nv && !replaces;
    float *partial = e.grad_weight && !few ? (float *)e.workspace : nullptr;
    const NormGradArgs a = {e.grad, e.h, e.weight, e.grad_h, e.rstd, e.grad_x, e.grad_residual, partial, few ? e.grad_weight : nullptr, (uint32_t)e.rows,
                            (uint32_t)e.cols, padded, shape.groups, e.grad_weight_dtype == ERI_DTYPE_F32, e.grad_stride, e.h_stride, e.grad_h_stride, e.grad_x_stride,
                            e.grad_residual_stride, e.weight_dtype == ERI_DTYPE_F32, e.x_dtype == ERI_DTYPE_F32, d};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (e.rows) {
        if (e.grad_dtype == ERI_DTYPE_F32) launch_of<float>(a, e.h_dtype == ERI_DTYPE_F32, shape, s);
        else launch_of<bf16>(a, e.h_dtype == ERI_DTYPE_F32, shape, s);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    const uint32_t w32 = e.grad_weight_dtype == ERI_DTYPE_F32;
    constexpr uint32_t kMost = 1u << 27; // columns of a launch: its threads are counted in 32 bits, 16 for each
    for (uint32_t at = 0; e.grad_weight && !few && at < padded; at += kMost) {
        const uint32_t now = padded - at < kMost ? padded - at : kMost;
        hipLaunchKernelGGL(rms_norm_grad_weight_kernel, dim3(now / 64), dim3(1024), 0, s, partial + at, shape.groups, padded, (char *)e.grad_weight + (uint64_t)at * (w32 ? 4 : 2),
                           (uint32_t)e.cols - at, w32);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

} // namespace eri_layers
