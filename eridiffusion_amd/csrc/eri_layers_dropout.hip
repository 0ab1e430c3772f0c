/*
 * Dropout of include/eri_layers.h: y = keep ? x / share : 0, the mask drawn from Philox4x32-10 where it is needed.
 *
 * One pass, 2 bytes read and 2 written per bf16 element; bound by HBM.  Eight elements share one call of the generator, 16 bits
 * each: with 32 bits it would be twice the calls, twenty 32x32->64 products each.  What that costs is that p counts in
 * steps of 1/65536; what is kept is divided by the share that is really kept, so the mean is exact.  16384 x 8192 bf16 takes 92 us,
 * 5.8 TB/s, where a copy of that size runs at 5.2; 1024 x 1280 takes 3.2 us, most of it the launch and one trip to memory.
 */
#include "eri_layers_device.h"

namespace eri_layers {
namespace {

constexpr uint32_t kThreads = 256;

struct DropoutArgs {
    const void *x;
    void *y;
    uint64_t cols, vectors; // vectors: of a row
    uint32_t rows;
    uint64_t x_stride, y_stride;
    Drop drop;
};

template <typename T, bool SHORT> __global__ __launch_bounds__(kThreads) void dropout_kernel(const DropoutArgs a) {
    const uint64_t offset = drop_offset(a.drop);
    for (uint32_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const T *x = (const T *)a.x + row * a.x_stride;
        T *y = (T *)a.y + row * a.y_stride;
        for (uint64_t v = (uint64_t)blockIdx.x * kThreads + threadIdx.x; v < a.vectors; v += (uint64_t)gridDim.x * kThreads) {
            const uint64_t col = v * 8;
            Raw<T> r;
            load8<SHORT>(r, x, col, a.cols);
            const u32x4 bits = draw8(row * a.cols + col, a.drop, offset);
            settle8<SHORT>(r, col, a.cols);
            float out[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) out[e] = dropped(r.get(e), bits, e, a.drop);
            store8(y, col, a.cols, out);
        }
    }
}

} // namespace

int launch_dropout(const EriDropout &e, const Drop &d, uint32_t compute_units, void *stream) {
    DropoutArgs a = {e.x, e.y, e.cols, 0, (uint32_t)e.rows, e.x_stride, e.y_stride, d};
    if (e.x_stride == e.cols && e.y_stride == e.cols) { // no gaps: one long row
        a.cols = e.rows * e.cols;
        a.rows = 1;
    }
    a.vectors = (a.cols + 7) / 8;
    const uint64_t x = (a.vectors + kThreads - 1) / kThreads, most = (uint64_t)compute_units * 64;
    const uint64_t across = x < most ? x : most, down = most / across; // of workgroups; the rest in turn
    const dim3 grid((uint32_t)across, (uint32_t)(a.rows < down ? a.rows : down));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = e.dtype_tag == ERI_DTYPE_F32, is_short = a.cols < 8;
    void (*const kernel)(const DropoutArgs) = f32 ? is_short ? dropout_kernel<float, true> : dropout_kernel<float, false>
                                                  : is_short ? dropout_kernel<bf16, true> : dropout_kernel<bf16, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a);
    return (int)hipGetLastError();
}

} // namespace eri_layers
