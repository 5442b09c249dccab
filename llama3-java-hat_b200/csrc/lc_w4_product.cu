// lc_w4_product.cu -- y = x W^T (+ a residual) with 4-bit weights (lc_w4.h).
//
// y[b][r] = sum over groups of s[r][group] * sum over its columns of (c - z) x.
// The inner sums are of whole numbers times x; a group's scale is applied once.
#include "lc_internal.h"
#include "lc_w4.h"

namespace lc {
namespace {

constexpr int kSimpleRows = 128, kSimpleBatch = 8;

template <typename T>
LC_DEV float w4_f32(T v) { return (float)v; }

template <typename T>
__global__ void __launch_bounds__(kSimpleRows) w4_simple_kernel(W4 w, W4Product p) {
    __shared__ float xs[kSimpleBatch][kW4Cols];
    const int row = blockIdx.x * kSimpleRows + threadIdx.x, b0 = blockIdx.y * kSimpleBatch;
    const int tile = row / kW4Rows, r = row % kW4Rows, g = r & 7, up = r >> 3, ng = kW4Cols / w.group;
    const T* x = (const T*)p.x;
    float total[kSimpleBatch] = {};
    for (int block = 0; block < w.blocks; ++block) {
        __syncthreads();
        for (int i = threadIdx.x; i < kSimpleBatch * kW4Cols; i += kSimpleRows) {
            const int b = i / kW4Cols, c = block * kW4Cols + i % kW4Cols;
            xs[b][i % kW4Cols] = b0 + b < p.batch && c < w.cols ? w4_f32(x[(b0 + b) * p.x_stride + c]) : 0.0f;
        }
        __syncthreads();
        if (tile >= w.tiles) continue;
        const int64_t u = (int64_t)tile * w.blocks + block;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(w.codes + u * kW4BlockBytes);
        for (int i = 0; i < ng; ++i) {
            const int64_t at = ((u * 8 + g) * ng + i) * 2 + up;
            const float s = __half2float(__ushort_as_half(w.scales[at]));
            const int zero = w.zeros ? w.zeros[at] : 8;
            float sum[kSimpleBatch] = {};
            for (int c = i * w.group; c < (i + 1) * w.group; ++c) {
                const int e = c & 3, bit = (e & 1 ? 16 : 0) + (e & 2 ? 8 : 0) + 4 * up;
                const uint32_t word = words[(c >> 6) * 128 + (4 * g + ((c >> 4) & 3)) * 4 + ((c >> 2) & 3)];
                const float v = (float)((int)((word >> bit) & 15u) - zero);
#pragma unroll
                for (int b = 0; b < kSimpleBatch; ++b) sum[b] = fmaf(v, xs[b][c], sum[b]);
            }
#pragma unroll
            for (int b = 0; b < kSimpleBatch; ++b) total[b] = fmaf(s, sum[b], total[b]);
        }
    }
    if (row >= w.rows) return;
    for (int b = 0; b < kSimpleBatch && b0 + b < p.batch; ++b) {
        float v = total[b];
        if (p.residual) v += w4_f32(((const T*)p.residual)[(b0 + b) * p.residual_stride + row]);
        ((T*)p.y)[(b0 + b) * p.y_stride + row] = (T)v;
    }
}

}  // namespace

cudaError_t launch_w4_product(const W4& w, const W4Product& p, int, cudaStream_t st) {
    const dim3 grid((w.rows + kSimpleRows - 1) / kSimpleRows, (p.batch + kSimpleBatch - 1) / kSimpleBatch);
    if (p.dtype == kRowF32) w4_simple_kernel<float><<<grid, kSimpleRows, 0, st>>>(w, p);
    else w4_simple_kernel<__half><<<grid, kSimpleRows, 0, st>>>(w, p);
    return cudaGetLastError();
}

}  // namespace lc
