// lc_rope.cu -- rotary positions with the layouts and frequency scalings of
// long-context models, and their transposed map.
//
// Pair j of a head at position p turns by p * f_j: (a, b) -> m (a cos - b sin,
// a sin + b cos); the transposed map (the gradient) turns the other way under
// the same factor m.  The rest of the head (rot_dim..head_dim) is copied.
#include "lc_internal.h"
#include "lc_paged.h"

namespace lc {
namespace {

constexpr int kRopeThreads = 256;

template <typename T>
LC_DEV float to_f(T v);
template <>
LC_DEV float to_f<float>(float v) { return v; }
template <>
LC_DEV float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
LC_DEV T from_f(float v);
template <>
LC_DEV float from_f<float>(float v) { return v; }
template <>
LC_DEV __half from_f<__half>(float v) { return __float2half_rn(v); }

// One CTA per row: (cos, sin) of the row's pairs go to shared memory once,
// for all heads.  The angle is reduced in fp64 turns: p * t_j carries 2^-53
// relative, so its fraction is exact to 2^-22 of a turn even at p = 2^31,
// where an fp32 angle would have no correct digit left.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_apply_kernel(RopeApply a, const __grid_constant__ RopeTurns turns) {
    griddep_launch();
    griddep_wait();
    __shared__ float2 cs[kRopeMaxPairs];
    const int pairs = a.rot_dim >> 1;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int p = a.pos[r];
        if (p < 0) continue;  // uniform over the CTA
        __syncthreads();
        for (int j = threadIdx.x; j < pairs; j += blockDim.x) {
            const double t = (double)p * turns.t[j];
            float s, c;
            sincospif(2.0f * (float)(t - rint(t)), &s, &c);
            cs[j] = make_float2(c * a.mult, s * a.mult * a.sign);
        }
        __syncthreads();
        const T* x = (const T*)a.x + (int64_t)r * a.x_stride;
        T* y = (T*)a.y + (int64_t)r * a.y_stride;
        for (int i = threadIdx.x; i < a.heads * pairs; i += blockDim.x) {
            const int h = i / pairs, j = i - h * pairs;
            const int at = h * a.head_dim + (a.half ? j : 2 * j), bt = at + (a.half ? pairs : 1);
            const float u = to_f(x[at]), v = to_f(x[bt]);
            y[at] = from_f<T>(u * cs[j].x - v * cs[j].y);
            y[bt] = from_f<T>(u * cs[j].y + v * cs[j].x);
        }
        const int rest = a.head_dim - a.rot_dim;
        if (rest && (const void*)x != (const void*)y)
            for (int i = threadIdx.x; i < a.heads * rest; i += blockDim.x) {
                const int h = i / rest, k = h * a.head_dim + a.rot_dim + i - h * rest;
                y[k] = x[k];
            }
    }
}

}  // namespace

cudaError_t launch_rope_apply(const RopeApply& a, const RopeTurns& turns, int num_sms, cudaStream_t st) {
    const int grid = a.rows < num_sms * 8 ? a.rows : num_sms * 8;
    if (a.dtype == kRowF32)
        return launch_ex(rope_apply_kernel<float>, dim3(grid), dim3(kRopeThreads), 0, st, true, a, turns);
    return launch_ex(rope_apply_kernel<__half>, dim3(grid), dim3(kRopeThreads), 0, st, true, a, turns);
}

}  // namespace lc
