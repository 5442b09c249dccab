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
constexpr int kRopeAhead = 4;         // loads of a thread under way together
constexpr int kRopeMaxRows = 16;      // rows of a CTA
constexpr int kRopeMaxAngles = 2048;  // (cos, sin) of a CTA: 16 KB

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

// Elements that a thread moves at once: 16 bytes.
template <typename T>
struct RopeVec {
    static constexpr int N = 16 / sizeof(T);
};

template <typename T>
LC_DEV void unpack(const uint4& w, float (&v)[RopeVec<T>::N]) {
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < RopeVec<T>::N; ++i) v[i] = to_f(e[i]);
}
template <typename T>
LC_DEV void store_vec(T* p, const float (&v)[RopeVec<T>::N]) {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < RopeVec<T>::N; ++i) e[i] = from_f<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = w;
}

// cos and sin of every pair of row r, for all heads.  The angle is reduced in
// fp64 turns: p * t_j carries 2^-53 relative, so its fraction is exact to 2^-22
// of a turn even at p = 2^31, where an fp32 angle would have no correct digit
// left.  What the fraction as an fp32 number leaves out, up to 1.57 units 2^-24
// of the angle, turns (c, s) on by its first order: without it they are off by
// up to 1.93 such units, with it by 1.5 at most.
LC_DEV float2 rope_turn(int p, double t, float mult, float sign) {
    const double x = (double)p * t, f = x - rint(x);
    const float h = (float)f, rest = (float)(f - h) * 6.2831853f;
    float s, c;
    sincospif(2.0f * h, &s, &c);
    return make_float2(__fmaf_rn(-rest, s, c) * mult, __fmaf_rn(rest, c, s) * mult * sign);
}

// Bound by memory.  A CTA takes `R` rows (a part of their heads where rows are
// few); (cos, sin) go to shared memory once per row and pair, and every thread
// moves 16 bytes (two times 16 in the half layout) at one place of the head
// over the rows and heads, so its loads are independent.  The first loads are
// under way while the angles are computed.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kRopeThreads) rope_vec_kernel(RopeApply a, const __grid_constant__ RopeTurns turns, int R, int share) {
    constexpr int N = RopeVec<T>::N;
    extern __shared__ __align__(16) float2 cs[];  // [R][pairs]
    __shared__ int at[kRopeMaxRows];
    const int pairs = a.rot_dim >> 1, rest = a.head_dim - a.rot_dim;
    const int turned = HALF ? pairs / N : a.rot_dim / N;  // places of a head that turn, and those copied
    const bool in_place = a.x == (const void*)a.y;
    const int places = turned + (in_place ? 0 : rest / N);
    const int per = kRopeThreads / places;                 // (row, head) items at a time
    const int place = threadIdx.x % places, item0 = threadIdx.x / places;
    const int row0 = blockIdx.x * R, rows = min(R, a.rows - row0);
    const int h0 = blockIdx.y * share, heads = min(share, a.heads - h0);  // at least one
    griddep_launch();
    griddep_wait();
    if (threadIdx.x < rows) at[threadIdx.x] = a.pos[row0 + threadIdx.x];
    const int items = item0 < per ? rows * heads : 0;
    const bool turn = place < turned;
    const int e0 = turn ? place * N : a.rot_dim + (place - turned) * N;
    const T* x = (const T*)a.x + (int64_t)row0 * a.x_stride + h0 * a.head_dim + e0;
    T* y = (T*)a.y + (int64_t)row0 * a.y_stride + h0 * a.head_dim + e0;
    uint4 u[kRopeAhead], v[kRopeAhead];
    int rl = item0 / heads, hl = item0 - rl * heads;  // row and head of the next load
    int rs = rl, hs = hl;                             // and of the next store
    auto next = [&](int& r, int& h) {
        for (h += per; h >= heads; h -= heads) ++r;
    };
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kRopeAhead; ++k) {
            if (i0 + k * per >= items) continue;
            const T* p = x + (int64_t)rl * a.x_stride + hl * a.head_dim;
            // Plain loads: in place, the kernel writes what it reads here.
            u[k] = *reinterpret_cast<const uint4*>(p);
            if (HALF && turn) v[k] = *reinterpret_cast<const uint4*>(p + pairs);
            next(rl, hl);
        }
    };
    load(item0);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * pairs; i += kRopeThreads) {
        const int r = i / pairs, j = i - r * pairs;
        cs[i] = rope_turn(at[r], turns.t[j], a.mult, a.sign);
    }
    __syncthreads();
    for (int i0 = item0; i0 < items;) {
#pragma unroll
        for (int k = 0; k < kRopeAhead; ++k) {
            if (i0 + k * per >= items) continue;
            const int r = rs;
            T* p = y + (int64_t)r * a.y_stride + hs * a.head_dim;
            next(rs, hs);
            if (at[r] < 0) continue;  // rows without a position are left as they are
            if (!turn) {
                *reinterpret_cast<uint4*>(p) = u[k];
                continue;
            }
            float c[2 * N], f[N], o[N];  // (cos, sin) of N pairs, or of N / 2
            const float4* z = reinterpret_cast<const float4*>(cs + r * pairs + (HALF ? e0 : e0 / 2));
#pragma unroll
            for (int e = 0; e < (HALF ? N / 2 : N / 4); ++e) {
                const float4 w = z[e];
                c[4 * e] = w.x, c[4 * e + 1] = w.y, c[4 * e + 2] = w.z, c[4 * e + 3] = w.w;
            }
            unpack<T>(u[k], f);
            if (HALF) {
                float g[N], q[N];
                unpack<T>(v[k], g);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    o[e] = f[e] * c[2 * e] - g[e] * c[2 * e + 1];
                    q[e] = f[e] * c[2 * e + 1] + g[e] * c[2 * e];
                }
                store_vec(p + pairs, q);
            } else {
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    o[e] = f[e] * c[e] - f[e + 1] * c[e + 1];
                    o[e + 1] = f[e] * c[e + 1] + f[e + 1] * c[e];
                }
            }
            store_vec(p, o);
        }
        i0 += kRopeAhead * per;
        if (i0 < items) load(i0);
    }
}

// Any size, stride and alignment: one CTA per row, one pair per thread.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_any_kernel(RopeApply a, const __grid_constant__ RopeTurns turns) {
    griddep_launch();
    griddep_wait();
    __shared__ float2 cs[kRopeMaxPairs];
    const int pairs = a.rot_dim >> 1;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int p = a.pos[r];
        if (p < 0) continue;  // uniform over the CTA
        __syncthreads();
        for (int j = threadIdx.x; j < pairs; j += blockDim.x) cs[j] = rope_turn(p, turns.t[j], a.mult, a.sign);
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

template <typename T>
cudaError_t launch_rope(const RopeApply& a, const RopeTurns& turns, int num_sms, cudaStream_t st) {
    constexpr int N = RopeVec<T>::N;
    const int pairs = a.rot_dim / 2;
    const bool vec = a.rot_dim > 0 && (a.half ? pairs : a.rot_dim) % N == 0 && (a.head_dim - a.rot_dim) % N == 0 &&
                     a.head_dim / N <= kRopeThreads && pairs % 2 == 0 &&
                     (((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)(a.x_stride * sizeof(T)) | (uintptr_t)(a.y_stride * sizeof(T))) & 15) == 0;
    if (!vec) {
        const int grid = a.rows < num_sms * 8 ? a.rows : num_sms * 8;
        return launch_ex(rope_any_kernel<T>, dim3(grid), dim3(kRopeThreads), 0, st, true, a, turns);
    }
    // A thread's loads cover `work` (row, head) items of a CTA.  Rows are
    // taken together while four CTAs remain for every SM; with fewer rows
    // than that a row's heads are shared out instead.
    const int places = (a.half ? pairs : a.rot_dim) / N + (a.x == (const void*)a.y ? 0 : (a.head_dim - a.rot_dim) / N);
    const int work = kRopeAhead * (kRopeThreads / places);
    int R = (2 * work + a.heads - 1) / a.heads, parts = 1;
    while (R > 1 && a.rows / R < 4 * num_sms) R = (R + 1) / 2;
    if (R > kRopeMaxRows) R = kRopeMaxRows;
    if (R * pairs > kRopeMaxAngles) R = kRopeMaxAngles / pairs;
    if (R == 1)
        while (parts < a.heads && (int64_t)a.rows * parts * 2 <= 2 * num_sms && a.heads / (parts * 2) >= kRopeThreads / places) parts *= 2;
    const int share = (a.heads + parts - 1) / parts;
    const dim3 grid((a.rows + R - 1) / R, (a.heads + share - 1) / share), block(kRopeThreads);
    const size_t smem = (size_t)R * pairs * sizeof(float2);
    return a.half ? launch_ex(rope_vec_kernel<T, true>, grid, block, smem, st, true, a, turns, R, share)
                  : launch_ex(rope_vec_kernel<T, false>, grid, block, smem, st, true, a, turns, R, share);
}

}  // namespace

cudaError_t launch_rope_apply(const RopeApply& a, const RopeTurns& turns, int num_sms, cudaStream_t st) {
    return a.dtype == kRowF32 ? launch_rope<float>(a, turns, num_sms, st) : launch_rope<__half>(a, turns, num_sms, st);
}

}  // namespace lc
