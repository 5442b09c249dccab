// lc_w4.cu -- 4-bit weights: quantising rows of values, packing codes that a
// checkpoint holds, and reading values back.  Layout: lc_w4.h.
//
// A warp has a block of 16 rows x 128 columns, a lane four runs of eight columns
// of two rows, as the layout wants them; a group's largest value is then a
// maximum over 4 lanes and 1, 2 or 4 of their runs.  With s the group's scale,
// every code is the nearest to the exact quotient x / s, ties to even.  x times a
// number below 1 / s and x times one above it lie on both sides of the quotient:
// where they round to the same whole number, it is the code (two FMAs, which add
// 1.5 * 2^23 and the zero point at once, so that the code is the sum's low bits; a
// multiplication puts them in their place).  Only a run of eight that has others,
// or a group of unusual scale, divides by the exact remainder.
//
// Bound by memory: values in once, codes out once, and the reverse.
#include "lc_internal.h"
#include "lc_w4.h"

namespace lc {
namespace {

constexpr int kW4Threads = 256;
constexpr int kW4Warps = kW4Threads / 32;
constexpr int kW4Half = 64;            // columns of half a block
constexpr int kW4Pitch = kW4Half + 4;  // floats between rows of the exchange buffer

LC_DEV uint32_t turned(uint32_t w) { return __funnelshift_l(w, w, kW4Turn); }
LC_DEV uint32_t unturned(uint32_t w) { return __funnelshift_r(w, w, kW4Turn); }

template <typename T>
LC_DEV float to_f32(T v);
template <>
LC_DEV float to_f32<float>(float v) { return v; }
template <>
LC_DEV float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
LC_DEV T from_f32(float v);
template <>
LC_DEV float from_f32<float>(float v) { return v; }
template <>
LC_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }

// (a + b) / 15 for a, b >= 0, correctly rounded in 64 bits, as fp32: the remainder
// of a first quotient by the rounded reciprocal corrects it.
LC_DEV float fifteenth(float a, float b) {
    constexpr double r = 1.0 / 15.0;
    const double n = (double)a + (double)b, q = n * r;
    return (float)__fma_rn(__fma_rn(-q, 15.0, n), r, q);
}

// Nearest whole number to x / s, ties to even, for |x / s| <= 2^20: `near` is
// at most one off.
LC_DEV float settle(float x, float s, float near) {
    const float rest = __fmaf_rn(-near, s, x);  // exact where it matters: at most one step, in units of x's
    const float a = 2.0f * fabsf(rest);
    const bool odd = (static_cast<int>(near) & 1) != 0;
    return a > s || (a == s && odd) ? near + copysignf(1.0f, rest) : near;
}

// Quotients of eight values as whole numbers in [-16, 16].
LC_DEV void quotients(const float (&x)[8], float s, float inv, float (&q)[8]) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
    const float sure = s * (0.5f - 0x1p-16f);
    bool all = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = fminf(fmaxf(x[i] * inv, -16.0f), 16.0f);
        q[i] = (t + kMagic) - kMagic;
        all = all && fabsf(__fmaf_rn(-q[i], s, x[i])) < sure;
    }
    if (all) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (fabsf(q[i]) < 16.0f) q[i] = settle(x[i], s, q[i]);
}

// Eight neighbouring values as they lie in memory.
template <typename T>
struct Run;
template <>
struct Run<float> {
    float4 lo, hi;
    LC_DEV float get(int i) const {
        const float4& v = i < 4 ? lo : hi;
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
    LC_DEV void load(const float* p) { lo = __ldg(reinterpret_cast<const float4*>(p)), hi = __ldg(reinterpret_cast<const float4*>(p) + 1); }
    LC_DEV void shared(const float* p) { lo = *reinterpret_cast<const float4*>(p), hi = *(reinterpret_cast<const float4*>(p) + 1); }
    LC_DEV void none() { lo = hi = make_float4(0, 0, 0, 0); }
    // Largest size; not finite where a value is not.
    LC_DEV float top() const {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(get(i))));
        return m;
    }
    LC_DEV void range(float& low, float& high) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) low = fminf(low, get(i)), high = fmaxf(high, get(i));
    }
};
template <>
struct Run<__half> {
    uint4 w;
    LC_DEV __half2 two(int i) const {
        const uint32_t v = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return *reinterpret_cast<const __half2*>(&v);
    }
    LC_DEV float get(int i) const { return i & 1 ? __high2float(two(i >> 1)) : __low2float(two(i >> 1)); }
    LC_DEV void load(const __half* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
    LC_DEV void shared(const float* p) {
        __half2 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(p[2 * i], p[2 * i + 1]);  // exact
        w = *reinterpret_cast<const uint4*>(h);
    }
    LC_DEV void none() { w = make_uint4(0, 0, 0, 0); }
    LC_DEV float top() const {
        const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(two(0)), __habs2(two(1))), __hmax2_nan(__habs2(two(2)), __habs2(two(3))));
        const __half2 n = __hmax2_nan(m, __lowhigh2highlow(m));
        return __low2float(n);
    }
    LC_DEV void range(float& low, float& high) const {
        const __half2 n = __hmin2(__hmin2(two(0), two(1)), __hmin2(two(2), two(3))), m = __hmax2(__hmax2(two(0), two(1)), __hmax2(two(2), two(3)));
        low = fminf(low, fminf(__low2float(n), __high2float(n)));
        high = fmaxf(high, fmaxf(__low2float(m), __high2float(m)));
    }
};

// The lane's runs of half a block: columns col0 + 32 q + 8 t and on, of its rows g
// (a) and g + 8 (b): read by the lane itself where 16-byte loads may be used, else
// row by row through shared memory, so that neighbours read neighbours.
template <typename T>
LC_DEV void load_half(const T* p, int64_t stride, int row0, int rows, int col0, int cols, bool vec, float* buf, int lane,
                      Run<T> (&a)[2], Run<T> (&b)[2]) {
    const int g = lane >> 2, t = lane & 3;
    if (vec && col0 + kW4Half <= cols) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const T* from = p + (row0 + g) * stride + col0 + 32 * q + 8 * t;
            a[q].none(), b[q].none();
            if (row0 + g < rows) a[q].load(from);
            if (row0 + g + 8 < rows) b[q].load(from + 8 * stride);
        }
        return;
    }
    __syncwarp();
    const T* from = p + row0 * stride + col0 + lane;
    const bool one = col0 + lane < cols, two = col0 + 32 + lane < cols;
    T v[kW4Rows][2];
#pragma unroll
    for (int r = 0; r < kW4Rows; ++r) {
        const bool there = row0 + r < rows;
        v[r][0] = there && one ? from[0] : (T)0.0f;
        v[r][1] = there && two ? from[32] : (T)0.0f;
        from += stride;
    }
#pragma unroll
    for (int r = 0; r < kW4Rows; ++r) {
        buf[r * kW4Pitch + lane] = to_f32<T>(v[r][0]);
        buf[r * kW4Pitch + 32 + lane] = to_f32<T>(v[r][1]);
    }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        a[q].shared(buf + g * kW4Pitch + 32 * q + 8 * t);
        b[q].shared(buf + (g + 8) * kW4Pitch + 32 * q + 8 * t);
    }
}

// Scale, its bits and the zero point of a group from its smallest and largest
// finite values, which are at most and at least 0.
struct Step {
    float s, zero;
    uint16_t bits;
};
template <bool ZEROS>
LC_DEV Step step_of(float low, float high) {
    Step o;
    const float step = ZEROS ? fifteenth(-low, high) : __fdiv_rn(fmaxf(-low, high), 7.0f);
    const __half h = __float2half_rn(fminf(step, 65504.0f));
    o.bits = __half_as_ushort(h);
    o.s = __half2float(h);
    o.zero = 8.0f;
    if (ZEROS) {
        o.zero = 0.0f;
        if (o.s > 0.0f) {
            const float near = rintf(fminf(__fdiv_rn(-low, o.s), 16.0f));
            o.zero = near < 16.0f ? fminf(settle(-low, o.s, near), 15.0f) : 15.0f;
        }
    }
    return o;
}

// Codes of a run under a group's scale: eight nibbles, that of value i at bit 4 i.
template <typename T, bool ZEROS>
LC_DEV void encode(const Run<T>& run, const Step& st, bool usual, float below, float above, uint32_t (&code)[8]) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
    const float base = kMagic + st.zero, end = kMagic + 15.0f;
    bool sure = usual;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = run.get(i);
        float m = __fmaf_rn(x, below, base);
        sure = sure && m == __fmaf_rn(x, above, base);
        if (ZEROS) m = fminf(m, end);
        code[i] = __float_as_uint(m) - 0x4b400000u;
    }
    if (sure) return;
    float v[8], q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = run.get(i), q[i] = 0.0f;
        if (!(v[i] == v[i])) v[i] = 0.0f;
    }
    if (st.s > 0.0f) quotients(v, st.s, __frcp_rn(st.s), q);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        code[i] = (uint32_t)(ZEROS ? fminf(fmaxf(q[i] + st.zero, 0.0f), 15.0f) : fminf(fmaxf(q[i], -7.0f), 7.0f) + 8.0f);
}

// Four CTAs of an SM, at the price of a few spilled registers, hide more of the
// loads' latency than two (32003 x 2085 fp32 with the read 264 against 191 us), but
// for F32 groups of 128, whose 64 values a lane keeps (124 against 147).
template <typename T, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4Threads, GROUP == 128 && sizeof(T) == 4 ? 2 : 4) w4_quantize_kernel(W4 w, const T* __restrict__ values, int64_t stride, bool vec) {
    __shared__ __align__(16) float buf[kW4Warps][kW4Rows * kW4Pitch];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    constexpr int NG = kW4Cols / GROUP;           // groups of a block
    constexpr int HALVES = GROUP == 128 ? 2 : 1;  // of a block, taken together
    constexpr int GROUPS = HALVES * kW4Half / GROUP > 0 ? HALVES * kW4Half / GROUP : 1, RUNS = GROUP / 32;  // groups in them, runs of a group
    const int64_t units = (int64_t)w.tiles * w.blocks;
    for (int64_t u = (int64_t)blockIdx.x * kW4Warps + warp; u < units; u += (int64_t)gridDim.x * kW4Warps) {
        const int tile = (int)(u / w.blocks), block = (int)(u - (int64_t)tile * w.blocks);
#pragma unroll 1
        for (int h0 = 0; h0 < 2; h0 += HALVES) {
            Run<T> x[2][2 * HALVES];  // [row g or g + 8][run of 32 columns]
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                Run<T> a[2], b[2];
                load_half<T>(values, stride, tile * kW4Rows, w.rows, block * kW4Cols + (h0 + h) * kW4Half, w.cols, vec, buf[warp], lane, a, b);
                x[0][2 * h] = a[0], x[0][2 * h + 1] = a[1], x[1][2 * h] = b[0], x[1][2 * h + 1] = b[1];
            }
            uint32_t word[4 * HALVES] = {};
            // Ranges of the groups, and of each quad's 2 or 4 (group, row) one per lane the step.
            constexpr int STEPS = 2 * GROUPS;
            float lows[STEPS], highs[STEPS];
            bool finite[STEPS];
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                const int i = j >> 1, k = j & 1;
                float top = 0.0f, low = 0.0f, high = 0.0f;
#pragma unroll
                for (int r = 0; r < RUNS; ++r) {
                    const float m = x[k][i * RUNS + r].top();
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(m));
                    if (ZEROS) x[k][i * RUNS + r].range(low, high);
                }
                finite[j] = top < INFINITY;
                if (!finite[j]) {  // what is not finite does not count
                    low = high = 0.0f;
                    for (int r = 0; r < RUNS; ++r)
                        for (int e = 0; e < 8; ++e) {
                            const float v = x[k][i * RUNS + r].get(e);
                            if (fabsf(v) < INFINITY) low = fminf(low, v), high = fmaxf(high, v);
                        }
                    top = fmaxf(-low, high);
                }
                if (!ZEROS) high = top;
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    if (ZEROS) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
                }
                lows[j] = low, highs[j] = high;
            }
            float my_low = lows[0], my_high = highs[0];
#pragma unroll
            for (int j = 1; j < STEPS; ++j)
                if (t % STEPS == j) my_low = lows[j], my_high = highs[j];
            const Step mine = step_of<ZEROS>(my_low, my_high);
            const uint32_t packed = mine.bits | (uint32_t)mine.zero << 16;
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                uint32_t both[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    both[k] = __shfl_sync(0xffffffffu, packed, (lane & ~3) | (2 * i + k));
                    Step st;
                    st.bits = (uint16_t)both[k];
                    st.s = __half2float(__ushort_as_half(st.bits));
                    st.zero = (float)(both[k] >> 16);
                    // Scales of at least 2^-14 (normal f16 numbers) that are not at the cap: no
                    // quotient is then past the last code by more than the scale's rounding.
                    const bool usual = finite[2 * i + k] && st.s >= 0x1p-14f && st.s < 65504.0f;
                    const float inv = __frcp_rn(st.s), below = inv * (1.0f - 0x1p-22f), above = inv * (1.0f + 0x1p-22f);
#pragma unroll
                    for (int r = 0; r < RUNS; ++r) {
                        uint32_t code[8];
                        encode<T, ZEROS>(x[k][i * RUNS + r], st, usual, below, above, code);
                        constexpr int kBit[4] = {0, 16, 8, 24};
#pragma unroll
                        for (int e = 0; e < 8; ++e) word[2 * (i * RUNS + r) + (e >> 2)] += code[e] * (1u << (kBit[e & 3] + 4 * k));
                    }
                }
                const int group = h0 * (kW4Half / 32) / RUNS + i;
                if (t == i) {
                    const bool there = block * kW4Cols + group * GROUP < w.cols;
                    const int64_t at = (u * 8 + g) * NG + group;
                    const uint32_t s0 = there && tile * kW4Rows + g < w.rows ? both[0] & 0xffffu : 0u;
                    const uint32_t s1 = there && tile * kW4Rows + g + 8 < w.rows ? both[1] & 0xffffu : 0u;
                    reinterpret_cast<uint32_t*>(w.scales)[at] = s0 | s1 << 16;
                    if (ZEROS) reinterpret_cast<uint16_t*>(w.zeros)[at] = (uint16_t)(both[0] >> 16 | both[1] >> 16 << 8);
                }
            }
            uint4* out = reinterpret_cast<uint4*>(w.codes + u * kW4BlockBytes) + h0 * 32 + lane;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
                out[h * 32] = make_uint4(turned(word[4 * h]), turned(word[4 * h + 1]), turned(word[4 * h + 2]), turned(word[4 * h + 3]));
        }
    }
}

// Codes [rows][ceil(cols / 2)], scales and zero points [rows][groups] as a
// checkpoint holds them.  A lane makes its 16 bytes from 8 bytes of two rows.
template <int GROUP>
__global__ void __launch_bounds__(kW4Threads) w4_pack_kernel(W4 w, const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                                                             const uint8_t* __restrict__ zeros) {
    constexpr int NG = kW4Cols / GROUP;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int64_t units = (int64_t)w.tiles * w.blocks;
    const int64_t pitch = (w.cols + 1) / 2;
    const int groups = (w.cols + GROUP - 1) / GROUP;
    for (int64_t u = (int64_t)blockIdx.x * kW4Warps + warp; u < units; u += (int64_t)gridDim.x * kW4Warps) {
        const int tile = (int)(u / w.blocks), block = (int)(u - (int64_t)tile * w.blocks);
        uint4* out = reinterpret_cast<uint4*>(w.codes + u * kW4BlockBytes);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = tile * kW4Rows + g + 8 * k;
                const int col = block * kW4Cols + h * kW4Half + 8 * t;
#pragma unroll
                for (int i = 0; i < 8; ++i) {  // a byte: column c (low half) and the next
                    const int c = col + 32 * (i >> 2) + 2 * (i & 3);
                    uint32_t b = row < w.rows && c < w.cols ? codes[row * pitch + (c >> 1)] : 0u;
                    if (c + 1 >= w.cols) b &= 15u;
                    constexpr int kBit[2] = {0, 8};
                    word[i >> 1] |= (b & 15u) << (kBit[i & 1] + 4 * k) | (b >> 4) << (kBit[i & 1] + 16 + 4 * k);
                }
            }
            out[h * 32 + lane] = make_uint4(turned(word[0]), turned(word[1]), turned(word[2]), turned(word[3]));
        }
        for (int i = lane; i < 8 * NG * 2; i += 32) {
            const int row = tile * kW4Rows + i / (2 * NG) + 8 * (i & 1);
            const int group = block * NG + (i >> 1) % NG;
            const bool there = row < w.rows && group < groups;
            const int64_t from = (int64_t)row * groups + group;
            w.scales[u * (16 * NG) + i] = there ? scales[from] : (uint16_t)0;
            if (zeros) w.zeros[u * (16 * NG) + i] = there ? zeros[from] & 15 : (uint8_t)0;
        }
    }
}

template <typename T, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4Threads) w4_read_kernel(W4 w, T* __restrict__ values, int64_t stride, bool vec) {
    __shared__ __align__(16) float buf[kW4Warps][kW4Rows * kW4Pitch];
    constexpr int NG = kW4Cols / GROUP;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int64_t units = (int64_t)w.tiles * w.blocks;
    for (int64_t u = (int64_t)blockIdx.x * kW4Warps + warp; u < units; u += (int64_t)gridDim.x * kW4Warps) {
        const int tile = (int)(u / w.blocks), block = (int)(u - (int64_t)tile * w.blocks);
        const uint4* in = reinterpret_cast<const uint4*>(w.codes + u * kW4BlockBytes);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 word = in[h * 32 + lane];
            const uint32_t ws[4] = {unturned(word.x), unturned(word.y), unturned(word.z), unturned(word.w)};
            const int col0 = block * kW4Cols + h * kW4Half;
            uint32_t sc[2], zp[2];  // of the two runs
#pragma unroll
            for (int run = 0; run < 2; ++run) {
                const int64_t at = (u * 8 + g) * NG + (2 * h + run) / (4 / NG);
                sc[run] = reinterpret_cast<const uint32_t*>(w.scales)[at];
                zp[run] = ZEROS ? reinterpret_cast<const uint16_t*>(w.zeros)[at] : 0x0808u;
            }
            const bool direct = vec && col0 + kW4Half <= w.cols;
            if (!direct) __syncwarp();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = tile * kW4Rows + g + 8 * k;
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    constexpr int kBit[4] = {0, 16, 8, 24};
                    const float s = __half2float(__ushort_as_half((uint16_t)(sc[i >> 3] >> (16 * k))));
                    v[i] = s * (float)((int)((ws[i >> 2] >> (kBit[i & 3] + 4 * k)) & 15u) - (int)((zp[i >> 3] >> (8 * k)) & 255u));
                }
                if (direct) {
                    constexpr int V = 16 / sizeof(T);
                    if (row < w.rows) {
#pragma unroll
                        for (int i = 0; i < 16 / V; ++i) {
                            T e[V];
#pragma unroll
                            for (int j = 0; j < V; ++j) e[j] = from_f32<T>(v[i * V + j]);
                            constexpr int R = 8 / V;
                            *(reinterpret_cast<uint4*>(values + row * stride + col0 + 32 * (i / R) + 8 * t) + i % R) = *reinterpret_cast<const uint4*>(e);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(&buf[warp][(g + 8 * k) * kW4Pitch + 32 * (i >> 1) + 8 * t + 4 * (i & 1)]) =
                            make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            }
            if (direct) continue;
            __syncwarp();
#pragma unroll
            for (int r = 0; r < kW4Rows; ++r) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int row = tile * kW4Rows + r, c = col0 + 32 * q + lane;
                    if (row < w.rows && c < w.cols) values[row * stride + c] = from_f32<T>(buf[warp][r * kW4Pitch + 32 * q + lane]);
                }
            }
        }
    }
}

unsigned w4_grid(const W4& w, int num_sms) {
    const int64_t ctas = ((int64_t)w.tiles * w.blocks + kW4Warps - 1) / kW4Warps, most = (int64_t)num_sms * 16;
    return (unsigned)(ctas < most ? ctas : most);
}

template <typename T>
bool vector_rows(const void* p, int64_t stride) {
    return (((uintptr_t)p | (uintptr_t)(stride * (int64_t)sizeof(T))) & 15) == 0;
}

template <typename T, int GROUP>
cudaError_t quantize_as(const W4& w, const void* v, int64_t stride, int num_sms, cudaStream_t st) {
    const bool vec = vector_rows<T>(v, stride);
    if (w.zeros) w4_quantize_kernel<T, GROUP, true><<<w4_grid(w, num_sms), kW4Threads, 0, st>>>(w, (const T*)v, stride, vec);
    else w4_quantize_kernel<T, GROUP, false><<<w4_grid(w, num_sms), kW4Threads, 0, st>>>(w, (const T*)v, stride, vec);
    return cudaGetLastError();
}
template <typename T, int GROUP>
cudaError_t read_as(const W4& w, void* v, int64_t stride, int num_sms, cudaStream_t st) {
    const bool vec = vector_rows<T>(v, stride);
    if (w.zeros) w4_read_kernel<T, GROUP, true><<<w4_grid(w, num_sms), kW4Threads, 0, st>>>(w, (T*)v, stride, vec);
    else w4_read_kernel<T, GROUP, false><<<w4_grid(w, num_sms), kW4Threads, 0, st>>>(w, (T*)v, stride, vec);
    return cudaGetLastError();
}

}  // namespace

#define LC_W4_GROUPS(fn, T, ...) \
    (w.group == 32 ? fn<T, 32>(__VA_ARGS__) : w.group == 64 ? fn<T, 64>(__VA_ARGS__) : fn<T, 128>(__VA_ARGS__))

cudaError_t launch_w4_quantize(const W4& w, const void* values, int64_t stride, int dtype, int num_sms, cudaStream_t st) {
    return dtype == kRowF32 ? LC_W4_GROUPS(quantize_as, float, w, values, stride, num_sms, st)
                            : LC_W4_GROUPS(quantize_as, __half, w, values, stride, num_sms, st);
}

cudaError_t launch_w4_read(const W4& w, void* values, int64_t stride, int dtype, int num_sms, cudaStream_t st) {
    return dtype == kRowF32 ? LC_W4_GROUPS(read_as, float, w, values, stride, num_sms, st)
                            : LC_W4_GROUPS(read_as, __half, w, values, stride, num_sms, st);
}

cudaError_t launch_w4_pack(const W4& w, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int num_sms, cudaStream_t st) {
    const unsigned grid = w4_grid(w, num_sms);
    if (w.group == 32) w4_pack_kernel<32><<<grid, kW4Threads, 0, st>>>(w, codes, scales, zeros);
    else if (w.group == 64) w4_pack_kernel<64><<<grid, kW4Threads, 0, st>>>(w, codes, scales, zeros);
    else w4_pack_kernel<128><<<grid, kW4Threads, 0, st>>>(w, codes, scales, zeros);
    return cudaGetLastError();
}

}  // namespace lc
