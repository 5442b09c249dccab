// lc_kv8.cu -- writing rows into the 8-bit pages and reading them back.
//
// Append.  A unit is the runs (neighbouring rows with consecutive slots) of one
// page, for one kv head, keys or values.  With s the page's scale (0 when the
// run starts the page) the new scale is s' = max(s, max |x| / limit); the codes
// that the page holds below the run become round(c s / s') when s' > s, and the
// run's are round(x / s').  Each rounding is to the nearest code of the exact
// quotient, so a value is within half a code step of what was stored before,
// whatever order the tokens came in.  No sums, and no order in which anything is
// added.
//
// Bound by memory: rows in once, codes out once.  A lane holds four neighbouring
// elements, a warp 2048 of a unit, in registers between the search for the
// maximum and the rounding; units of larger pages have 2, 4 or 8 warps, which meet
// over the maximum (8000 rows of 8 heads x 128, f32: 30 us in pages of 16 or 32, 58
// in pages of 128, where few units are left to go round; 71 with one warp a unit).
// The quotient is x * (1 / s), two units of the last place off at most; only where
// that could change the code (next to a tie) is it divided out.
#include "lc_internal.h"
#include "lc_kv8.cuh"

namespace lc {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kAppendWindow = 32;  // rows whose slots one CTA looks at together, at most
constexpr int kAppendHold = 16;    // groups of four that a lane keeps

// Four elements as they lie in memory.
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    float4 w;
    LC_DEV void load(const float* p, bool aligned) { w = aligned ? __ldg(reinterpret_cast<const float4*>(p)) : make_float4(p[0], p[1], p[2], p[3]); }
    LC_DEV float4 get() const { return w; }
    LC_DEV void zero() { w = make_float4(0, 0, 0, 0); }
    // Running largest size; a NaN never is.
    typedef float Top;
    static LC_DEV Top none() { return 0.0f; }
    LC_DEV Top top(Top t) const { return fmaxf(fmaxf(fmaxf(t, fabsf(w.x)), fabsf(w.y)), fmaxf(fabsf(w.z), fabsf(w.w))); }
    static LC_DEV float value(Top t) { return t; }
};
template <>
struct Raw<__half> {
    uint2 w;
    LC_DEV void load(const __half* p, bool aligned) {
        if (aligned) {
            w = __ldg(reinterpret_cast<const uint2*>(p));
        } else {
            const __half2 a = __halves2half2(p[0], p[1]), b = __halves2half2(p[2], p[3]);
            w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
    }
    LC_DEV float4 get() const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    LC_DEV void zero() { w = make_uint2(0, 0); }
    typedef __half2 Top;
    static LC_DEV Top none() { return __half2half2(__ushort_as_half(0)); }
    LC_DEV Top top(Top t) const {
        return __hmax2(t, __hmax2(__habs2(*reinterpret_cast<const __half2*>(&w.x)), __habs2(*reinterpret_cast<const __half2*>(&w.y))));
    }
    static LC_DEV float value(Top t) { return fmaxf(__low2float(t), __high2float(t)); }
};
template <typename T>
LC_DEV float4 load4(const T* p, bool aligned) {
    Raw<T> r;
    r.load(p, aligned);
    return r.get();
}

template <typename T>
LC_DEV void store4(T* p, float4 v, bool aligned);
template <>
LC_DEV void store4<float>(float* p, float4 v, bool aligned) {
    if (aligned) *reinterpret_cast<float4*>(p) = v;
    else p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
}
template <>
LC_DEV void store4<__half>(__half* p, float4 v, bool aligned) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    if (aligned) *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    else p[0] = __low2half(a), p[1] = __high2half(a), p[2] = __low2half(b), p[3] = __high2half(b);
}

// Largest finite size of four values, over `top`.
LC_DEV float top4(float4 v, float top) {
    const float f[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (f[i] < INFINITY) top = fmaxf(top, f[i]);
    return top;
}

// Four codes under scale s, inv = 1 / s rounded; byte i is value i.  SMALL as in
// quotient_odd: half rows that are not zero make no scale below 2^-33.
template <int FMT, bool SMALL>
LC_DEV uint32_t encode4(float4 v, float s, float inv) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint32_t w = 0;
    bool sure = true;
    if (FMT == kKv8I8) {
        // x inv + 1.5 * 2^23 rounds to a whole number, which stands in the sum's low
        // bits.  A quotient of at most 127 is off by 2^-16 at most; what is left
        // within 2^-14 of a half, or not finite, is not sure.
        uint32_t t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float m = __fmaf_rn(x[i], inv, 12582912.0f);
            t[i] = __float_as_uint(m);
            sure = sure && fabsf(__fmaf_rn(x[i], inv, 12582912.0f - m)) < 0.5f - 0x1p-14f;
        }
        w = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    } else {
        // A tie of a normal e4m3 value is 0x80000 in the low 20 bits of y; within
        // four units of that, below the normal range, or not finite, it is not sure.
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = x[i] * inv;
            sure = sure && ((__float_as_uint(y[i]) - (0x80000u - 4u)) & 0xfffffu) > 8u;
        }
        const float low = fminf(fminf(fabsf(y[0]), fabsf(y[1])), fminf(fabsf(y[2]), fabsf(y[3])));
        const float sum = fabsf(y[0]) + fabsf(y[1]) + fabsf(y[2]) + fabsf(y[3]);  // carries a NaN or an infinity
        sure = sure && low >= 0x1p-6f && sum < 2048.0f;
        w = e4m3x2(y[0], y[1]) | (e4m3x2(y[2], y[3]) << 16);
    }
    if (!sure || !(inv < INFINITY) || !(s > 0.0f)) {
        w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= kv8_encode<FMT, SMALL>(x[i], s) << (8 * i);
    }
    return w;
}

// Three CTAs of half rows on an SM, two of fp32 rows: what a lane keeps is 32 or
// 64 registers.  The compiler spills with teams (32 to 124 bytes).
template <typename T, int FMT, int D, bool TEAMS>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 2 ? 3 : 2) kv8_append_kernel(Kv8 c, Kv8Rows r, int window, int windows, int team_size) {
    constexpr int LPR = D / 4, RPI = 32 / LPR;  // lanes per row, rows at a time
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sh = c.page_shift, page = 1 << sh;
    const int64_t n_slots = (int64_t)c.n_pages << sh;
    const bool aligned = (((uintptr_t)r.k | (uintptr_t)r.v | (uintptr_t)(r.row_stride * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
    auto slot_of = [&](int64_t i) {
        const int v = r.slots[i];
        return v >= 0 && v < n_slots ? v : -1;
    };
    // `team` warps have a unit together, in TEAMS one at least two.
    const int team = TEAMS ? team_size : 1;
    const int part = warp % team, teams = kAppendWarps / team, mine = warp / team;
    __shared__ float tops[2][kAppendWarps];
    int flip = 0;
    auto meet = [&]() {
        if (TEAMS) named_bar_sync(1 + mine, team * 32);
        else __syncwarp();
    };
    auto team_max = [&](float v) {  // of all lanes of the team
        v = warp_max(v);
        if (!TEAMS) return v;
        if (lane == 0) tops[flip][warp] = v;
        meet();
        for (int k = 0; k < team; ++k) v = fmaxf(v, tops[flip][mine * team + k]);
        flip ^= 1;  // the next one does not touch what others may still read
        return v;
    };
    const int sub = lane / LPR, e0 = (lane % LPR) * 4;  // this lane's row of those at a time, and its elements
    const int at0 = part * RPI + sub, step = team * RPI;  // this lane's first row of a unit, and the distance to the next
    int n = 0;                                            // unit number within the CTA
    for (int win = 0; win < (TEAMS ? windows : 1); ++win) {
        const int64_t row0 = ((int64_t)blockIdx.x * windows + win) * window;
        if (row0 >= r.rows) break;
        // Lane i: is row row0 + i the first of its page's rows?  Rows without a
        // slot are passed over.
        const int64_t my = row0 + lane;
        int slot = -1;
        bool starts = false;
        if (lane < window && my < r.rows) {
            slot = slot_of(my);
            if (slot >= 0) {
                int prev = my > 0 ? slot_of(my - 1) : -1;
                for (int64_t i = my - 2; prev < 0 && i >= 0; i -= 8) {  // behind skipped rows, eight at a time
                    int v[8];
#pragma unroll
                    for (int b = 0; b < 8; ++b) v[b] = i - b >= 0 ? slot_of(i - b) : -1;
#pragma unroll
                    for (int b = 7; b >= 0; --b)
                        if (v[b] >= 0) prev = v[b];
                }
                starts = prev < 0 || (prev >> sh) != (slot >> sh);
            }
        }
        unsigned starters = __ballot_sync(0xffffffffu, starts);
        while (starters) {
            const int l = __ffs(starters) - 1;
            starters &= starters - 1;
            const int pg = __shfl_sync(0xffffffffu, slot, l) >> sh;
            for (int u = blockIdx.y; u < 2 * c.n_kv; u += gridDim.y, ++n) {
                if (n % teams != mine) continue;
                const int head = u >> 1;
                const T* rows = (const T*)((u & 1) ? r.v : r.k) + head * D + e0;
                uint8_t* codes = ((u & 1) ? c.v : c.k) + ((((int64_t)pg * c.n_kv + head) << sh) * D) + e0;
                float* scale = ((u & 1) ? c.v_scale : c.k_scale) + (int64_t)pg * c.n_kv + head;
                float held = *scale;
                // The page's runs, one after the other: usually there is one.
                for (int64_t row = row0 + l; row < r.rows;) {
                    const int first = slot_of(row);
                    if (first < 0) {  // skipped rows, 128 at a time: a padded batch ends in many
                        int v[4];
#pragma unroll
                        for (int b = 0; b < 4; ++b) v[b] = row + b * 32 + lane < r.rows ? slot_of(row + b * 32 + lane) : -1;
                        int skip = 128;
#pragma unroll
                        for (int b = 3; b >= 0; --b) {
                            const unsigned m = __ballot_sync(0xffffffffu, v[b] >= 0);
                            if (m) skip = b * 32 + __ffs(m) - 1;
                        }
                        row += skip;
                        continue;
                    }
                    if ((first >> sh) != pg) break;
                    const int off = first & (page - 1);
                    // Rows row .. row + len - 1, at most to the page's end; those of this
                    // window are in the lanes' `slot`.
                    int len = 1;
                    if (row < row0 + window) {
                        const int k = (int)(my - row);
                        const unsigned m = __ballot_sync(0xffffffffu, k < 0 || (lane < window && off + k < page && slot == first + k));
                        len = (m == 0xffffffffu ? 32 : __ffs(~m) - 1) - (int)(row - row0);
                    }
                    for (; row + len >= row0 + window && off + len < page; len += 32) {
                        const int k = len + lane;
                        const bool ok = off + k < page && row + k < r.rows && r.slots[row + k] == first + k;
                        const unsigned m = __ballot_sync(0xffffffffu, ok);
                        if (m != 0xffffffffu) {
                            len += __ffs(~m) - 1;
                            break;
                        }
                    }
                    const T* x = rows + row * r.row_stride;
                    Raw<T> v[kAppendHold];
                    typename Raw<T>::Top most = Raw<T>::none();
#pragma unroll
                    for (int i = 0; i < kAppendHold; ++i) {
                        const int k = at0 + i * step;
                        if (k < len) v[i].load(x + (int64_t)k * r.row_stride, aligned);
                        else v[i].zero();
                    }
#pragma unroll
                    for (int i = 0; i < kAppendHold; ++i) most = v[i].top(most);
                    float top = team_max(Raw<T>::value(most));
                    if (top == INFINITY) {  // infinities do not set the scale
                        top = 0.0f;
#pragma unroll
                        for (int i = 0; i < kAppendHold; ++i) top = top4(v[i].get(), top);
                        top = team_max(top);
                    }
                    const float old = off ? held : 0.0f;
                    const float now = fmaxf(old, __fdiv_rn(top, kv8_limit(FMT)));
                    const float inv = __fdiv_rn(1.0f, now);
                    if (now > old)
                        for (int k = at0; k < off; k += step) {
                            uint32_t* at = reinterpret_cast<uint32_t*>(codes + k * D);
                            const uint32_t w = *at;
                            uint32_t z = 0;
#pragma unroll
                            for (int b = 0; b < 4; ++b) z |= kv8_requant<FMT>((w >> (8 * b)) & 0xffu, old, now) << (8 * b);
                            *at = z;
                        }
#pragma unroll
                    for (int i = 0; i < kAppendHold; ++i) {
                        const int k = at0 + i * step;
                        if (k < len) *reinterpret_cast<uint32_t*>(codes + (off + k) * D) = encode4<FMT, sizeof(T) == 4>(v[i].get(), now, inv);
                    }
                    held = now;
                    row += len;
                    meet();  // the next run rounds these codes anew
                }
                if (part == 0 && lane == 0) *scale = held;
            }
        }
    }
}

// Four codes -> values.
template <int FMT>
LC_DEV float4 decode4(uint32_t w, float s) {
    if (FMT == kKv8I8) {
        w ^= 0x80808080u;  // 0x4b000000 | u is 2^23 + u, u = code + 128
        const float m = 8388736.0f;
        return make_float4((__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - m) * s,
                           (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - m) * s,
                           (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - m) * s,
                           (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - m) * s);
    }
    uint32_t a, b;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(a), "=r"(b) : "r"(w));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    return make_float4(x.x * s, x.y * s, y.x * s, y.y * s);
}

// A thread per eight elements of a row, of keys and of values, two rows under
// way together; bound by the rows written.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, Kv8Rows r) {
    griddep_launch();
    griddep_wait();
    const int d = c.head_dim, sh = c.page_shift, octs = c.n_kv * d / 8;
    const int64_t n_slots = (int64_t)c.n_pages << sh;
    const bool aligned = (((uintptr_t)r.k | (uintptr_t)r.v | (uintptr_t)(r.row_stride * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
    const int per = octs < 256 ? 256 / octs : 1;  // rows of the CTA at a time
    const int sub = threadIdx.x / octs, q0 = per > 1 ? threadIdx.x - sub * octs : threadIdx.x;
    if (per > 1 && sub >= per) return;
    const int64_t step = (int64_t)gridDim.x * per;
    for (int64_t row = blockIdx.x * per + (per > 1 ? sub : 0); row < r.rows; row += 2 * step) {
        int slot[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            slot[b] = row + b * step < r.rows ? r.slots[row + b * step] : -1;
            if (slot[b] >= n_slots) slot[b] = -1;
        }
        for (int q = q0; q < octs; q += 256) {
            const int head = q * 8 / d, e = q * 8 - head * d;
            uint2 kw[2], vw[2];
            float ks[2], vs[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (slot[b] < 0) continue;
                const int64_t st = (int64_t)(slot[b] >> sh) * c.n_kv + head;
                const int64_t at = ((st << sh) + (slot[b] & ((1 << sh) - 1))) * d + e;
                kw[b] = __ldg(reinterpret_cast<const uint2*>(c.k + at)), vw[b] = __ldg(reinterpret_cast<const uint2*>(c.v + at));
                ks[b] = __ldg(c.k_scale + st), vs[b] = __ldg(c.v_scale + st);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (slot[b] < 0) continue;  // rows without a slot are left as they are
                T* k = (T*)r.k + (row + b * step) * r.row_stride + q * 8;
                T* v = (T*)r.v + (row + b * step) * r.row_stride + q * 8;
                store4(k, decode4<FMT>(kw[b].x, ks[b]), aligned);
                store4(k + 4, decode4<FMT>(kw[b].y, ks[b]), aligned);
                store4(v, decode4<FMT>(vw[b].x, vs[b]), aligned);
                store4(v + 4, decode4<FMT>(vw[b].y, vs[b]), aligned);
            }
        }
    }
}

}  // namespace

template <typename T, int FMT>
static cudaError_t append(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st) {
    // A CTA looks at as many rows as leave every SM four CTAs (with 64 rows of
    // 64 sequences and 32 rows a CTA, two CTAs took 119 us), at most at a page
    // or 32; a team of warps holds a page of one head, and the units of a page
    // are shared out so that every team has one.
    int window = r.rows / (num_sms * 4);
    window = window < 1 ? 1 : window > kAppendWindow ? kAppendWindow : window;
    const int page = 1 << c.page_shift, windows = window == kAppendWindow && page > window ? page / window : 1;
    const int unit = page * c.head_dim, team = unit <= 2048 ? 1 : unit / 2048;
    const int64_t span = (int64_t)window * windows;
    int shares = 2 * c.n_kv * team / kAppendWarps;
    shares = shares < 1 ? 1 : shares > 2 * c.n_kv ? 2 * c.n_kv : shares;
    const dim3 grid((unsigned)((r.rows + span - 1) / span), shares), block(kAppendThreads);
    auto go = [&](auto kernel) { return launch_ex(kernel, grid, block, 0, st, true, c, r, window, windows, team); };
    if (c.head_dim == 64) return team > 1 ? go(kv8_append_kernel<T, FMT, 64, true>) : go(kv8_append_kernel<T, FMT, 64, false>);
    return team > 1 ? go(kv8_append_kernel<T, FMT, 128, true>) : go(kv8_append_kernel<T, FMT, 128, false>);
}

cudaError_t launch_kv8_append(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st) {
    if (r.dtype == kRowF32) return c.format == kKv8I8 ? append<float, kKv8I8>(c, r, num_sms, st) : append<float, kKv8E4M3>(c, r, num_sms, st);
    return c.format == kKv8I8 ? append<__half, kKv8I8>(c, r, num_sms, st) : append<__half, kKv8E4M3>(c, r, num_sms, st);
}

cudaError_t launch_kv8_read(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st) {
    const int octs = c.n_kv * c.head_dim / 8, per = octs < 256 ? 256 / octs : 1, ctas = (r.rows + per - 1) / per;
    const dim3 grid(ctas < num_sms * 8 ? ctas : num_sms * 8), block(256);
    if (r.dtype == kRowF32)
        return c.format == kKv8I8 ? launch_ex(kv8_read_kernel<float, kKv8I8>, grid, block, 0, st, true, c, r)
                                  : launch_ex(kv8_read_kernel<float, kKv8E4M3>, grid, block, 0, st, true, c, r);
    return c.format == kKv8I8 ? launch_ex(kv8_read_kernel<__half, kKv8I8>, grid, block, 0, st, true, c, r)
                              : launch_ex(kv8_read_kernel<__half, kKv8E4M3>, grid, block, 0, st, true, c, r);
}

}  // namespace lc
