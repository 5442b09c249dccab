// lc_kv8.cuh -- the 8-bit codes of the paged KV cache.
//
// A page holds `page` tokens of every kv head: codes [n_kv][page][d] and one
// fp32 scale per head; a value is code * scale.  Codes are signed bytes in
// [-127, 127] or e4m3 values up to 448, so with scale = max |x| / limit the
// largest value of a page sits at the end of the range.
#pragma once

#include "lc_common.cuh"
#include "lc_paged.h"

namespace lc {

__host__ __device__ constexpr float kv8_limit(int format) { return format == kKv8I8 ? 127.0f : 448.0f; }

template <int FMT>
LC_DEV float kv8_decode(uint32_t byte) {
    if (FMT == kKv8I8) return (float)(int8_t)byte;
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)byte));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

// Two fp32 values of at most 448 in size -> two e4m3 bytes (low byte: a).
LC_DEV uint32_t e4m3x2(float a, float b) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

// The quotient x / s rounded to odd: the nearest fp32 value, moved to the
// neighbour on the true value's side when it is inexact and its last bit is
// even.  Rounding that to a code of 8 bits or fewer gives the code nearest to
// the exact quotient, ties to even only where the quotient IS a tie (a plain
// fp32 quotient can land on a tie that it is not).  SMALL: s may be below 2^-100;
// such numbers are scaled up first, for beside a tie x - q s can be half the
// smallest number there is.
template <bool SMALL>
LC_DEV float quotient_odd(float x, float s) {
    if (SMALL && s < 0x1p-100f) x *= 0x1p64f, s *= 0x1p64f;  // |x| is below 2^9 s, or infinite
    const float q = __fdiv_rn(x, s);
    if (!(fabsf(q) < 1024.0f)) return q;  // saturates below; infinities stay themselves
    const float r = __fmaf_rn(-q, s, x);
    const int b = __float_as_int(q);
    if (r == 0.0f || (b & 1)) return q;
    return __int_as_float(b + (((__float_as_int(r) ^ b) >= 0) ? 1 : -1));
}

template <int FMT>
LC_DEV uint32_t kv8_round(float q) {
    if (FMT == kKv8I8) {
        const int c = __float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f));
        return (uint32_t)c & 0xffu;
    }
    return e4m3x2(q, 0.0f) & 0xffu;
}

// x under scale s: NaN becomes 0, infinities the end of the range, and a zero
// scale gives code 0.
template <int FMT, bool SMALL>
LC_DEV uint32_t kv8_encode(float x, float s) {
    if (!(s > 0.0f) || x != x) return 0;
    return kv8_round<FMT>(quotient_odd<SMALL>(x, s));
}

// A held code under a grown scale: round(code * s_old / s_new).  The product
// is exact in fp64 and the quotient is at least 2^-32 away from any tie that
// it is not, so one fp64 division decides it; fp32 takes the value rounded
// toward zero with a sticky last bit (round to odd again).
template <int FMT>
LC_DEV uint32_t kv8_requant(uint32_t byte, float s_old, float s_new) {
    const double q = (double)kv8_decode<FMT>(byte) * (double)s_old / (double)s_new;
    float f = __double2float_rz(q);
    if ((double)f != q) f = __int_as_float(__float_as_int(f) | 1);
    if (f != f) return 0;
    return kv8_round<FMT>(f);
}

}  // namespace lc
