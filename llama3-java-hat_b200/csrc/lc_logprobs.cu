// lc_logprobs.cu -- log probabilities of given tokens with their ranks, the
// entropy and the best alternatives, from rows of logits, in one pass.
//
// With m the largest logit of a row, u_i = scale log2(e) (x_i - m), S = sum
// 2^u_i and T = sum u_i 2^u_i: ln p_i = scale (x_i - m) - ln S and
// H = ln S - ln 2 T / S.  A thread keeps its own m, S and T; when m grows by d
// (in units of u) S becomes 2^-d S and T 2^-d (T - d S).  u is held at -200 and
// above, where 2^u is 0 already: masked logits (-inf, the type's lowest) then
// add nothing, and not 0 * inf.
//
// The best k cost the pass nothing: it has every thread's largest logit anyway.
// A thread with k larger ones above its own holds none of the best k, so about
// k of the CTA's threads are left, whose elements are read again (from L2) and
// compared with the least of their largest.  The order of tokens is that of
// 64-bit keys (the logit's bits, then the index), so it does not depend on who
// finds them.  A rank is counted where a chunk's largest logit reaches the
// token's, which few chunks do for likely tokens.
//
// F16 rows: 9 instructions per logit, two thirds of the issue slots, and 69 to 73 % of
// the measured copy's rate (2048 rows of 128256: 110 to 117 us on several GPUs, 80 at
// that rate); neither alone is the bound, a thread's sums wait for its loads and its
// loads' registers for its sums.  Short rows: by the beginnings and ends of CTAs.
// Few rows are cut over a cluster of up to 16 CTAs, whose parts meet in the shared
// memory of the first: no workspace, nothing kept.
#include <type_traits>

#include "lc_internal.h"
#include "lc_w4.h"

namespace lc {
namespace {

constexpr int kLpThreads = 256, kLpShort = 128;  // of a CTA, and where rows are many and short
constexpr int kLpPieces = 4;       // 16-byte pieces of a thread's chunk
constexpr uint32_t kLpFound = 256;  // candidates that are put in order by counting
constexpr int kLpMaxCluster = 16;  // more than 8 is opt-in
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLpFloor = -200.0f;

LC_DEV float max_nan(float a, float b) {  // a NaN wins
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
LC_DEV float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
LC_DEV float exp2_fast(float x) {  // 2 units of the last place; 0 below 2^-126
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}
LC_DEV uint64_t pack2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
LC_DEV float2 unpack2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
LC_DEV uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
LC_DEV uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
LC_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

// Bits that order as the logits do; NaN as -inf, zeros of both signs alike.
LC_DEV uint32_t ordered(float v) {
    v = v == v ? v + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(v);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
LC_DEV float unordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
LC_DEV uint64_t order_key(float v, int i) { return (uint64_t)ordered(v) << 32 | (uint32_t)~i; }
constexpr uint32_t kOrderedMasked = 0x007fffffu;  // of -inf

// The unit of exponents: u = a b c (x - m), a b c = scale log2(e).  a and b are 1 for
// F16, where c is held at 2^100: unlike logits are 2^-24 apart and more, so that beyond
// it the smaller ones have p 0 all the same.  F32 logits can lie closer and further
// apart: b = 2^26 for scales above 2^100, with which c is finite, and a = 2^-26 for
// scales below 2^-100, with which a x - a m is, and c has all its bits.
struct Unit {
    float a, b, c;
};
Unit unit_of(float scale, int dtype) {
    Unit u = {1.0f, 1.0f, scale};
    if (dtype == kRowF32 && scale > 0x1p100f) u.b = 0x1p26f, u.c *= 0x1p-26f;
    if (dtype == kRowF32 && scale < 0x1p-100f) u.a = 0x1p-26f, u.c *= 0x1p26f;
    u.c *= kLog2e;
    if (dtype != kRowF32 && u.c > 0x1p100f) u.c = 0x1p100f;
    return u;
}

// 16 bytes of logits.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
    static constexpr int N = 4;
    uint4 w;
    LC_DEV float get(int i) const { return __uint_as_float(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w); }
    LC_DEV float at(int i) const {  // of a place known only at run time
        const uint32_t lo = i & 1 ? w.y : w.x, hi = i & 1 ? w.w : w.z;
        return __uint_as_float(i & 2 ? hi : lo);
    }
    LC_DEV float top() const { return max_nan(max3_nan(get(0), get(1), get(2)), get(3)); }
    // c (x - ref) of elements 2 i and 2 i + 1, kLpFloor where it is less.  FAR: under
    // a scale for which it takes all of the unit's factors.
    template <bool FAR>
    LC_DEV float2 powers(int i, float ref, const Unit& unit) const {
        const uint64_t x = pack2(get(2 * i), get(2 * i + 1)), c2 = pack2(unit.c, unit.c);
        const float2 u = FAR ? unpack2(mul2(mul2(fma2(x, pack2(unit.a, unit.a), pack2(-ref * unit.a, -ref * unit.a)), pack2(unit.b, unit.b)), c2))
                             : unpack2(mul2(add2(x, pack2(-ref, -ref)), c2));
        return make_float2(fmaxf(u.x, kLpFloor), fmaxf(u.y, kLpFloor));
    }
    // How many are larger than v.
    LC_DEV uint32_t above(float v) const { return (get(0) > v) + (get(1) > v) + (get(2) > v) + (get(3) > v); }
    // The next smaller number: what is larger than it is v or larger.
    static LC_DEV float below(float v) {
        const int b = __float_as_int(v);
        return __int_as_float(v > 0.0f ? b - 1 : v < 0.0f ? b + 1 : (int)0x80000001u);
    }
};
template <>
struct Piece<__half> {
    static constexpr int N = 8;
    uint4 w;
    LC_DEV __half2 two(int i) const {
        const uint32_t v = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return *reinterpret_cast<const __half2*>(&v);
    }
    LC_DEV float get(int i) const { return i & 1 ? __high2float(two(i >> 1)) : __low2float(two(i >> 1)); }
    LC_DEV float at(int i) const {
        const uint32_t lo = i & 2 ? w.y : w.x, hi = i & 2 ? w.w : w.z, v = i & 4 ? hi : lo;
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? v >> 16 : v)));
    }
    LC_DEV float top() const {
        const __half2 m = __hmax2_nan(__hmax2_nan(two(0), two(1)), __hmax2_nan(two(2), two(3)));
        return max_nan(__low2float(m), __high2float(m));
    }
    // As above.  FAR: ref is so far above the lowest number (-65504) that its
    // power is 0; -inf may then stand as that number, whose product with c is
    // finite (c is 2^100 at most).  A pair's clamp is one instruction so.
    template <bool FAR>
    LC_DEV float2 powers(int i, float ref, const Unit& unit) const {
        const uint64_t c2 = pack2(unit.c, unit.c);
        if (!FAR) {
            const float2 u = unpack2(mul2(add2(pack2(get(2 * i), get(2 * i + 1)), pack2(-ref, -ref)), c2));
            return make_float2(fmaxf(u.x, kLpFloor), fmaxf(u.y, kLpFloor));
        }
        const __half2 v = __hmax2_nan(two(i), __half2half2(__ushort_as_half(0xfbff)));
        float a, b;
        asm("sub.rn.f32.f16 %0, %1, %2;" : "=f"(a) : "h"(__half_as_ushort(__low2half(v))), "f"(ref));
        asm("sub.rn.f32.f16 %0, %1, %2;" : "=f"(b) : "h"(__half_as_ushort(__high2half(v))), "f"(ref));
        return unpack2(mul2(pack2(a, b), c2));
    }
    LC_DEV uint32_t above(float v) const {
        const __half2 t = __half2half2(__float2half_rn(v));  // exact
        const __half2 n = __hadd2(__hadd2(__hgt2(two(0), t), __hgt2(two(1), t)), __hadd2(__hgt2(two(2), t), __hgt2(two(3), t)));
        return (uint32_t)(__low2float(n) + __high2float(n));
    }
    static LC_DEV float below(float v) {
        const int b = __half_as_ushort(__float2half_rn(v));
        return __half2float(__ushort_as_half((unsigned short)(v > 0.0f ? b - 1 : v < 0.0f ? b + 1 : 0x8001)));
    }
};

LC_DEV uint4 load_once(const void* p) {
    uint4 w;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p));
    return w;
}

// A row as 16-byte pieces of memory: piece j holds elements j N - skew and on.
template <typename T>
struct Row {
    const T* x;
    int skew, vocab;
    LC_DEV int first(int j) const { return j * Piece<T>::N - skew; }
    LC_DEV bool has(int i) const { return (unsigned)i < (unsigned)vocab; }
    // -inf in the places before and behind the row.
    LC_DEV Piece<T> load(int j) const {
        const int i = first(j);
        Piece<T> p;
        if (i >= 0 && i + Piece<T>::N <= vocab) {
            p.w = load_once(x + i);
        } else {
            T e[Piece<T>::N];
#pragma unroll
            for (int k = 0; k < Piece<T>::N; ++k) e[k] = has(i + k) ? x[i + k] : (T)-INFINITY;
            p.w = *reinterpret_cast<const uint4*>(e);
        }
        return p;
    }
};

// The 32 largest of two descending lists of a key per lane, descending.
LC_DEV uint64_t merge_lists(uint64_t a, uint64_t b, int lane) {
    uint64_t v = max(a, (uint64_t)__shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, v, o);
        v = (lane & o) ? min(v, other) : max(v, other);
    }
    return v;
}

// lists[0] = the largest of n lists (a power of two), by all warps of the CTA.
template <int WARPS>
LC_DEV void join_lists(uint64_t (*lists)[32], int n, int warp, int lane) {
    for (n >>= 1; n > 0; n >>= 1) {
        __syncthreads();
        for (int i = warp; i < n; i += WARPS) lists[i][lane] = merge_lists(lists[i][lane], lists[i + n][lane], lane);
    }
    __syncthreads();
}

LC_DEV uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
LC_DEV uint32_t map_to(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
LC_DEV void put32(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
LC_DEV void put64(uint32_t a, uint64_t v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
LC_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
LC_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

struct Part {  // of a CTA's share of a row
    float m, s, t;
    uint32_t before;
};

// ENDS: F32 rows under a scale with which a or b is not 1.
template <typename T, bool TOP, int THREADS, bool ENDS>
__global__ void __launch_bounds__(THREADS, 768 / THREADS) logprobs_kernel(Logprobs p, Unit unit, int cluster) {
    constexpr int WARPS = THREADS / 32;
    __shared__ Part parts[kLpMaxCluster];
    __shared__ __align__(16) __half tops[TOP ? THREADS : 1];
    __shared__ uint64_t found[TOP ? kLpFound + 32 * WARPS : 1];
    __shared__ uint64_t lists[TOP ? kLpMaxCluster : 1][32];
    __shared__ uint64_t ours[TOP ? WARPS : 1][32];
    __shared__ uint16_t chosen[TOP ? THREADS : 1];
    __shared__ uint32_t warp_top[WARPS], warp_before[WARPS], n_chosen, n_found, least;
    __shared__ float warp_s[WARPS], warp_t[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
    if (cluster > 1) cluster_arrive();  // all CTAs of the cluster have begun when the wait below is over
    griddep_wait();
    griddep_launch();
    const int64_t r = blockIdx.x / cluster;
    Row<T> row;
    row.x = (const T*)p.x + r * p.stride;
    row.skew = (int)(((uintptr_t)row.x & 15) / sizeof(T));
    row.vocab = p.vocab;
    constexpr int N = Piece<T>::N;
    const int64_t pieces = ((int64_t)row.skew + p.vocab + N - 1) / N;
    const int p0 = (int)(pieces * rank / cluster), p1 = (int)(pieces * (rank + 1) / cluster);
    // ---- the pass ----
    const float far_from = -65504.0f - kLpFloor / unit.c;
    auto down_to = [&](float ref, float now) {  // the exponent of ref's unit in now's
        return fmaxf((ENDS ? (ref * unit.a - now * unit.a) * unit.b : ref - now) * unit.c, kLpFloor);
    };
    float m = -INFINITY, ref = -3.4028234663852886e38f;  // ref: what exponents are taken from
    uint64_t s2 = 0, t2 = 0;  // pairs of sums
    uint32_t before = 0;
    // Pieces whose elements all belong to the row, and the CTA's share of them.
    const int whole0 = max(p0, row.skew ? 1 : 0), whole1 = min(p1, (int)(((int64_t)row.skew + p.vocab) / N));
    Piece<T> next[kLpPieces];
    auto fetch = [&](int base) {  // the thread's pieces of the chunk at base, -inf behind the share
        const int j = base + tid;
        if (base >= whole0 && base + kLpPieces * THREADS <= whole1) {
            const T* from = row.x + row.first(j);
#pragma unroll
            for (int k = 0; k < kLpPieces; ++k) next[k].w = load_once(from + k * THREADS * N);
        } else {
#pragma unroll
            for (int k = 0; k < kLpPieces; ++k) {
                const int at = j + k * THREADS;
                if (at < p1) next[k] = row.load(at);
                else next[k].w = sizeof(T) == 4 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u)
                                                : make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
            }
        }
    };
    fetch(p0);
    int token = p.tokens ? p.tokens[r] : -1;
    if (token >= p.vocab) token = -1;
    float mine = INFINITY;  // the token's logit
    if (token >= 0) {
        mine = (float)row.x[token];
        if (!(mine == mine)) mine = -INFINITY;
    }
    const bool ranked = token >= 0 && p.token_ranks && mine > -INFINITY;
    const float under = Piece<T>::below(mine);
    for (int base = p0; base < p1; base += kLpPieces * THREADS) {
        const int j = base + tid;
        Piece<T> w[kLpPieces];
#pragma unroll
        for (int k = 0; k < kLpPieces; ++k) w[k] = next[k];
        if (base + kLpPieces * THREADS < p1) fetch(base + kLpPieces * THREADS);
        float top = w[0].top();
#pragma unroll
        for (int k = 1; k < kLpPieces; ++k) top = max_nan(top, w[k].top());
        m = max_nan(m, top);
        const float now = fmaxf(m, ref);
        const float d = down_to(ref, now), down = exp2_fast(d);
        ref = now;
        t2 = mul2(fma2(s2, pack2(d, d), t2), pack2(down, down));
        s2 = mul2(s2, pack2(down, down));
        auto add_up = [&](auto far) {
#pragma unroll
            for (int k = 0; k < kLpPieces; ++k) {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    const float2 u = w[k].template powers<decltype(far)::value>(i, ref, unit);
                    const uint64_t e2 = pack2(exp2_fast(u.x), exp2_fast(u.y));
                    s2 = add2(s2, e2);
                    t2 = fma2(e2, pack2(u.x, u.y), t2);
                }
            }
        };
        if (ENDS || (sizeof(T) == 2 && ref > far_from)) add_up(std::true_type());
        else add_up(std::false_type());
        if (ranked && !(top < mine)) {
#pragma unroll
            for (int k = 0; k < kLpPieces; ++k) {
                const int i = row.first(j + k * THREADS);
                before += i + N <= token ? w[k].above(under) : w[k].above(mine);
                if (i < token && i + N > token && j + k * THREADS < p1)  // the token's own piece: what stands before it counts when equal
                    for (int e = i; e < token; ++e) before += row.has(e) && (float)row.x[e] == mine;
            }
        }
    }
    if (token >= 0 && p.token_ranks && !ranked) {  // a masked token comes behind all that are not, and masked ones before it
        for (int64_t i = (int64_t)p0 * N - row.skew + tid, end = (int64_t)p1 * N - row.skew; i < end; i += THREADS)
            before += i >= 0 && i < p.vocab && ((float)row.x[i] > -INFINITY || i < token);
    }

    // ---- the CTA's part ----
    const bool nan = !(m == m);
    const uint32_t my_top = nan ? 0xffffffffu : ordered(m);  // a NaN above all
    const uint32_t wt = __reduce_max_sync(0xffffffffu, my_top);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) warp_top[warp] = wt, warp_before[warp] = before;
    if (tid == 0) n_chosen = n_found = 0, least = 0xffffffffu;
    if (TOP) tops[tid] = __float2half_rd(m);
    __syncthreads();
    uint32_t cta_top = warp_top[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) cta_top = max(cta_top, warp_top[i]);
    const float cta_m = cta_top == 0xffffffffu ? NAN : unordered(cta_top);
    {
        const float now = fmaxf(cta_m, -3.4028234663852886e38f);
        const float d = down_to(ref, now), down = exp2_fast(d);
        const float2 s = unpack2(s2), t = unpack2(t2);
        const float sum = s.x + s.y;
        const float ws = warp_sum(sum * down), wt2 = warp_sum(fmaf(sum, d, t.x + t.y) * down);
        if (lane == 0) warp_s[warp] = ws, warp_t[warp] = wt2;
    }
    if (TOP) {
        // Threads with fewer than `top` larger maxima above their own.
        bool in = cta_top == 0xffffffffu;  // a NaN hides a maximum: then all
        if (!in) {
            // Rounded down to f16 they keep their order, but for ties, which let in more.
            const __half2 m2 = __half2half2(tops[tid]);
            __half2 above = __half2half2(__ushort_as_half(0));
#pragma unroll 8
            for (int i = 0; i < THREADS / 8; ++i) {
                const uint4 o = reinterpret_cast<const uint4*>(tops)[i];
                const __half2* h = reinterpret_cast<const __half2*>(&o);
                above = __hadd2(above, __hadd2(__hadd2(__hgt2(h[0], m2), __hgt2(h[1], m2)), __hadd2(__hgt2(h[2], m2), __hgt2(h[3], m2))));
            }
            in = (int)(__low2float(above) + __high2float(above)) < p.top;
        }
        const uint32_t low = __reduce_min_sync(0xffffffffu, in ? (cta_top == 0xffffffffu ? kOrderedMasked : my_top) : 0xffffffffu);
        const unsigned who = __ballot_sync(0xffffffffu, in);
        int at = 0;
        if (lane == 0 && who) {
            at = atomicAdd(&n_chosen, __popc(who));
            atomicMin(&least, low);
        }
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
        if (in) chosen[at] = (uint16_t)tid;
        __syncthreads();
        // The pieces of all chosen threads side by side, one per lane; what reaches
        // the least of their maxima is set aside.
        const float floor = unordered(least);
        const uint64_t bar = (uint64_t)least << 32;
        const int per = (p1 - p0 + THREADS - 1) / THREADS, items = (int)n_chosen * per;
        auto item_of = [&](int item, Piece<T>& w) {
            const int q = item / per, j = item < items ? p0 + chosen[q] + (item - q * per) * THREADS : p1;
            if (j < p1) w = row.load(j);
            return j;
        };
        auto collect = [&](uint64_t from, bool above) {  // keys from `from` on; above: larger than floor
            for (int item = tid; item < items && *(volatile uint32_t*)&n_found <= kLpFound; item += 4 * THREADS) {
                Piece<T> w[4];
                int j[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) j[z] = item_of(item + z * THREADS, w[z]);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    if (j[z] >= p1 || (above ? w[z].top() <= floor : w[z].top() < floor)) continue;
#pragma unroll 1
                    for (int e = 0, i = row.first(j[z]); e < N; ++e, ++i) {
                        const uint64_t key = order_key(w[z].at(e), i);
                        if (key < from || !row.has(i)) continue;
                        const uint32_t at = atomicAdd(&n_found, 1u);
                        if (at < kLpFound) found[at] = key;
                    }
                }
            }
        };
        // Where so few are allowed that masked ones are among the best there are
        // more of these than fit, as a rule.
        bool fit = least > ordered(sizeof(T) == 4 ? -3.4028234663852886e38f : -65504.0f);
        if (fit) collect(bar, false);
        if (warp == 0) ours[0][lane] = 0;
        __syncthreads();
        fit = fit && n_found <= kLpFound;
        if (!fit) {
            // Equal logits by the hundred, such as masked ones where few are allowed:
            // those above them, and then of each warp's part of the share the first
            // that are equal, as many as may be needed.
            __syncthreads();
            if (tid == 0) n_found = 0;
            __syncthreads();
            if (least < cta_top) collect(bar + (1ull << 32), true);
            __syncthreads();
            fit = n_found <= kLpFound;
            if (fit) {
                const int q0 = p0 + (int)((int64_t)(p1 - p0) * warp / WARPS), q1 = p0 + (int)((int64_t)(p1 - p0) * (warp + 1) / WARPS);
                __syncthreads();  // all have read the count
                int got = 0;
                for (int j = q0 + lane; __any_sync(0xffffffffu, j < q1) && got < p.top; j += 32) {
                    Piece<T> w;
                    if (j < q1) w = row.load(j);
                    const int i = row.first(j);
                    unsigned equal = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) equal |= (unsigned)(j < q1 && row.has(i + e) && ordered(w.get(e)) == least) << e;
                    int upto = __popc(equal);
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int u = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += u;
                    }
                    int place = got + upto - __popc(equal);
                    for (; equal && place < p.top; equal &= equal - 1, ++place) {
                        const uint32_t at = atomicAdd(&n_found, 1u);
                        found[at] = (uint64_t)least << 32 | (uint32_t)~(i + __ffs(equal) - 1);
                    }
                    got += __shfl_sync(0xffffffffu, upto, 31);
                }
                __syncthreads();
            }
        }
        if (fit) {
            // Each one's place is the number of larger ones.
            for (int q = tid; q < (int)n_found; q += THREADS) {
                const uint64_t key = found[q];
                int place = 0;
                for (int o = 0; o < (int)n_found; ++o) place += found[o] > key;
                if (place < 32) ours[0][place] = key;
            }
            __syncthreads();
        } else {
            // Hundreds above the least maximum in the few threads that have them: every
            // warp keeps the best of its share in order, a key per lane.
            uint64_t list = 0, edge = bar - 1;
            for (int base = warp * 32; base < items; base += THREADS) {
                Piece<T> w;
                w.w = make_uint4(0, 0, 0, 0);
                const int j = item_of(base + lane, w), i = row.first(j);
#pragma unroll 1
                for (int e = 0; e < N; ++e) {
                    const uint64_t key = j < p1 && row.has(i + e) ? order_key(w.at(e), i + e) : 0;
                    unsigned todo = __ballot_sync(0xffffffffu, key > edge);
                    while (todo) {
                        const uint64_t k = __shfl_sync(0xffffffffu, key, __ffs(todo) - 1);
                        const int place = __popc(__ballot_sync(0xffffffffu, list > k));
                        const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
                        list = lane < place ? list : lane == place ? k : up;
                        edge = max(edge, (uint64_t)__shfl_sync(0xffffffffu, list, p.top - 1));
                        todo &= todo - 1;
                        todo &= __ballot_sync(0xffffffffu, key > edge);
                    }
                }
            }
            ours[warp][lane] = list;
            join_lists<WARPS>(ours, WARPS, warp, lane);
        }
    } else {
        __syncthreads();
    }

    // ---- the row ----
    if (cluster > 1) cluster_wait();
    if (warp == 0) {
        Part mine_part = {cta_m, 0.0f, 0.0f, 0};
#pragma unroll
        for (int i = 0; i < WARPS; ++i) mine_part.s += warp_s[i], mine_part.t += warp_t[i], mine_part.before += warp_before[i];
        if (cluster == 1) {
            if (lane == 0) parts[0] = mine_part;
            if (TOP) lists[0][lane] = ours[0][lane];
        } else {
            const uint32_t to = map_to(&parts[rank], 0);
            if (lane == 0) {
                put32(to, __float_as_uint(mine_part.m)), put32(to + 4, __float_as_uint(mine_part.s));
                put32(to + 8, __float_as_uint(mine_part.t)), put32(to + 12, mine_part.before);
            }
            if (TOP) put64(map_to(&lists[rank][lane], 0), ours[0][lane]);
        }
    }
    if (cluster > 1) {
        cluster_arrive();
        if (rank != 0) return;  // what it wrote lies in the first CTA
        cluster_wait();
    }
    if (TOP && cluster > 1) join_lists<WARPS>(lists, cluster, warp, lane);
    if (warp != 0) return;
    __syncwarp();
    float high = parts[0].m;
    for (int i = 1; i < cluster; ++i) high = max_nan(high, parts[i].m);
    const float from = fmaxf(high, -3.4028234663852886e38f);
    float s = 0.0f, t = 0.0f;
    uint32_t all_before = 0;
    for (int i = 0; i < cluster; ++i) {
        const float d = down_to(fmaxf(parts[i].m, -3.4028234663852886e38f), from), down = exp2_fast(d);
        s = fmaf(parts[i].s, down, s);
        t = fmaf(fmaf(parts[i].s, d, parts[i].t), down, t);
        all_before += parts[i].before;
    }
    const bool bad = !(high < INFINITY), empty = high == -INFINITY;
    const float ln_s = logf(s);
    auto logp = [&](float v) {
        if (bad) return NAN;
        const float below = v - high;  // where fp32 does not hold it, its half
        if (below == -INFINITY && v > -INFINITY) return (0.5f * v - 0.5f * high) * p.scale * 2.0f - ln_s;
        return v == -INFINITY ? -INFINITY : below * p.scale - ln_s;
    };
    if (lane == 0) {
        if (p.token_logprobs) p.token_logprobs[r] = token >= 0 ? logp(mine) : 0.0f;
        if (p.token_ranks) p.token_ranks[r] = token >= 0 ? (int)all_before : -1;
        if (p.entropy) p.entropy[r] = bad ? NAN : empty ? 0.0f : ln_s - t / s * kLn2;
    }
    if (TOP && lane < p.top) {
        const uint64_t key = lists[0][lane];
        const int64_t at = r * p.top + lane;
        if (p.top_ids) p.top_ids[at] = key ? (int)~(uint32_t)key : -1;
        if (p.top_logprobs) p.top_logprobs[at] = logp(key ? unordered((uint32_t)(key >> 32)) : -INFINITY);
    }
}

template <typename T, bool TOP, int THREADS, bool ENDS>
cudaError_t launch_with(const Logprobs& p, const Unit& unit, int cluster, cudaStream_t st) {
    auto* kernel = logprobs_kernel<T, TOP, THREADS, ENDS>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.rows * cluster);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cluster > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    return cudaLaunchKernelEx(&cfg, kernel, p, unit, cluster);
}

// More rows than are resident, of 64 KB and less, go in CTAs of 128 threads, of which
// twice as many hide each other's beginnings and ends: 2025 F16 rows of 11627 27 us
// instead of 43, 600 F32 rows of it 13 and 16, 1200 F16 rows of 4000 13 and 21 (333
// F16 rows of 32003, all resident, 28 and 17).
template <typename T, bool TOP>
cudaError_t launch_as(const Logprobs& p, int cluster, bool brief, cudaStream_t st) {
    const Unit unit = unit_of(p.scale, p.dtype);
    if constexpr (sizeof(T) == 4) {
        if (unit.a != 1.0f || unit.b != 1.0f) return launch_with<T, TOP, kLpThreads, true>(p, unit, cluster, st);
    }
    return brief ? launch_with<T, TOP, kLpShort, false>(p, unit, cluster, st) : launch_with<T, TOP, kLpThreads, false>(p, unit, cluster, st);
}

}  // namespace

cudaError_t launch_logprobs(const Logprobs& p, int num_sms, cudaStream_t st) {
    // CTAs of a row: as many as are resident at once, three on an SM, each with two
    // chunks' work for its threads.  More of them cost their beginnings and ends (64 F16
    // rows of 128256 in 512 CTAs 11.3 us, in 256 10.2; 2048 rows in 2 and 4 CTAs each
    // 6 and 29 % longer than in one).
    const int64_t pieces = (int64_t)p.vocab * (p.dtype == kRowF32 ? 4 : 2) / 16;
    int cluster = 1;
    while (cluster < kLpMaxCluster && (int64_t)p.rows * cluster * 2 <= 3 * num_sms && pieces / (4 * cluster) >= kLpThreads) cluster *= 2;
    const bool brief = p.rows > 3 * num_sms && pieces <= 4096;
    if (p.dtype == kRowF32) return p.top ? launch_as<float, true>(p, cluster, brief, st) : launch_as<float, false>(p, cluster, brief, st);
    return p.top ? launch_as<__half, true>(p, cluster, brief, st) : launch_as<__half, false>(p, cluster, brief, st);
}

}  // namespace lc
