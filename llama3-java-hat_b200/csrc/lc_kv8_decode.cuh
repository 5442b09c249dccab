// lc_kv8_decode.cuh -- attention over the 8-bit pages for few queries per
// sequence (decode, short continuations).
//
// Bound by the bytes of the codes: every code is read once and used by up to
// 8 rows, a row being one (query, head) pair that shares the kv head.
//
// Products.  mma.m16n8k16 on f16: codes are exact in f16 (signed bytes and
// e4m3 both), a query row is split into f16 hi + lo under a power-of-two row
// scale (22 bits), hi in MMA row g and lo in row g + 8, so both halves of the
// sum sit in one thread and the split costs no instruction beyond the 8 rows
// that GQA leaves unused anyway.  The weights p are split the same way.
// tcgen05 has no use for 8 rows of 128.
//
// Softmax.  In powers of two, with a running maximum that is only moved when
// a score passes it by more than 1; p is held as 2^(x - m + 12), times the
// page's value scale over a running reference scale (at most 4), which stays
// below 2^15 and leaves 37 bits between the largest weight and the smallest
// step of the lo half.
//
// Work.  A step is 32 tokens of one (sequence, kv head, 8 rows); all steps of
// the call form one line, cut into equal pieces, one per warp, so ragged
// lengths leave no warp idle.  A unit (all steps of 8 rows) that one warp
// covers is written at once; pieces of a unit are joined first within the
// CTA, then by the last CTA to finish, always in the order of the line, so
// the result does not depend on timing.
//
// Each warp streams its own pages through a ring in shared memory with 16-byte
// cp.async, swizzled so that the fragment loads are free of bank conflicts,
// across unit borders; warps meet only to join pieces.
#pragma once

#include "lc_internal.h"
#include "lc_kv8.cuh"

namespace lc {

constexpr int kDecWarps = 8;    // per CTA
constexpr int kDecStages = 3;   // ring stages per warp
constexpr int kDecStep = 32;    // tokens of a step
constexpr int kDecRows = 8;     // (query, head) rows of a unit

template <int D>
struct DecShape {
    static constexpr int kCtasPerSm = D == 64 ? 2 : 1;
    static constexpr int kStageBytes = 2 * kDecStep * D + 32;  // K, V, four scales and the page flags
    static constexpr int kRingBytes = kDecWarps * kDecStages * kStageBytes;
    static constexpr int kPartFloats = kDecRows * (D + 2);  // O[8][D], m[8], l[8]
};

// Workspace: a counter per CTA (zero between calls), then per warp two pieces
// and per CTA two joined pieces.
inline size_t kv8_counter_bytes(int num_sms) { return ((size_t)num_sms * 2 * sizeof(int) + 255) / 256 * 256; }
inline size_t kv8_decode_ws_bytes(int num_sms) {
    const size_t a = DecShape<64>::kCtasPerSm * DecShape<64>::kPartFloats, b = DecShape<128>::kCtasPerSm * DecShape<128>::kPartFloats;
    return kv8_counter_bytes(num_sms) + (size_t)num_sms * (kDecWarps + 1) * 2 * (a > b ? a : b) * sizeof(float);
}

LC_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

LC_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

LC_DEV uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// (a, b) -> f16 hi pair and the f16 pair of what hi leaves.
LC_DEV void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_f16(a - f.x, b - f.y);
}

// Four codes of a word -> two f16 pairs, exactly.  Signed bytes: 0x6400 | u is
// 1024 + u in f16, u = code + 128.
template <int FMT>
LC_DEV void codes_f16(uint32_t w, uint32_t& p01, uint32_t& p23) {
    if (FMT == kKv8I8) {
        const uint32_t bias = 0x64806480u;  // 1152
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
        const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
        p01 = *reinterpret_cast<const uint32_t*>(&x);
        p23 = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(p01), "=r"(p23)
            : "r"(w));
    }
}

LC_DEV void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
LC_DEV void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
LC_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
LC_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

LC_DEV uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
LC_DEV uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}

// Byte offset of 16-byte chunk c of token row r in a stage's K or V half.
template <int D>
LC_DEV int ring_offset(int r, int c) {
    if (D == 64) return (r ^ ((r >> 2) & 1)) * 64 + ((c ^ (r & 2)) << 4);
    return r * 128 + ((c ^ (r & 6) ^ ((r & 1) << 2)) << 4);
}

// The queries of sequence s: first row, count, and the positions of its cache.
struct SeqInfo {
    int row0, nq, len;
};
LC_DEV SeqInfo kv8_seq(const Kv8Attention& a, int page_shift, int s) {
    SeqInfo q;
    if (a.q_start) {
        q.row0 = a.q_start[s];
        const int e = a.q_start[s + 1];
        q.nq = q.row0 < 0 || e > a.rows || e < q.row0 ? 0 : e - q.row0;  // rows outside the buffers are no queries
    } else {
        q.row0 = s;
        q.nq = 1;
    }
    q.len = a.kv_lens[s];
    return q;
}

// A place on the line of steps.
struct DecCursor {
    int s, head, chunk;  // unit
    int step, steps;     // within the unit
    SeqInfo q;
    int chunks;          // of the sequence
};

// Steps of rows [8 chunk, 8 chunk + 8) of a sequence: up to the last query's
// last position, at least one (which then sees nothing and writes zeros).
LC_DEV int dec_seen(const SeqInfo& q, int group, int room, int row) {
    const int j = row / group;
    const int seen = q.len - q.nq + (j < q.nq ? j : q.nq - 1) + 1;
    return seen < 0 ? 0 : seen > room ? room : seen;
}
LC_DEV int dec_steps(const SeqInfo& q, int group, int room, int chunk) {
    const int seen = dec_seen(q, group, room, chunk * kDecRows + kDecRows - 1);
    return seen <= 0 ? 1 : (seen + kDecStep - 1) / kDecStep;
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kDecWarps * 32, DecShape<D>::kCtasPerSm)
kv8_decode_kernel(Kv8 c, Kv8Attention a, float* __restrict__ ws, int* __restrict__ counters) {
    using S = DecShape<D>;
    constexpr int KS = D / 16;   // k-steps of a score
    constexpr int NV = D / 8;    // n-tiles of the output
    extern __shared__ __align__(128) uint8_t smem[];
    unsigned* prefix = reinterpret_cast<unsigned*>(smem + S::kRingBytes);  // [n_seqs + 1] steps before sequence s
    __shared__ unsigned scan[kDecWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.n_heads / c.n_kv, sh = c.page_shift;
    const int room = (int)min((long long)a.table_stride << sh, 0x7fffffffll);
    griddep_launch();
    griddep_wait();

    // ---- the line of steps ----
    unsigned carry = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += kDecWarps * 32) {
        const int s = s0 + tid;
        unsigned cost = 0;
        if (s < a.n_seqs) {
            const SeqInfo q = kv8_seq(a, sh, s);
            const int chunks = (q.nq * group + kDecRows - 1) / kDecRows;
            for (int k = 0; k < chunks; ++k) cost += dec_steps(q, group, room, k);
            cost *= c.n_kv;
        }
        unsigned v = cost;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        unsigned before = carry, all = carry;
        for (int w = 0; w < kDecWarps; ++w) {
            if (w < warp) before += scan[w];
            all += scan[w];
        }
        if (s < a.n_seqs) prefix[s] = before + v - cost;
        carry = all;
        __syncthreads();
    }
    if (tid == 0) prefix[a.n_seqs] = carry;
    __syncthreads();
    const long long total = carry;
    if (total == 0) return;
    const long long workers = min((long long)gridDim.x * kDecWarps, total);
    auto begin_of = [&](long long w) { return w * total / workers; };
    auto worker_of = [&](long long x) { return ((x + 1) * workers - 1) / total; };  // the worker of step x
    const long long w0 = (long long)blockIdx.x * kDecWarps;  // this CTA's first worker
    if (w0 >= workers) return;
    const int my_warps = (int)min((long long)kDecWarps, workers - w0);
    const long long cta_lo = begin_of(w0), cta_hi = begin_of(w0 + my_warps);
    const long long lo = warp < my_warps ? begin_of(w0 + warp) : cta_hi;
    const long long hi = warp < my_warps ? begin_of(w0 + warp + 1) : cta_hi;

    auto locate = [&](DecCursor& cur, long long x) {  // the unit and step at place x
        int a0 = 0, a1 = a.n_seqs;
        while (a1 - a0 > 1) {
            const int mid = (a0 + a1) >> 1;
            if (prefix[mid] <= x) a0 = mid;
            else a1 = mid;
        }
        cur.s = a0;
        cur.q = kv8_seq(a, sh, a0);
        cur.chunks = (cur.q.nq * group + kDecRows - 1) / kDecRows;
        unsigned rem = (unsigned)(x - prefix[a0]);
        const unsigned per = (prefix[a0 + 1] - prefix[a0]) / c.n_kv;
        cur.head = rem / per;
        rem -= cur.head * per;
        cur.chunk = 0;
        cur.steps = dec_steps(cur.q, group, room, 0);
        while (rem >= (unsigned)cur.steps) {
            rem -= cur.steps;
            cur.steps = dec_steps(cur.q, group, room, ++cur.chunk);
        }
        cur.step = rem;
    };
    auto next_unit = [&](DecCursor& cur) {
        cur.step = 0;
        if (++cur.chunk == cur.chunks) {
            cur.chunk = 0;
            if (++cur.head == c.n_kv) {
                cur.head = 0;
                do ++cur.s;
                while (cur.s < a.n_seqs - 1 && prefix[cur.s + 1] == prefix[cur.s]);
                cur.q = kv8_seq(a, sh, cur.s);
                cur.chunks = (cur.q.nq * group + kDecRows - 1) / kDecRows;
            }
        }
        cur.steps = dec_steps(cur.q, group, room, cur.chunk);
    };

    float* const warp_parts = ws;                                                            // [workers][2]
    float* const cta_parts = ws + (size_t)gridDim.x * kDecWarps * 2 * S::kPartFloats;       // [CTAs][2]
    const uint32_t ring = smem_u32(smem) + warp * kDecStages * S::kStageBytes;
    const int row_sel = sh == 4 ? 1 : 0;  // pages of 16 tokens: a step's second half is another page

    // Writes row r (0..7 of the unit at `cur`) of the result.
    auto out_row = [&](const DecCursor& cur, int r) -> T* {
        const int row = cur.chunk * kDecRows + r, j = row / group;
        if (j >= cur.q.nq) return nullptr;
        return (T*)a.out + (int64_t)(cur.q.row0 + j) * a.out_stride + (cur.head * group + row - j * group) * D;
    };

    if (lo < hi) {
        // ---- issue side ----
        DecCursor ic;  // the next step to ask for
        locate(ic, lo);
        long long ahead = lo;
        int id0 = 0, id1 = 0;  // its pages
        auto ids = [&]() {
            const int seen = dec_seen(ic.q, group, room, ic.chunk * kDecRows + kDecRows - 1);
            const int32_t* row = a.table + (int64_t)ic.s * a.table_stride;
            const int t0 = ic.step * kDecStep;
            id0 = t0 < seen ? row[t0 >> sh] : -1;
            id1 = !row_sel ? id0 : t0 + 16 < seen ? row[(t0 + 16) >> sh] : -1;
        };
        ids();
        const int off0 = lane * 16;  // this lane's first chunk of a half
        const int r0 = off0 / D, ch0 = (off0 % D) / 16;
        const int dst0 = ring_offset<D>(r0, ch0);
        constexpr int kCopies = kDecStep * D / 512;  // 16-byte copies per lane for K, and for V
        auto issue = [&](int stage) {
            if (ahead < hi) {
                const uint32_t st = ring + stage * S::kStageBytes;
                const bool ok0 = (unsigned)id0 < (unsigned)c.n_pages, ok1 = (unsigned)id1 < (unsigned)c.n_pages;
                const int in_page = (ic.step * kDecStep) & ((1 << sh) - 1);
                const int64_t b0 = ((((int64_t)id0 * c.n_kv + ic.head) << sh) + in_page) * D;
                const int64_t b1 = row_sel ? (((int64_t)id1 * c.n_kv + ic.head) << sh) * D : b0 + 16 * D;
#pragma unroll
                for (int k = 0; k < kCopies; ++k) {
                    const bool second = k >= kCopies / 2;
                    if (second ? ok1 : ok0) {
                        const int64_t at = (second ? b1 + (k - kCopies / 2) * 512 : b0 + k * 512) + off0;
                        // rows of copy k are 512 / D further: a multiple of the swizzle's period only for D = 64
                        const uint32_t d = D == 64 ? dst0 + k * 512 : ring_offset<D>(r0 + k * (512 / D), ch0);
                        cp_async16(st + d, c.k + at);
                        cp_async16(st + kDecStep * D + d, c.v + at);
                    }
                }
                if (lane < 4) {
                    const bool ok = (lane & 1) ? ok1 : ok0;
                    const int64_t at = (int64_t)((lane & 1) ? id1 : id0) * c.n_kv + ic.head;
                    if (ok) cp_async4(st + 2 * kDecStep * D + lane * 4, (lane & 2 ? c.v_scale : c.k_scale) + at);
                }
                if (lane == 0)
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(st + 2 * kDecStep * D + 16), "r"((ok0 ? 1 : 0) | (ok1 ? 2 : 0)) : "memory");
                ++ahead;
                if (++ic.step == ic.steps && ahead < hi) next_unit(ic);
                if (ahead < hi) ids();
            }
            cp_async_commit();
        };
        for (int k = 0; k < kDecStages - 1; ++k) issue(k);

        // ---- compute side ----
        DecCursor cur;
        locate(cur, lo);
        int stage = 0;
        for (long long x = lo; x < hi;) {
            // One segment: steps [cur.step, last) of the unit.
            const int first_step = cur.step;
            const int last = (int)min((long long)cur.steps, cur.step + (hi - x));
            const int row = cur.chunk * kDecRows + g, j = row / group;
            const bool live = j < cur.q.nq;
            const int seen = live ? dec_seen(cur.q, group, room, row) : 0;
            const int seen_min = dec_seen(cur.q, group, room, cur.chunk * kDecRows);
            const int seen_max = dec_seen(cur.q, group, room, cur.chunk * kDecRows + kDecRows - 1);
            const bool all_live = (cur.chunk + 1) * kDecRows <= cur.q.nq * group;
            // Query fragments: k-step ks of thread t covers 4 neighbouring elements.
            uint32_t qa[KS][4];
            float qf;
            {
                float v[KS * 4];
                const T* q = (const T*)a.q + (int64_t)(cur.q.row0 + (live ? j : 0)) * a.q_stride +
                             (cur.head * group + (live ? row - j * group : 0)) * D;
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < KS * 4; ++i) {
                    v[i] = live ? (float)q[(i / 16) * 64 + t * 16 + i % 16] : 0.0f;
                    top = fmaxf(top, fabsf(v[i]));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^e puts the row's largest element in [2^9, 2^10)
                int e = top > 0.0f ? 9 - (((__float_as_int(top) >> 23) & 0xff) - 127) : 0;
                e = max(-126, min(126, e));
                const float up = __int_as_float((127 + e) << 23);
                qf = a.scale * 1.4426950408889634f * __int_as_float((127 - e) << 23);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    split_f16(v[4 * ks] * up, v[4 * ks + 1] * up, qa[ks][0], qa[ks][1]);
                    split_f16(v[4 * ks + 2] * up, v[4 * ks + 3] * up, qa[ks][2], qa[ks][3]);
                }
            }
            float o[NV][4];
#pragma unroll
            for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            float m = -INFINITY, l = 0.0f, vref = 0.0f, vinv = 0.0f;

            for (; cur.step < last; ++cur.step, ++x) {
                cp_async_wait<kDecStages - 2>();
                __syncwarp();  // the stage's copies of all lanes are there, and the previous stage is read
                issue(stage == 0 ? kDecStages - 1 : stage - 1);
                const uint32_t kb = ring + stage * S::kStageBytes, vb = kb + kDecStep * D, sb = vb + kDecStep * D;
                const uint4 sc = lds128(sb);
                uint32_t flags;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(flags) : "r"(sb + 16));
                const float ks0 = (flags & 1) ? __uint_as_float(sc.x) : 0.0f, ks1 = (flags & 2) ? __uint_as_float(sc.y) : 0.0f;
                const float vs0 = (flags & 1) ? __uint_as_float(sc.z) : 0.0f, vs1 = (flags & 2) ? __uint_as_float(sc.w) : 0.0f;
                const int t0 = cur.step * kDecStep;

                float s[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
                    for (int hf = 0; hf < D / 64; ++hf) {
                        const uint4 w = lds128(kb + n * 8 * D + ring_offset<D>(g, hf * 4 + t));
                        const uint32_t wk[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t b0, b1;
                            codes_f16<FMT>(wk[k], b0, b1);
                            mma_f16(s[n], qa[hf * 4 + k], b0, b1);
                        }
                    }
                }
                // Scores in powers of two; hi and lo halves meet here.
                float p[8];
                const float c0 = qf * ks0, c1 = qf * ks1;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    p[2 * n] = (s[n][0] + s[n][2]) * (n < 2 ? c0 : c1);
                    p[2 * n + 1] = (s[n][1] + s[n][3]) * (n < 2 ? c0 : c1);
                }
                const bool whole = t0 + kDecStep <= seen_min && flags == 3 && all_live;
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int tok = t0 + (i >> 1) * 8 + 2 * t + (i & 1);
                        if (tok >= seen || !(flags & (i < 4 ? 1 : 2))) p[i] = -INFINITY;
                    }
                }
                float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const bool move = top > m + 1.0f;
                const float vmax = fmaxf(vs0, vs1);
                if (__any_sync(0xffffffffu, move) || vmax > 4.0f * vref) {
                    float f = 1.0f;
                    if (move) {
                        f = ex2(m - top);
                        l *= f;
                        m = top;
                    }
                    if (vmax > 4.0f * vref) {
                        const float next = fmaxf(vmax, 1e-30f);
                        vinv = 1.0f / next;
                        f *= vref * vinv;
                        vref = next;
                    }
#pragma unroll
                    for (int i = 0; i < NV; ++i) o[i][0] *= f, o[i][1] *= f, o[i][2] *= f, o[i][3] *= f;
                }
                const float bias = m == -INFINITY ? 0.0f : 12.0f - m;
                const float v0 = vs0 * vinv, v1 = vs1 * vinv;
                uint32_t pa[2][4];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = ex2(p[i] + bias);
                    l += p[i];
                    p[i] *= i < 4 ? v0 : v1;
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) split_f16(p[2 * n], p[2 * n + 1], pa[n >> 1][(n & 1) * 2], pa[n >> 1][(n & 1) * 2 + 1]);
                // Values: thread t's tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each 16, elements g D / 8 ...
                const bool clean = FMT == kKv8I8 || (t0 + kDecStep <= seen_max && flags == 3);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    uint32_t w[4][D / 32];  // token, word
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int r = 2 * t + (b & 1);
                        const uint32_t at = vb + (kk * 16 + (b >> 1) * 8) * D;
                        if (D == 64) {
                            const uint2 u = lds64(at + ring_offset<D>(r, g >> 1) + (g & 1) * 8);
                            w[b][0] = u.x, w[b][1] = u.y;
                        } else {
                            const uint4 u = lds128(at + ring_offset<D>(r, g));
                            w[b][0] = u.x, w[b][1] = u.y, w[b][D / 32 - 2] = u.z, w[b][D / 32 - 1] = u.w;
                        }
                        if (!clean) {  // what lies behind the end may be NaN
                            const int tok = t0 + kk * 16 + (b >> 1) * 8 + r;
                            if (tok >= seen_max || !(flags & (kk ? 2 : 1)))
#pragma unroll
                                for (int e = 0; e < D / 32; ++e) w[b][e] = 0;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) {
                        // bytes of two tokens side by side: (token 2t, token 2t + 1) of an element
                        uint32_t b0[4], b1[4];
                        codes_f16<FMT>(__byte_perm(w[0][e], w[1][e], 0x5140), b0[0], b0[1]);
                        codes_f16<FMT>(__byte_perm(w[0][e], w[1][e], 0x7362), b0[2], b0[3]);
                        codes_f16<FMT>(__byte_perm(w[2][e], w[3][e], 0x5140), b1[0], b1[1]);
                        codes_f16<FMT>(__byte_perm(w[2][e], w[3][e], 0x7362), b1[2], b1[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma_f16(o[e * 4 + i], pa[kk], b0[i], b1[i]);
                    }
                }
                stage = stage == kDecStages - 1 ? 0 : stage + 1;
            }
            // ---- the segment's end ----
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            // Thread t holds elements [2t D/8, (2t + 2) D/8) of row g.
            const bool whole_unit = first_step == 0 && last == cur.steps;
            const float f = whole_unit ? (l > 0.0f ? vref / l : (l == 0.0f ? 0.0f : l)) : vref;
            if (whole_unit) {
                T* dst = out_row(cur, g);
                if (dst) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < NV; ++i) dst[(2 * t + b) * NV + i] = (T)(l == 0.0f ? 0.0f : (o[i][b] + o[i][2 + b]) * f);
                }
            } else {
                float* part = warp_parts + ((size_t)(w0 + warp) * 2 + (first_step == 0 ? 1 : 0)) * S::kPartFloats;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < NV; ++i) part[g * D + (2 * t + b) * NV + i] = (o[i][b] + o[i][2 + b]) * f;
                if (t == 0) {
                    part[kDecRows * D + g] = m;
                    part[kDecRows * D + kDecRows + g] = l;
                }
            }
            if (cur.step == cur.steps && x < hi) next_unit(cur);
        }
        cp_async_wait<0>();
    }
    __syncthreads();

    // ---- joining pieces ----
    // Sum of n pieces (piece(i) gives the i-th) by one warp: lane's four
    // neighbouring elements of rows (lane * 4 + 128 k) / D.
    constexpr int KM = kDecRows * D / 128;
    auto join = [&](int n, auto piece, float* to, const DecCursor& cur, bool finish) {
        float mx[KM], sum[KM];
        float4 acc[KM];
#pragma unroll
        for (int k = 0; k < KM; ++k) mx[k] = -INFINITY, sum[k] = 0.0f, acc[k] = make_float4(0, 0, 0, 0);
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int k = 0; k < KM; ++k) mx[k] = fmaxf(mx[k], __ldcg(piece(i) + kDecRows * D + (lane * 4 + 128 * k) / D));
        for (int i = 0; i < n; ++i) {
            const float* p = piece(i);
#pragma unroll
            for (int k = 0; k < KM; ++k) {
                const int e = lane * 4 + 128 * k, r = e / D;
                const float pm = __ldcg(p + kDecRows * D + r);
                const float f = pm == -INFINITY ? 0.0f : ex2(pm - mx[k]);
                const float4 v = __ldcg(reinterpret_cast<const float4*>(p + e));
                sum[k] += f * __ldcg(p + kDecRows * D + kDecRows + r);
                acc[k].x += f * v.x, acc[k].y += f * v.y, acc[k].z += f * v.z, acc[k].w += f * v.w;
            }
        }
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            const int e = lane * 4 + 128 * k, r = e / D;
            if (finish) {
                T* dst = out_row(cur, r);
                if (!dst) continue;
                dst += e % D;
                const float inv = sum[k] == 0.0f ? 0.0f : 1.0f / sum[k];
                dst[0] = (T)(acc[k].x * inv), dst[1] = (T)(acc[k].y * inv);
                dst[2] = (T)(acc[k].z * inv), dst[3] = (T)(acc[k].w * inv);
            } else {
                *reinterpret_cast<float4*>(to + e) = acc[k];
                if (e % D == 0) to[kDecRows * D + r] = mx[k], to[kDecRows * D + kDecRows + r] = sum[k];
            }
        }
    };
    // A warp joins the pieces of the unit that begins in it and goes on, and
    // warp 0 those of the unit that was under way at the CTA's start.
    if (lo >= hi) return;
    for (int side = warp == 0 ? 0 : 1; side < 2; ++side) {
        DecCursor cur;
        const long long at = side == 0 ? lo : hi - 1;
        locate(cur, at);
        const long long u0 = at - cur.step, u1 = u0 + cur.steps;  // the unit's place on the line
        if (side == 0 ? u0 >= lo : !(u0 >= lo && u1 > hi)) continue;
        const long long end = min(u1, cta_hi);
        const int wn = (int)(worker_of(end - 1) - (w0 + warp)) + 1;  // warps with a piece, from this one
        auto mine = [&](int i) -> const float* {
            return warp_parts + ((size_t)(w0 + warp + i) * 2 + (i == 0 ? side : 0)) * S::kPartFloats;
        };
        if (u0 >= cta_lo && u1 <= cta_hi) {
            join(wn, mine, nullptr, cur, true);
            continue;
        }
        join(wn, mine, cta_parts + ((size_t)blockIdx.x * 2 + side) * S::kPartFloats, cur, false);
        const int first = (int)(worker_of(u0) / kDecWarps), final = (int)(worker_of(u1 - 1) / kDecWarps);
        __threadfence();
        __syncwarp();
        int old = 0;
        if (lane == 0) old = atomicAdd(counters + first, 1);
        old = __shfl_sync(0xffffffffu, old, 0);
        if (old != final - first) continue;
        if (lane == 0) counters[first] = 0;
        __threadfence();
        auto all = [&](int i) -> const float* {
            return cta_parts + ((size_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * S::kPartFloats;
        };
        join(final - first + 1, all, nullptr, cur, true);
    }
}

template <typename T, int FMT, int D>
cudaError_t kv8_decode_prepare() {
    return cudaFuncSetAttribute(kv8_decode_kernel<T, FMT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                DecShape<D>::kRingBytes + (kPagesMaxSeqs + 1) * (int)sizeof(unsigned));
}

template <typename T, int FMT, int D>
cudaError_t launch_kv8_decode(const Kv8& c, const Kv8Attention& a, int num_sms, void* ws, cudaStream_t st) {
    const int smem = DecShape<D>::kRingBytes + (a.n_seqs + 1) * (int)sizeof(unsigned);
    int* counters = (int*)ws;
    float* parts = (float*)((uint8_t*)ws + kv8_counter_bytes(num_sms));
    return launch_ex(kv8_decode_kernel<T, FMT, D>, dim3(num_sms * DecShape<D>::kCtasPerSm), dim3(kDecWarps * 32), smem, st,
                     true, c, a, parts, counters);
}

}  // namespace lc
