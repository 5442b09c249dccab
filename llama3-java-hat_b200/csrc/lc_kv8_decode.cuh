// lc_kv8_decode.cuh -- attention over the 8-bit pages for few queries per
// sequence (decode, short continuations).
//
// Bound by the bytes of the codes: every code is read once and used by up to
// 8 rows, a row being one (query, head) pair that shares the kv head.
//
// Products.  mma.m16n8k16 on f16: codes are exact in f16 (signed bytes and
// e4m3 both).  Keys and values are the 16-row operand (tokens, or elements of
// the head), the rows of the unit the 8-column one: row h is split into f16
// hi + lo under a power-of-two row scale (22 bits), columns 2h and 2h + 1 of a
// tile, so both halves of a sum meet in one thread and four rows, a common
// group, fill a tile.  The weights p are split the same way and change from
// the score's layout (tokens over lanes) to the operand's (tokens along k)
// through 512 bytes of shared memory.  With the rows as the 16-row operand
// instead half the products and half the exponentials were spent on empty
// rows.  tcgen05 has no use for 8 rows of 128.
//
// Sums.  The tensor cores' own fp32 sums lose up to one unit of the last place,
// always toward zero, at every product that is added: over a unit of 65536
// positions 4.3e-4 of the result where all values have one sign.  So a product
// of weights and values begins at zero, its hi and lo sums meet, and are added
// to the unit's in round-to-nearest (4.4e-6).  That also halves the
// accumulators' registers: 64 sequences of 1 to 8191 positions, fp32, take 60.7
// us at head size 64 (60.3 with the tensor cores' sums) and 106.8 at 128 (112.5).
//
// Softmax.  In powers of two, with a running maximum that is only moved when
// a score passes it by more than 1; p is held as 2^(x - m + 12), times the
// page's value scale over a running reference scale (at most 4), which stays
// below 2^15 and leaves 37 bits between the largest weight and the smallest
// step of the lo half.
//
// Work.  A step is 4 KB of codes, 32 tokens of head size 64 or 16 of 128, of
// one (sequence, kv head, 4 or 8 rows); all steps of the call form one line, cut
// into equal pieces, one per warp, so ragged lengths leave no warp idle.  A unit
// (all steps of those rows) that one warp covers is written at once; pieces of
// a unit are joined first within the CTA, then by the last CTA to finish, always
// in the order of the line, so the result does not depend on timing.
//
// Each warp streams its own pages through a ring in shared memory with 16-byte
// cp.async, swizzled so that the fragment loads are free of bank conflicts,
// across unit borders; warps meet only to join pieces.
#pragma once

#include "lc_internal.h"
#include "lc_kv8.cuh"

namespace lc {

constexpr int kDecWarps = 8;  // per CTA
constexpr int kDecUnitCost = 1;     // a unit's beginning and end, in steps
constexpr int kDecSeqsShared = 512;  // up to here the sequences' places are kept in shared memory

// D: head size; NR: tiles of 4 rows of a unit, 1 or 2.
template <int D, int NR>
struct DecShape {
    static constexpr int kRows = 4 * NR;
    static constexpr int kStep = 2048 / D;  // tokens of a step: 4 KB of codes
    static constexpr int kCtasPerSm = D == 128 && NR == 2 ? 1 : 2;  // 128 registers would spill there
    static constexpr int kStages = 3;
    static constexpr int kStageBytes = 2 * kStep * D + 32;              // K, V, four scales and the page flags
    static constexpr int kWarpBytes = kStages * kStageBytes + 512 * NR;  // and the weights
    static constexpr int kRingBytes = kDecWarps * kWarpBytes;
    static constexpr int kPartFloats = kRows * (D + 2);  // O[rows][D], m[rows], l[rows]
    static_assert(kPartFloats * 4 <= kStages * kStageBytes, "a piece fits the warp's ring");
};

// Workspace: a counter per CTA (zero between calls), then per warp a piece and
// per CTA two joined pieces.
inline size_t kv8_counter_bytes(int num_sms) { return ((size_t)num_sms * 2 * sizeof(int) + 255) / 256 * 256; }
inline size_t kv8_decode_ws_bytes(int num_sms) {
    return kv8_counter_bytes(num_sms) + (size_t)num_sms * 2 * (kDecWarps + 2) * DecShape<128, 2>::kPartFloats * sizeof(float);
}

LC_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The product alone.
LC_DEV void mma_f16_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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
LC_DEV void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
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
    q.len = max(0, a.kv_lens[s]);
    return q;
}

// A unit of the line of steps: rows [R chunk, R chunk + R) of the (query, head)
// pairs of one sequence and kv head, and a step within it.
struct DecCursor {
    SeqInfo q;
    int s, head, chunk, chunks;
    int seen;         // positions that its last row sees
    int step, steps;  // steps up to there; at least one, which then sees nothing and writes zeros
};

// Positions that row `row` (query row / group) of a sequence sees.
LC_DEV int dec_seen(const SeqInfo& q, int group, int room, int row) {
    const int j = row / group;
    const int seen = q.len - q.nq + (j < q.nq ? j : q.nq - 1) + 1;
    return seen < 0 ? 0 : seen > room ? room : seen;
}
template <int STEP>
LC_DEV int dec_steps(int seen) {
    return seen <= STEP ? 1 : (seen + STEP - 1) / STEP;
}

template <typename T, int FMT, int D, int NR>
__global__ void __launch_bounds__(kDecWarps * 32, DecShape<D, NR>::kCtasPerSm)
kv8_decode_kernel(Kv8 c, Kv8Attention a, float* __restrict__ ws, int* __restrict__ counters) {
    using S = DecShape<D, NR>;
    constexpr int R = S::kRows;
    constexpr int KS = D / 16;  // k-steps of a score, and tiles of 16 elements of the output
    constexpr int E = D / 8;    // elements of a row that a thread holds
    constexpr int STEP = S::kStep, MT = STEP / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    unsigned* prefix = reinterpret_cast<unsigned*>(smem + S::kRingBytes);  // [n_seqs + 1] the line before sequence s
    __shared__ unsigned long long scan[kDecWarps];
    __shared__ SeqInfo infos[kDecSeqsShared];
    __shared__ DecCursor first_unit;  // warp 0's first unit, for the joining
    __shared__ DecCursor done_cursor[2];
    __shared__ int done_pieces[2];
    __shared__ int done_unit[2];  // cross-CTA units whose last piece this CTA brought
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.n_heads / c.n_kv, sh = c.page_shift;
    const int room = (int)min((long long)a.table_stride << sh, 0x7fffffffll);
    griddep_launch();
    griddep_wait();

    // The queries come to L2 while the line is laid out.
    {
        const int64_t bytes = (int64_t)a.n_heads * D * sizeof(T);  // of a row, 128 at a time
        const int per = (int)((bytes + 127) / 128);
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + tid; i < (int64_t)a.rows * per; i += (int64_t)gridDim.x * blockDim.x)
            asm volatile("prefetch.global.L2 [%0];" ::"l"((const uint8_t*)a.q + (i / per) * a.q_stride * (int)sizeof(T) + min((i % per) * 128, bytes - 1)));
    }
    if (tid < 2) done_unit[tid] = 0;

    // ---- the line of steps ----
    // A unit takes its steps and kDecUnitCost empty places behind them.
    unsigned long long carry = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += kDecWarps * 32) {
        const int s = s0 + tid;
        unsigned long long cost = 0;
        if (s < a.n_seqs) {
            const SeqInfo q = kv8_seq(a, sh, s);
            if (s < kDecSeqsShared) infos[s] = q;
            const int chunks = (q.nq * group + R - 1) / R;
            for (int k = 0; k < chunks; ++k) cost += kDecUnitCost + dec_steps<STEP>(dec_seen(q, group, room, k * R + R - 1));
            cost *= c.n_kv;
        }
        unsigned long long v = cost;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        unsigned long long before = carry, all = carry;
        for (int w = 0; w < kDecWarps; ++w) {
            if (w < warp) before += scan[w];
            all += scan[w];
        }
        if (s < a.n_seqs) prefix[s] = (unsigned)(before + v - cost);
        carry = all;
        __syncthreads();
    }
    if (carry > 0xffffffffull) return;  // the host has checked it for ascending q_start
    if (tid == 0) prefix[a.n_seqs] = (unsigned)carry;
    __syncthreads();
    // Worker w has steps [begin_of(w), begin_of(w + 1)): equal shares, the first
    // `extra` workers one step more.
    const unsigned total = (unsigned)carry;
    if (total == 0) return;
    const unsigned workers = min(gridDim.x * kDecWarps, total);
    const unsigned share = total / workers, extra = total - share * workers;
    auto begin_of = [&](unsigned w) { return w * share + min(w, extra); };
    auto worker_of = [&](unsigned x) {
        const unsigned big = extra * (share + 1);
        return x < big ? x / (share + 1) : extra + (x - big) / share;
    };
    const unsigned w0 = blockIdx.x * kDecWarps;  // this CTA's first worker
    if (w0 >= workers) return;
    const unsigned my_warps = min((unsigned)kDecWarps, workers - w0);
    const unsigned cta_lo = begin_of(w0), cta_hi = begin_of(w0 + my_warps);
    unsigned lo = warp < my_warps ? begin_of(w0 + warp) : cta_hi;
    const unsigned hi = warp < my_warps ? begin_of(w0 + warp + 1) : cta_hi;

    auto set_chunk = [&](DecCursor& cur, int chunk) {
        cur.chunk = chunk;
        cur.seen = dec_seen(cur.q, group, room, chunk * R + R - 1);
        cur.steps = dec_steps<STEP>(cur.seen);
    };
    auto set_seq = [&](DecCursor& cur, int s) {
        cur.s = s;
        cur.q = s < kDecSeqsShared ? infos[s] : kv8_seq(a, sh, s);
        cur.chunks = (cur.q.nq * group + R - 1) / R;
    };
    auto locate = [&](DecCursor& cur, unsigned x) {  // the unit and step at place x
        int a0 = 0, a1 = a.n_seqs;
        while (a1 - a0 > 1) {
            const int mid = (a0 + a1) >> 1;
            if (prefix[mid] <= x) a0 = mid;
            else a1 = mid;
        }
        set_seq(cur, a0);
        unsigned rem = x - prefix[a0];
        const unsigned per = (prefix[a0 + 1] - prefix[a0]) / c.n_kv;
        cur.head = rem / per;
        rem -= cur.head * per;
        set_chunk(cur, 0);
        while (rem >= (unsigned)(cur.steps + kDecUnitCost)) {
            rem -= cur.steps + kDecUnitCost;
            set_chunk(cur, cur.chunk + 1);
        }
        cur.step = rem;
    };
    auto next_unit = [&](DecCursor& cur) {
        cur.step = 0;
        if (cur.chunk + 1 < cur.chunks) {
            set_chunk(cur, cur.chunk + 1);
            return;
        }
        if (++cur.head == c.n_kv) {
            cur.head = 0;
            int s = cur.s;
            do ++s;
            while (s < a.n_seqs - 1 && prefix[s + 1] == prefix[s]);
            set_seq(cur, s);
        }
        if (cur.chunk != 0 || cur.head == 0) set_chunk(cur, 0);
    };

    float* const warp_parts = ws;                                                   // [workers]
    float* const cta_parts = ws + (size_t)gridDim.x * kDecWarps * S::kPartFloats;  // [CTAs][2]
    auto ring_part = [&](int w) { return reinterpret_cast<float*>(smem + w * S::kWarpBytes); };
    const uint32_t ring = smem_u32(smem) + warp * S::kWarpBytes;
    const uint32_t weights = ring + S::kStages * S::kStageBytes;
    const int row_sel = sh == 4 ? 1 : 0;  // pages of 16 tokens: a step's second half is another page

    // Row r of the unit at `cur` in the result.
    auto out_row = [&](const DecCursor& cur, int r) -> T* {
        const int row = cur.chunk * R + r, j = row / group;
        if (j >= cur.q.nq) return nullptr;
        return (T*)a.out + (int64_t)(cur.q.row0 + j) * a.out_stride + (cur.head * group + row - j * group) * D;
    };

    DecCursor cur;       // in the end: the unit of the warp's last step, cur.step behind it
    unsigned x_end = 0;  // the place behind the warp's last step
    if (lo < hi) {
        // ---- issue side ----
        DecCursor ic;  // the next step to ask for
        locate(ic, lo);
        if (ic.step >= ic.steps) {  // the empty places behind a unit
            lo = min(hi, lo + ic.steps + kDecUnitCost - ic.step);
            if (lo < hi) next_unit(ic);
        }
        if (warp == 0 && lane == 0) first_unit = ic;
        unsigned ahead = lo;
        int id0 = 0, id1 = 0;  // its pages
        auto ids = [&]() {
            const int32_t* row = a.table + (int64_t)ic.s * a.table_stride;
            const int t0 = ic.step * STEP;
            id0 = t0 < ic.seen ? row[t0 >> sh] : -1;
            id1 = MT == 1 || !row_sel ? id0 : t0 + 16 < ic.seen ? row[(t0 + 16) >> sh] : -1;
        };
        if (lo < hi) ids();
        const int off0 = lane * 16;  // this lane's first chunk of a half
        const int r0 = off0 / D, ch0 = (off0 % D) / 16;
        const int dst0 = ring_offset<D>(r0, ch0);
        constexpr int kCopies = STEP * D / 512;  // 16-byte copies per lane for K, and for V
        auto issue = [&](int stage) {
            if (ahead < hi) {
                const uint32_t st = ring + stage * S::kStageBytes;
                const bool ok0 = (unsigned)id0 < (unsigned)c.n_pages, ok1 = (unsigned)id1 < (unsigned)c.n_pages;
                const int in_page = (ic.step * STEP) & ((1 << sh) - 1);
                const int64_t b0 = ((((int64_t)id0 * c.n_kv + ic.head) << sh) + in_page) * D;
                const int64_t b1 = row_sel ? (((int64_t)id1 * c.n_kv + ic.head) << sh) * D : b0 + 16 * D;
#pragma unroll
                for (int k = 0; k < kCopies; ++k) {
                    const bool second = MT == 2 && k >= kCopies / 2;
                    if (second ? ok1 : ok0) {
                        const int64_t at = (second ? b1 + (k - kCopies / 2) * 512 : b0 + k * 512) + off0;
                        // rows of copy k are 512 / D further: a multiple of the swizzle's period only for D = 64
                        const uint32_t d = D == 64 ? dst0 + k * 512 : ring_offset<D>(r0 + k * (512 / D), ch0);
                        cp_async16(st + d, c.k + at);
                        cp_async16(st + STEP * D + d, c.v + at);
                    }
                }
                if (lane < 4) {
                    const bool ok = (lane & 1) ? ok1 : ok0;
                    const int64_t at = (int64_t)((lane & 1) ? id1 : id0) * c.n_kv + ic.head;
                    if (ok) cp_async4(st + 2 * STEP * D + lane * 4, (lane & 2 ? c.v_scale : c.k_scale) + at);
                }
                if (lane == 0)
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(st + 2 * STEP * D + 16), "r"((ok0 ? 1 : 0) | (MT == 2 && ok1 ? 2 : 0)) : "memory");
                ++ahead;
                if (++ic.step == ic.steps) {
                    ahead += kDecUnitCost;
                    if (ahead < hi) next_unit(ic);
                }
                if (ahead < hi) ids();
            }
            cp_async_commit();
        };
        const DecCursor ic0 = ic;
        for (int k = 0; k < S::kStages - 1; ++k) issue(k);

        // ---- compute side ----
        cur = ic0;
        int stage = 0;
        for (unsigned x = lo; x < hi;) {
            // One segment: steps [cur.step, last) of the unit.
            const int first_step = cur.step;
            const int last = min(cur.steps, cur.step + (int)(hi - x));
            const int seen_min = dec_seen(cur.q, group, room, cur.chunk * R);
            const int seen_max = cur.seen;
            const bool all_live = (cur.chunk + 1) * R <= cur.q.nq * group;
            // Rows 4 r + t are this thread's in scores and output.
            int seen[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = cur.chunk * R + 4 * r + t;
                seen[r] = row < cur.q.nq * group ? dec_seen(cur.q, group, room, row) : 0;
            }
            // Query columns: this thread holds column g of tile r, the hi (g even)
            // or lo part of row 4 r + g / 2; k-step ks covers 4 neighbouring elements.
            uint32_t qb[NR][KS][2];
            float qf[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = cur.chunk * R + 4 * r + (g >> 1), j = row / group;
                const bool live = j < cur.q.nq;
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
                const float down = a.scale * 1.4426950408889634f * __int_as_float((127 - e) << 23);
                qf[r] = __shfl_sync(0xffffffffu, down, 8 * t);  // of row 4 r + t: column 2 t
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t h0, l0, h1, l1;
                    split_f16(v[4 * ks] * up, v[4 * ks + 1] * up, h0, l0);
                    split_f16(v[4 * ks + 2] * up, v[4 * ks + 3] * up, h1, l1);
                    qb[r][ks][0] = (g & 1) ? l0 : h0;
                    qb[r][ks][1] = (g & 1) ? l1 : h1;
                }
            }
            float o[NR][KS][2];
            float m[NR], l[NR], vref = 0.0f, vinv = 0.0f;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
                for (int i = 0; i < KS; ++i) o[r][i][0] = o[r][i][1] = 0.0f;
            }

            for (; cur.step < last; ++cur.step, ++x) {
                cp_async_wait<S::kStages - 2>();
                __syncwarp();  // the stage's copies of all lanes are there, and the previous stage is read
                issue(stage == 0 ? S::kStages - 1 : stage - 1);
                const uint32_t kb = ring + stage * S::kStageBytes, vb = kb + STEP * D, sb = vb + STEP * D;
                const uint4 sc = lds128(sb);
                uint32_t flags;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(flags) : "r"(sb + 16));
                const float ks0 = (flags & 1) ? __uint_as_float(sc.x) : 0.0f, ks1 = (flags & 2) ? __uint_as_float(sc.y) : 0.0f;
                const float vs0 = (flags & 1) ? __uint_as_float(sc.z) : 0.0f, vs1 = (flags & 2) ? __uint_as_float(sc.w) : 0.0f;
                const int t0 = cur.step * STEP;

                // Scores: 16 tokens (rows g, g + 8) by 4 rows' hi and lo columns.
                float s[MT][NR][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) s[mt][r][0] = s[mt][r][1] = s[mt][r][2] = s[mt][r][3] = 0.0f;
#pragma unroll
                    for (int hf = 0; hf < D / 64; ++hf) {
                        const uint4 wa = lds128(kb + mt * 16 * D + ring_offset<D>(g, hf * 4 + t));
                        const uint4 wb = lds128(kb + (mt * 16 + 8) * D + ring_offset<D>(g, hf * 4 + t));
                        const uint32_t ka[4] = {wa.x, wa.y, wa.z, wa.w}, kc[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t f[4];
                            codes_f16<FMT>(ka[k], f[0], f[2]);
                            codes_f16<FMT>(kc[k], f[1], f[3]);
#pragma unroll
                            for (int r = 0; r < NR; ++r) mma_f16(s[mt][r], f, qb[r][hf * 4 + k][0], qb[r][hf * 4 + k][1]);
                        }
                    }
                }
                // In powers of two; hi and lo meet here.  Token of p[r][i]: 8 i + g.
                float p[NR][2 * MT];
                const bool whole = t0 + STEP <= seen_min && flags == (MT == 2 ? 3 : 1) && all_live;
                bool move = false;
                float top[NR];
#pragma unroll
                for (int r = 0; r < NR; ++r) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const float f = qf[r] * (mt ? ks1 : ks0);
                        p[r][2 * mt] = (s[mt][r][0] + s[mt][r][1]) * f;
                        p[r][2 * mt + 1] = (s[mt][r][2] + s[mt][r][3]) * f;
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 2 * MT; ++i)
                            if (t0 + 8 * i + g >= seen[r] || !(flags & (i < 2 ? 1 : 2))) p[r][i] = -INFINITY;
                    }
                    top[r] = fmaxf(p[r][0], p[r][1]);
                    if (MT == 2) top[r] = fmaxf(top[r], fmaxf(p[r][2 * MT - 2], p[r][2 * MT - 1]));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 4));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 8));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 16));
                    move |= top[r] > m[r] + 1.0f;
                }
                const float vmax = MT == 2 ? fmaxf(vs0, vs1) : vs0;
                if (__any_sync(0xffffffffu, move) || vmax > 4.0f * vref) {
                    float fv = 1.0f;
                    if (vmax > 4.0f * vref) {
                        const float next = fmaxf(vmax, 0x1p-126f);  // whose inverse is finite
                        vinv = 1.0f / next;
                        fv = vref * vinv;
                        vref = next;
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        float f = fv;
                        if (top[r] > m[r] + 1.0f) {
                            const float fm = ex2(m[r] - top[r]);
                            l[r] *= fm;
                            f *= fm;
                            m[r] = top[r];
                        }
#pragma unroll
                        for (int i = 0; i < KS; ++i) o[r][i][0] *= f, o[r][i][1] *= f;
                    }
                }
                const float v0 = vs0 * vinv, v1 = vs1 * vinv;
                // Weights: from (token 8 i + g, row t) to columns of the operand.  A lane's
                // 16 bytes {hi of tokens g, g + 8; hi of g + 16, g + 24; lo of both} lie at
                // place t ^ (g / 2) of line g.
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float bias = m[r] == -INFINITY ? 0.0f : 12.0f - m[r];
#pragma unroll
                    for (int i = 0; i < 2 * MT; ++i) {
                        p[r][i] = ex2(p[r][i] + bias);
                        l[r] += p[r][i];
                        p[r][i] *= i < 2 ? v0 : v1;
                    }
                    uint4 w = make_uint4(0, 0, 0, 0);
                    split_f16(p[r][0], p[r][1], w.x, w.z);
                    if (MT == 2) split_f16(p[r][2 * MT - 2], p[r][2 * MT - 1], w.y, w.w);
                    sts128(weights + r * 512 + (g * 4 + (t ^ (g >> 1))) * 16, w);
                }
                __syncwarp();
                uint2 pb[NR][2];  // k 2t, 2t + 1: tokens 2t, 2t + 8; k 2t + 8, 2t + 9: tokens 2t + 1, 2t + 9
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const uint32_t at = weights + r * 512 + t * 128 + ((g >> 1) ^ t) * 16 + (g & 1) * 8;
                    pb[r][0] = lds64(at);
                    pb[r][1] = lds64(at + 64);
                }
                // Values: elements g E .. g E + E - 1 of tokens 2t, 2t + 8, 2t + 1, 2t + 9 of each 16.
                const bool clean = FMT == kKv8I8 || (t0 + STEP <= seen_max && flags == (MT == 2 ? 3 : 1));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint32_t w[4][D / 32];  // token, word
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int r = 2 * t + (b >> 1), r8 = (b & 1) * 8;
                        const uint32_t at = vb + (mt * 16 + r8) * D;
                        if (D == 64) {
                            const uint2 u = lds64(at + ring_offset<D>(r, g >> 1) + (g & 1) * 8);
                            w[b][0] = u.x, w[b][1] = u.y;
                        } else {
                            const uint4 u = lds128(at + ring_offset<D>(r, g));
                            w[b][0] = u.x, w[b][1] = u.y, w[b][D / 32 - 2] = u.z, w[b][D / 32 - 1] = u.w;
                        }
                        if (!clean) {  // what lies behind the end may be NaN
                            const int tok = t0 + mt * 16 + r8 + r;
                            if (tok >= seen_max || !(flags & (mt ? 2 : 1)))
#pragma unroll
                                for (int e = 0; e < D / 32; ++e) w[b][e] = 0;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) {
                        // bytes of two tokens side by side; tile 2 e + i: elements 4 e + 2 i and + 1
                        uint32_t f[2][4];
                        codes_f16<FMT>(__byte_perm(w[0][e], w[1][e], 0x5140), f[0][0], f[0][1]);
                        codes_f16<FMT>(__byte_perm(w[0][e], w[1][e], 0x7362), f[1][0], f[1][1]);
                        codes_f16<FMT>(__byte_perm(w[2][e], w[3][e], 0x5140), f[0][2], f[0][3]);
                        codes_f16<FMT>(__byte_perm(w[2][e], w[3][e], 0x7362), f[1][2], f[1][3]);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int r = 0; r < NR; ++r) {
                                float z[4];
                                mma_f16_zero(z, f[i], mt ? pb[r][0].y : pb[r][0].x, mt ? pb[r][1].y : pb[r][1].x);
                                o[r][2 * e + i][0] += z[0] + z[1];  // hi and lo meet here
                                o[r][2 * e + i][1] += z[2] + z[3];
                            }
                    }
                }
                stage = stage == S::kStages - 1 ? 0 : stage + 1;
            }
            // ---- the segment's end ----
            const bool whole_unit = first_step == 0 && last == cur.steps;
            x_end = x;
            if (cur.step == cur.steps) x += kDecUnitCost;
            // The warp's last segment: its ring is read out and takes the piece.
            // An earlier one (the end of a unit begun before): global memory.
            float* part = warp_parts + (size_t)(w0 + warp) * S::kPartFloats;
            if (!whole_unit && x >= hi) {
                cp_async_wait<0>();
                __syncwarp();
                part = ring_part(warp);
            }
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 4);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 8);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 16);
                if (whole_unit) {
                    T* dst = out_row(cur, 4 * r + t);
                    if (!dst) continue;
                    dst += g * E;
                    const float f = l[r] == 0.0f ? 0.0f : 1.0f / l[r];  // vref / l could be too small a number
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        dst[i] = (T)(l[r] == 0.0f ? 0.0f : o[r][i >> 1][i & 1] * f * vref);
                } else {
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        part[(4 * r + t) * D + g * E + i] = o[r][i >> 1][i & 1] * vref;
                    if (g == 0) {
                        part[R * D + 4 * r + t] = m[r];
                        part[R * D + R + 4 * r + t] = l[r];
                    }
                }
            }
            if (cur.step == cur.steps && x < hi) next_unit(cur);
        }
    }
    __syncthreads();

    // ---- joining pieces ----
    // Adds n pieces (piece(i) is the i-th) by one warp, two at a time so that
    // their loads are under way together: lane's four neighbouring elements of
    // rows (lane * 4 + 128 k) / D.
    constexpr int KM = R * D / 128;
    struct Sum {
        float m[KM], l[KM];
        float4 o[KM];
    };
    auto clear = [&](Sum& z) {
#pragma unroll
        for (int k = 0; k < KM; ++k) z.m[k] = -INFINITY, z.l[k] = 0.0f, z.o[k] = make_float4(0, 0, 0, 0);
    };
    auto add = [&](Sum& z, int n, auto piece) {
        for (int i0 = 0; i0 < n; i0 += 2) {
            float pm[2][KM], pl[2][KM];
            float4 po[2][KM];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i0 + i >= n) continue;
                const float* p = piece(i0 + i);
#pragma unroll
                for (int k = 0; k < KM; ++k) {
                    const int e = lane * 4 + 128 * k, r = e / D;
                    pm[i][k] = p[R * D + r];
                    pl[i][k] = p[R * D + R + r];
                    po[i][k] = *reinterpret_cast<const float4*>(p + e);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i0 + i >= n) continue;
#pragma unroll
                for (int k = 0; k < KM; ++k) {
                    const float m = fmaxf(z.m[k], pm[i][k]);
                    const float f = z.m[k] == -INFINITY ? 0.0f : ex2(z.m[k] - m), h = pm[i][k] == -INFINITY ? 0.0f : ex2(pm[i][k] - m);
                    z.m[k] = m;
                    z.l[k] = z.l[k] * f + pl[i][k] * h;
                    z.o[k].x = z.o[k].x * f + po[i][k].x * h, z.o[k].y = z.o[k].y * f + po[i][k].y * h;
                    z.o[k].z = z.o[k].z * f + po[i][k].z * h, z.o[k].w = z.o[k].w * f + po[i][k].w * h;
                }
            }
        }
    };
    auto store = [&](const Sum& z, float* to) {
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            const int e = lane * 4 + 128 * k, r = e / D;
            *reinterpret_cast<float4*>(to + e) = z.o[k];
            if (e % D == 0) to[R * D + r] = z.m[k], to[R * D + R + r] = z.l[k];
        }
    };
    auto finish = [&](const Sum& z, const DecCursor& u) {
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            const int e = lane * 4 + 128 * k;
            T* dst = out_row(u, e / D);
            if (!dst) continue;
            dst += e % D;
            const float inv = z.l[k] == 0.0f ? 0.0f : 1.0f / z.l[k];
            dst[0] = (T)(z.o[k].x * inv), dst[1] = (T)(z.o[k].y * inv);
            dst[2] = (T)(z.o[k].z * inv), dst[3] = (T)(z.o[k].w * inv);
        }
    };
    // A warp joins the pieces of the unit that begins in it and goes on, and
    // warp 0 those of the unit that was under way at the CTA's start.
    for (int side = warp == 0 ? 0 : 1; side < 2 && lo < hi; ++side) {
        const DecCursor u = side == 0 ? first_unit : cur;
        // The unit's place on the line: `cur` stands behind the warp's last step.
        const unsigned u0 = side == 0 ? lo - u.step : x_end - u.step, u1 = u0 + u.steps;
        if (side == 0 ? u0 >= lo : !(u0 >= lo && u1 > hi)) continue;
        const int wn = (int)(worker_of(min(u1, cta_hi) - 1) - (w0 + warp)) + 1;  // warps with a piece, from this one
        Sum z;
        clear(z);
        // All but the last lie in the ring; so does the last unless that warp went on to another unit.
        const bool tail_out = begin_of(w0 + warp + wn) > u1 + kDecUnitCost;
        add(z, wn, [&](int i) -> const float* {
            return i == wn - 1 && tail_out ? warp_parts + (size_t)(w0 + warp + i) * S::kPartFloats : ring_part(warp + i);
        });
        if (u0 >= cta_lo && u1 <= cta_hi) {
            finish(z, u);
            continue;
        }
        store(z, cta_parts + ((size_t)blockIdx.x * 2 + side) * S::kPartFloats);
        const int first = (int)(worker_of(u0) / kDecWarps), final = (int)(worker_of(u1 - 1) / kDecWarps);
        __threadfence();
        __syncwarp();
        if (lane == 0 && atomicAdd(counters + first, 1) == final - first) {
            counters[first] = 0;
            __threadfence();
            done_unit[side] = 1 + first;
            done_cursor[side] = u;
            done_pieces[side] = final - first + 1;
        }
    }
    __syncthreads();
    // The pieces of a unit that spans CTAs, by all warps of the last CTA to
    // finish: each a range of them, then one adds the warps' sums in order.
    for (int side = 0; side < 2; ++side) {
        if (!done_unit[side]) continue;  // uniform over the CTA
        const DecCursor u = done_cursor[side];
        const int first = done_unit[side] - 1, n = done_pieces[side];
        const int i0 = n * warp / kDecWarps, i1 = n * (warp + 1) / kDecWarps;
        Sum z;
        clear(z);
        add(z, i1 - i0, [&](int i) -> const float* {
            return cta_parts + ((size_t)(first + i0 + i) * 2 + (i0 + i == 0 ? 1 : 0)) * S::kPartFloats;
        });
        __syncthreads();  // the ring's pieces are read
        store(z, ring_part(warp));
        __syncthreads();
        if (warp == 0) {
            clear(z);
            add(z, kDecWarps, [&](int i) -> const float* { return ring_part(i); });
            finish(z, u);
        }
        __syncthreads();
    }
}

template <typename T, int FMT, int D, int NR>
cudaError_t kv8_decode_prepare() {
    return cudaFuncSetAttribute(kv8_decode_kernel<T, FMT, D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                DecShape<D, NR>::kRingBytes + (kPagesMaxSeqs + 1) * (int)sizeof(unsigned));
}

template <typename T, int FMT, int D, int NR>
cudaError_t launch_kv8_decode(const Kv8& c, const Kv8Attention& a, int num_sms, void* ws, cudaStream_t st) {
    using S = DecShape<D, NR>;
    const int smem = S::kRingBytes + (a.n_seqs + 1) * (int)sizeof(unsigned);
    int* counters = (int*)ws;
    float* parts = (float*)((uint8_t*)ws + kv8_counter_bytes(num_sms));
    return launch_ex(kv8_decode_kernel<T, FMT, D, NR>, dim3(num_sms * S::kCtasPerSm), dim3(kDecWarps * 32), smem, st, true,
                     c, a, parts, counters);
}

}  // namespace lc
