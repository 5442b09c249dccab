// lc_kv8_prefill.cuh -- attention over the 8-bit pages for many queries per
// sequence (prompt chunks), on the tcgen05 tensor cores.
//
// A unit is 256 (query, head) rows that share a kv head, as two tiles of 128
// MMA rows; a step is NT = 64 tokens.  Per step and row tile
//   S = Q K^T   M 128, N NT, K head size: Q and K codes f16 in shared memory
//   p = 2^(S c + b), running maximum and sum, one thread per row
//   O += P V    M 128, N head size, K NT: P in tensor memory over S's columns
// The codes are exact in f16, so scales enter only where scores leave tensor
// memory: the key scale of a 16-token group in c, the value scale (over a
// running reference, as its logarithm) in b; the sum takes it out again.
// fp32 rows are split into f16 hi + lo under a power-of-two row scale (22 bits),
// at the price of twice the products; f16 rows are exact.  P is split the same
// way for both: rounded to one f16 it is off by 2^-12 of each weight, which adds
// as much error as the rounding of an f16 result itself (1.4 times its norm in
// all; six chunks of f16 rows over 500 to 4000 positions 133 against 145 us with
// the split).
//
// The tensor cores' fp32 sums lose up to one unit of the last place, always
// toward zero, at every product that is added; over thousands of tokens that
// drifts (4.8e-6 of the result at 4096 tokens, against 1e-6 of fp32 sums), so
// after kFlush steps O is added to a second accumulator in round-to-nearest
// and begun anew: in tensor memory where there is room (head size 64), in the
// CTA's piece in L2 otherwise.
//
// What bounds it: for head size 64 one exponential costs as much as the 128
// products of its score, so the softmax, not the tensor cores, sets the pace
// (4096 fp32 queries, 32 heads: 249 us, of which the products need 81; with the
// softmax's arithmetic left out it is 207: the rest is the steps' chain of
// barriers and loads).
// Hence two row tiles per CTA, one dequantised tile for both, and loops over
// 32 columns that are kept loops: unrolled over the step, their code no longer
// fits the schedulers' instruction caches (297 against 263 us).
//
// Warps 0-3 and 4-7: softmax of row tiles 0 and 1.  Warps 8-11: codes to f16
// operands.  Warps 12 and 13: issue the MMAs of a row tile each.  Warps 14 and 15:
// queries to f16 operands, while the unit before is under way (as a part of the
// operand warps' work: head size 128 420 against 397 us, head size 64 the same).
// Registers move from the MMA warps' group to the softmax.  All steps of the call
// form one line that is cut into equal pieces, one per CTA; pieces of a unit are
// joined, warp by warp, by the last CTA to finish, in the order of the line.
#pragma once

#include "lc_internal.h"
#include "lc_kv8_decode.cuh"
#include "lc_tcgen05.cuh"

namespace lc {

constexpr int kPreRows = 256;      // rows of a unit
constexpr int kPreThreads = 16 * 32;
constexpr int kPreTok = 64;        // tokens of a step
constexpr int kPreUnitCost = 3;    // a unit's beginning and end, in steps
constexpr float kPreNoScale = -160.0f;  // log2 of a value scale of zero: below those of all numbers
constexpr int kPreScaleRing = 8;   // more steps than the operand warps can be ahead of the softmax

template <typename T, int D>
struct PreShape {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kGroups = kPreTok / 16;
    static constexpr int kStages = D == 64 ? 4 : 2;        // operand tiles of K, and of V
    static constexpr int kQBufs = kSplit && D == 128 ? 1 : 2;  // units whose queries are held
    static constexpr int kQPart = 128 * D * 2;            // bytes of one part (hi or lo) of one row tile
    static constexpr int kQBytes = 2 * (kSplit ? 2 : 1) * kQPart;
    static constexpr int kTileBytes = kPreTok * D * 2;
    static constexpr int kScaleBytes = kPreScaleRing * (kGroups * 8 + 8);
    static constexpr int kSmem = kQBufs * (kQBytes + kPreRows * 4) + 2 * kStages * kTileBytes + kScaleBytes;
    static constexpr int kPieceFloats = kPreRows * (D + 2);
    // Registers of the softmax, operand and MMA warpgroups after the split; their
    // sum over 128 threads each must not pass the launch's (checked on the host).
    // With 168, 120 and 56 the compiler spills more (4096 fp32 queries, 32 heads:
    // 269 against 255 us; f16 of head size 128, twice the codes: 310 against 280);
    // with these, fp32 of head size 128 alone (144 bytes stored, 340 loaded).
    static constexpr int kRegsSoftmax = 144, kRegsOperand = 128, kRegsMma = 96;
    static constexpr int kRegsLaunch = (2 * kRegsSoftmax + kRegsOperand + kRegsMma + 3) / 4;
    // Tensor memory: two buffers of S for each tile, so that the next step's
    // scores are there when a step's weights are done; O of both tiles;
    // and for head size 64 the second accumulators.
    static constexpr uint32_t kOCol = 4 * kPreTok, kSumCol = kOCol + 2 * D;
    static constexpr bool kSumInTmem = D == 64;
    // Steps between additions to it: 256 tokens (D 64) or 512 in fp32; 2048 in f16,
    // whose 256 products lose 1e-5, a fortieth of the result's own rounding (after
    // 1024 tokens 146.6 us instead of 145.5 for the chunks above, after 8192 145.0).
    static constexpr int kFlush = kSplit ? (D == 64 ? 4 : 8) : 32;
};

inline size_t kv8_prefill_counter_bytes(int num_sms) { return ((size_t)num_sms * 8 * sizeof(int) + 255) / 256 * 256; }
inline size_t kv8_prefill_ws_bytes(int num_sms) {
    return kv8_prefill_counter_bytes(num_sms) + (size_t)num_sms * 2 * PreShape<float, 128>::kPieceFloats * sizeof(float);
}

LC_DEV void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One thread of a converged warp.  The compiler then keeps the operands of the
// instructions behind it in uniform registers: products issued by "lane == 0"
// took 48 to 200 cycles each, by the elected thread the tensor cores' own 32
// (128 x 64 x 16) or 64 (128 x 128 x 16).
LC_DEV bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}

LC_DEV void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
// The loads before it are done; the values pass through, so that no use moves up.
LC_DEV void tmem_wait_ld32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                   "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                   "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
LC_DEV void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
LC_DEV void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
LC_DEV void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
// Two fp32 values in one register pair, and the instructions that take them.
LC_DEV uint64_t pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
LC_DEV float2 unpair(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
LC_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
LC_DEV uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

LC_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A unit of the line and the step within it.
struct PreCursor {
    SeqInfo q;
    int s, head, chunk, chunks;
    int seen;         // positions that its last row sees
    int step, steps;
};

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kPreThreads, 1)
kv8_prefill_kernel(Kv8 c, Kv8Attention a, float* __restrict__ pieces, int* __restrict__ counters, int* err, uint64_t timeout_ns) {
    using S = PreShape<T, D>;
    constexpr int NT = kPreTok, G = S::kGroups, NS = S::kStages;
    constexpr bool SPLIT = S::kSplit;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int NQ = S::kQBufs;
    uint8_t* const sq = smem;                                   // [buffers][tile][part]
    uint8_t* const sk = sq + NQ * S::kQBytes;                   // [stages]
    uint8_t* const sv = sk + NS * S::kTileBytes;                // [stages]
    float2* const scales = reinterpret_cast<float2*>(sv + NS * S::kTileBytes);  // [ring][group]: key scale, log2 of the value scale
    unsigned* const valid = reinterpret_cast<unsigned*>(scales + kPreScaleRing * G);  // [ring][2]
    float* const qscale = reinterpret_cast<float*>(valid + kPreScaleRing * 2);         // [buffers][rows] score factor of each row
    unsigned* const prefix = reinterpret_cast<unsigned*>(qscale + NQ * kPreRows);      // [n_seqs + 1]
    __shared__ __align__(8) uint64_t k_full[NS], v_full[NS], k_empty[NS], v_empty[NS], s_full[4], p_ready[4], pv_done[2], q_full[NQ], q_seen[NQ],
        sc_full[kPreScaleRing], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int unset;  // an error word of its own for the drain, which waits also after a failure
    __shared__ unsigned long long scan[kPreThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.n_heads / c.n_kv, sh = c.page_shift;
    const int room = (int)min((long long)a.table_stride << sh, 0x7fffffffll);

    if (tid == 0) {
        unset = 0;
        for (int i = 0; i < NS; ++i) {
            mbar_init(&k_full[i], 4), mbar_init(&v_full[i], 4);
            mbar_init(&k_empty[i], 2), mbar_init(&v_empty[i], 2);  // both MMA warps
        }
        for (int i = 0; i < 4; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_ready[i], 4);  // [tile][buffer]
        mbar_init(&pv_done[0], 1), mbar_init(&pv_done[1], 1);
        for (int i = 0; i < kPreScaleRing; ++i) mbar_init(&sc_full[i], 1);
        for (int i = 0; i < NQ; ++i) mbar_init(&q_full[i], 6), mbar_init(&q_seen[i], 10);  // by operand and query warps; softmax and MMA warps
        mbar_init(&drained, 2);
        fence_mbar_init();
    }
    griddep_wait();

    auto seen_of = [&](const SeqInfo& q, int row) { return dec_seen(q, group, room, row); };
    auto steps_of = [&](const SeqInfo& q, int chunk) { return dec_steps<NT>(seen_of(q, chunk * kPreRows + kPreRows - 1)); };
    auto chunks_of = [&](const SeqInfo& q) { return (int)(((int64_t)q.nq * group + kPreRows - 1) / kPreRows); };

    // ---- the line of steps: a warp per sequence, lanes over its chunks ----
    for (int s = warp; s < a.n_seqs; s += kPreThreads / 32) {
        const SeqInfo q = kv8_seq(a, sh, s);
        const int chunks = chunks_of(q);
        unsigned long long cost = 0;
        for (int k = lane; k < chunks; k += 32) cost += steps_of(q, k) + kPreUnitCost;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
        cost *= c.n_kv;
        if (lane == 0) prefix[s] = cost > 0xffffffffull ? 0xffffffffu : (unsigned)cost;
    }
    __syncthreads();
    unsigned long long carry = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += kPreThreads) {
        const int s = s0 + tid;
        const unsigned cost = s < a.n_seqs ? prefix[s] : 0;
        unsigned long long v = cost;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        unsigned long long before = carry, all = carry;
        for (int w = 0; w < kPreThreads / 32; ++w) {
            if (w < warp) before += scan[w];
            all += scan[w];
        }
        if (s < a.n_seqs) prefix[s] = (unsigned)(before + v - cost);
        carry = all;
        __syncthreads();
    }
    if (carry > 0xffffffffull) return;  // the host has checked it for ascending q_start
    if (tid == 0) prefix[a.n_seqs] = (unsigned)carry;
    // CTA b has steps [begin_of(b), begin_of(b + 1)).
    const unsigned total = (unsigned)carry;
    const unsigned workers = min(gridDim.x, total);
    if (blockIdx.x >= workers) return;  // also where there is nothing at all
    if (warp == 12) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_launch();  // here: the next kernel may ask for tensor memory before it waits for this one
    const uint32_t tmem = tmem_slot;
    const unsigned share = total / workers, extra = total - share * workers;
    auto begin_of = [&](unsigned w) { return w * share + min(w, extra); };
    auto worker_of = [&](unsigned x) {
        const unsigned big = extra * (share + 1);
        return x < big ? x / (share + 1) : extra + (x - big) / share;
    };
    const unsigned hi = begin_of(blockIdx.x + 1);
    unsigned lo = begin_of(blockIdx.x);

    auto set_chunk = [&](PreCursor& cur, int chunk) {
        cur.chunk = chunk;
        cur.seen = seen_of(cur.q, chunk * kPreRows + kPreRows - 1);
        cur.steps = dec_steps<NT>(cur.seen);
    };
    auto set_seq = [&](PreCursor& cur, int s) {
        cur.s = s;
        cur.q = kv8_seq(a, sh, s);
        cur.chunks = chunks_of(cur.q);
    };
    auto next_unit = [&](PreCursor& cur) {
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
        set_chunk(cur, 0);
    };
    // The unit and step at place x; by whole warps.
    PreCursor cur;
    {
        int a0 = 0, a1 = a.n_seqs;
        while (a1 - a0 > 1) {
            const int mid = (a0 + a1) >> 1;
            if (prefix[mid] <= lo) a0 = mid;
            else a1 = mid;
        }
        set_seq(cur, a0);
        unsigned rem = lo - prefix[a0];
        const unsigned per = (prefix[a0 + 1] - prefix[a0]) / c.n_kv;
        cur.head = rem / per;
        rem -= cur.head * per;
        for (int k0 = 0;; k0 += 32) {
            const unsigned cost = k0 + lane < cur.chunks ? steps_of(cur.q, k0 + lane) + kPreUnitCost : 0;
            unsigned v = cost;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            const unsigned over = __ballot_sync(0xffffffffu, v > rem);
            if (over || k0 + 32 >= cur.chunks) {
                const int l = over ? __ffs(over) - 1 : 31;
                rem -= __shfl_sync(0xffffffffu, v - cost, l);
                set_chunk(cur, k0 + l);
                break;
            }
            rem -= __shfl_sync(0xffffffffu, v, 31);
        }
        cur.step = rem;
        if (cur.step >= cur.steps) {  // the empty places behind a unit
            lo = min(hi, lo + cur.steps + kPreUnitCost - cur.step);
            if (lo < hi) next_unit(cur);
        }
    }
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        // Whole warps wait; they go on together, as the tensor-memory instructions ask.
        // The limit is each wait's own: a call of long prompts may take seconds.
        return (bool)__all_sync(0xffffffffu, mbar_try_wait(bar, parity) ||
                                                 mbar_wait_bounded(bar, parity, err, globaltimer_ns() + timeout_ns, kDevTimeoutGrid));
    };
    auto tiles_of = [&](const PreCursor& u) { return (int64_t)u.q.nq * group - (int64_t)u.chunk * kPreRows > 128 ? 2 : 1; };
    // The unit's rows, each scaled so that its largest element lies in
    // [2^9, 2^10), as f16 hi (and lo).
    const bool q16 = ((uintptr_t)a.q | (uintptr_t)(a.q_stride * sizeof(T))) % 16 == 0;
    auto query = [&](const PreCursor& u, int r) -> const T* {  // row r of the unit; null behind its last
        const int row = u.chunk * kPreRows + r, j = row / group;
        if (j >= u.q.nq) return nullptr;
        return (const T*)a.q + (int64_t)(u.q.row0 + j) * a.q_stride + (int64_t)(u.head * group + row - j * group) * D;
    };
    auto prefetch_queries = [&](PreCursor u, int part, int parts) {  // of the next unit, to L2
        next_unit(u);
        const int rows = tiles_of(u) * 128;
        for (int r = part * 32 + lane; r < rows; r += parts * 32) {
            const T* q = query(u, r);
            if (!q) break;
#pragma unroll
            for (int o = 0; o < D * (int)sizeof(T); o += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"((const uint8_t*)q + o));
        }
    };
    auto put_queries = [&](const PreCursor& u, int buf, int part, int parts) {  // by warp `part` of `parts`
        const int rows = tiles_of(u) * 128;
        constexpr int TPR = D / 32;                // threads of a row, 32 elements each
        constexpr int V = 16 / sizeof(T), N = 32 / V;  // elements of 16 bytes, loads of a thread
#pragma unroll 1
        for (int r = part * (32 / TPR) + lane / TPR; r < rows; r += parts * (32 / TPR)) {
            const int e0 = (lane % TPR) * 32;
            const T* q = query(u, r);
            uint4 w[N];
#pragma unroll
            for (int b = 0; b < N; ++b) {
                w[b] = make_uint4(0, 0, 0, 0);
                if (q && q16) {
                    w[b] = __ldg(reinterpret_cast<const uint4*>(q + e0 + b * V));
                } else if (q) {
                    T* e = reinterpret_cast<T*>(&w[b]);
#pragma unroll
                    for (int i = 0; i < V; ++i) e[i] = q[e0 + b * V + i];
                }
            }
            const T* e = reinterpret_cast<const T*>(w);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf((float)e[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            if (TPR == 4) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int ex = top > 0.0f ? 9 - (((__float_as_int(top) >> 23) & 0xff) - 127) : 0;
            ex = max(-126, min(126, ex));
            const float up = pow2f(ex);
            if (e0 == 0) qscale[buf * kPreRows + r] = a.scale * 1.4426950408889634f * pow2f(-ex);
            const uint32_t at = smem_u32(sq) + buf * S::kQBytes + (r >> 7) * (SPLIT ? 2 : 1) * S::kQPart +
                                ((r & 127) >> 3) * (D * 16) + (r & 7) * 16 + (e0 >> 3) * 128;
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (float)e[o * 8 + i] * up;
                uint4 h, l;
                split_octet(v, h, l);
                sts128(at + o * 128, h);
                if (SPLIT) sts128(at + S::kQPart + o * 128, l);
            }
        }
        fence_async_shared();
        __syncwarp();
    };
    bool ok = true;

    if (warp >= 8 && warp < 12) {
        // ---- operands to f16 ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRegsOperand));
        const int cw = warp - 8;
        constexpr int CH = NT * D / 16 / 128;  // 16-code chunks per thread, for K and for V
        // What a step needs from memory.  The next step's keys are asked for as soon as
        // this one's are written as operands, then its values: each has a step's time.
        uint4 wk[CH], wv[CH];
        float ks = 0.0f, vs = 0.0f;  // scales of 16-token group `lane`, in the first warp
        bool there = false;
        int id[CH], group_id = -1;
        auto token_of = [&](int k) {  // of this thread's k-th chunk
            const int i = k * 4 + cw;
            return (D == 64 ? i : i >> 1) * 8 + (lane & 7);
        };
        auto chunk_of = [&](int k) { return (D == 64 ? 0 : ((k * 4 + cw) & 1) * 4) + (lane >> 3); };
        auto load_ids = [&](const PreCursor& u) {
            const int32_t* row = a.table + (int64_t)u.s * a.table_stride;
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int t = u.step * NT + token_of(k);
                id[k] = t < u.seen ? row[t >> sh] : -1;
            }
            if (cw == 0 && lane < G) {
                const int t = u.step * NT + lane * 16;
                group_id = t < u.seen ? row[t >> sh] : -1;
            }
        };
        auto load_codes = [&](const PreCursor& u, const uint8_t* from, uint4 (&w)[CH]) {
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int t = u.step * NT + token_of(k);
                w[k] = make_uint4(0, 0, 0, 0);  // tokens that nobody sees stay zero: there may be NaN codes
                if ((unsigned)id[k] < (unsigned)c.n_pages)
                    w[k] = __ldg(reinterpret_cast<const uint4*>(
                        from + ((((int64_t)id[k] * c.n_kv + u.head) << sh) + (t & ((1 << sh) - 1))) * D + chunk_of(k) * 16));
            }
        };
        auto load_scales = [&](const PreCursor& u) {
            if (cw == 0 && lane < G) {
                there = (unsigned)group_id < (unsigned)c.n_pages;
                ks = there ? c.k_scale[(int64_t)group_id * c.n_kv + u.head] : 0.0f;
                vs = there ? c.v_scale[(int64_t)group_id * c.n_kv + u.head] : 0.0f;
            }
        };
        auto put = [&](uint8_t* tile, const uint4 (&w)[CH]) {
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                uint32_t f[8];
                codes_f16<FMT>(w[k].x, f[0], f[1]);
                codes_f16<FMT>(w[k].y, f[2], f[3]);
                codes_f16<FMT>(w[k].z, f[4], f[5]);
                codes_f16<FMT>(w[k].w, f[6], f[7]);
                const uint32_t at = smem_u32(tile) + (token_of(k) >> 3) * (D * 16) + chunk_of(k) * 256 + (lane & 7) * 16;
                sts128(at, make_uint4(f[0], f[1], f[2], f[3]));
                sts128(at + 128, make_uint4(f[4], f[5], f[6], f[7]));
            }
        };
        // `nx` is the next step to load, its pages' numbers under way; `cur` the
        // one whose tiles are written.
        PreCursor nx = cur;
        unsigned ahead = lo, x = lo;
        auto load_keys = [&]() {
            if (ahead >= hi) return;
            load_codes(nx, c.k, wk);
            load_scales(nx);
        };
        auto load_values = [&]() {
            if (ahead >= hi) return;
            load_codes(nx, c.v, wv);
            ++ahead;
            if (++nx.step == nx.steps) {
                ahead += kPreUnitCost;
                if (ahead < hi) next_unit(nx);
            }
            if (ahead < hi) load_ids(nx);
        };
        if (x < hi) load_ids(nx);
        load_keys();
        load_values();
        int i = 0, units = 0;
#pragma unroll 1
        while (x < hi && ok) {
            if (i == 0 || cur.step == 0) {
                // A unit is also announced here, behind all steps before it: a softmax
                // group that had no rows in the unit before has not followed them.
                const int buf = units % NQ;
                if (units >= NQ) ok = wait(&q_seen[buf], (units / NQ - 1) & 1);
                if (!ok) break;
                if (NQ == 1 || units == 0) put_queries(cur, buf, cw, 6);
                if (lane == 0) mbar_arrive(&q_full[buf]);
                ++units;
            }
            const int st = i % NS, use = i / NS;
            if (use > 0) ok = wait(&k_empty[st], (use - 1) & 1);
            if (!ok) break;
            put(sk + st * S::kTileBytes, wk);
            if (cw == 0) {
                const int ring = i % kPreScaleRing;
                if (lane < G) scales[ring * G + lane] = make_float2(ks, vs <= 0.0f ? kPreNoScale : log2f(vs));  // NaN stays
                const unsigned m = __ballot_sync(0xffffffffu, lane < G && there);
                if (lane == 0) valid[ring * 2] = m;
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&k_full[st]);
                if (cw == 0) mbar_arrive(&sc_full[i % kPreScaleRing]);
            }
            load_keys();
            if (use > 0) ok = wait(&v_empty[st], (use - 1) & 1);
            if (!ok) break;
            put(sv + st * S::kTileBytes, wv);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[st]);
            load_values();
            ++i;
            ++x;
            if (++cur.step == cur.steps) {
                x += kPreUnitCost;
                if (x < hi) next_unit(cur);
            }
        }
    } else if (warp >= 12) {
        // ---- MMAs: a warp per row tile, one thread of it issues ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRegsMma));
        if (warp < 14) {
            const int tile = warp - 12;
            constexpr uint32_t id_qk = tc_idesc_f16_f32(128, NT);
            constexpr uint32_t id_pv = tc_idesc_f16_f32(128, D) | (1u << 16);  // B (values) with the head's elements contiguous
            constexpr int PARTS = SPLIT ? 2 : 1;
            const uint64_t qd0 = tc_desc_kmajor(smem_u32(sq + tile * PARTS * S::kQPart), 128, D * 16);
            uint64_t qd = qd0;
            const uint64_t kd0 = tc_desc_kmajor(smem_u32(sk), 128, D * 16);
            // Values: 8-token groups D * 16 bytes apart, 8-element groups 128 bytes.
            const uint64_t vd0 = tc_desc_kmajor(smem_u32(sv), D * 16, 128);
            const uint32_t sbuf = tmem + tile * 2 * NT, obuf = tmem + S::kOCol + tile * D;
            int i0 = 0, np = 0, units = 0;  // steps before this unit, those of this tile, units
            for (unsigned x = lo; x < hi && ok;) {
                const int n = min(cur.steps - cur.step, (int)(hi - x));
                const bool live = tile < tiles_of(cur);
                const int buf = units % NQ;
                // Scores of step k: its buffer's weights, two steps back, have been read.
                auto scores = [&](int k) {
                    const int st = (i0 + k) % NS;
                    ok = wait(&k_full[st], ((i0 + k) / NS) & 1);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t d = sbuf + ((np + k) & 1) * NT;
                    const uint64_t kd = kd0 + st * (S::kTileBytes / 16);
                    if (elect_one()) {
                        if (live) {
#pragma unroll
                            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                                for (int e = 0; e < D / 16; ++e)
                                    tc_mma_f16(d, qd + part * (S::kQPart / 16) + e * 16, kd + e * 16, id_qk, part + e > 0);
                            tc_commit(&s_full[tile * 2 + ((np + k) & 1)]);
                            tc_commit(&k_empty[st]);
                            if (k == n - 1) tc_commit(&q_seen[buf]);
                        } else {
                            mbar_arrive(&k_empty[st]);
                            if (k == n - 1) mbar_arrive(&q_seen[buf]);
                        }
                    }
                    __syncwarp();
                };
                ok = wait(&q_full[buf], (units++ / NQ) & 1);
                qd = qd0 + buf * (S::kQBytes / 16);
                for (int k = 0; k < 2 && k < n && ok; ++k) scores(k);
                for (int k = 0; k < n && ok; ++k) {
                    const int st = (i0 + k) % NS, b = np + k;
                    ok = wait(&v_full[st], ((i0 + k) / NS) & 1);
                    if (ok && live) ok = wait(&p_ready[tile * 2 + (b & 1)], (b >> 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t p = sbuf + (b & 1) * NT;
                    const uint64_t vd = vd0 + st * (S::kTileBytes / 16);
                    const uint32_t more = k % S::kFlush != 0;
                    if (elect_one()) {
                        if (live) {
#pragma unroll
                            for (int e = 0; e < NT / 16; ++e) {
                                const uint32_t ac = p + e * 16;
                                tc_mma_f16_ta(obuf, ac, vd + e * (2 * D), id_pv, e > 0 ? 1 : more);
                                tc_mma_f16_ta(obuf, ac + 8, vd + e * (2 * D), id_pv, 1);
                            }
                            tc_commit(&pv_done[tile]);
                            tc_commit(&v_empty[st]);
                        } else {
                            mbar_arrive(&v_empty[st]);
                        }
                    }
                    __syncwarp();
                    if (live) ok = wait(&pv_done[tile], b & 1);
                    if (ok && k + 2 < n) scores(k + 2);
                }
                if (live) np += n;
                i0 += n;
                x += n;
                cur.step += n;
                if (cur.step == cur.steps) {
                    x += kPreUnitCost;
                    if (x < hi) next_unit(cur);
                }
            }
        } else {
            // ---- queries to f16 operands, a unit's while the unit before is under way ----
            int units = 0;
            for (unsigned x = lo; x < hi && ok; ++units) {
                const int n = min(cur.steps - cur.step, (int)(hi - x)), buf = units % NQ;
                // The buffer's last unit: its scores are computed, its factors read.
                if (units >= NQ) ok = wait(&q_seen[buf], (units / NQ - 1) & 1);
                if (!ok) break;
                // The first unit's, and all where there is one buffer, with the operand warps.
                const bool alone = NQ == 2 && units > 0;
                put_queries(cur, buf, alone ? warp - 14 : warp - 10, alone ? 2 : 6);
                if (lane == 0) mbar_arrive(&q_full[buf]);
                x += n;
                cur.step += n;
                if (cur.step == cur.steps) {
                    x += kPreUnitCost;
                    if (x < hi) {
                        prefetch_queries(cur, warp - 14, 2);
                        next_unit(cur);
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: one thread per row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kRegsSoftmax));
        const int tile = warp >> 2, r = tid & 127;  // row of the tile, its TMEM lane
        const uint32_t lane_base = (uint32_t)(warp & 3) << 21;  // lanes 32 (warp % 4)
        const uint32_t to = tmem + lane_base + S::kOCol + tile * D;
        const uint32_t tsum = tmem + lane_base + S::kSumCol + tile * D;
        int i = 0, np = 0, units = 0;
        const bool o16 = ((uintptr_t)a.out | (uintptr_t)(a.out_stride * sizeof(T))) % 16 == 0;
        for (unsigned x = lo; x < hi && ok;) {
            const int n = min(cur.steps - cur.step, (int)(hi - x));
            const int tiles = tiles_of(cur);
            const int row = cur.chunk * kPreRows + tile * 128 + r, j = row / group;
            const bool live = j < cur.q.nq;
            const int seen = live ? seen_of(cur.q, row) : 0;
            const int64_t col = (int64_t)(cur.head * group + (live ? row - j * group : 0)) * D;
            // The tile's first row sees least: below that nothing is masked.
            const int seen_min = cur.chunk * kPreRows + tile * 128 + 127 < cur.q.nq * group
                                     ? seen_of(cur.q, cur.chunk * kPreRows + tile * 128) : 0;
            const int buf = units % NQ;
            ok = wait(&q_full[buf], (units++ / NQ) & 1);
            if (!ok) break;
            const float qf = qscale[buf * kPreRows + tile * 128 + r];
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_seen[buf]);
            const int unit_row = tile * 128 + r;
            const int side = cur.step == 0 ? 1 : 0;  // the piece begins its unit, or goes on with it
            float* piece = pieces + ((size_t)blockIdx.x * 2 + side) * S::kPieceFloats;
            // Adds O to the second accumulator, which carries the factor `since` behind its last addition.
            bool flushed = false;
            float since = 1.0f;
            auto sum_at = [&](int e4) { return reinterpret_cast<float4*>(piece + ((size_t)e4 * kPreRows + unit_row) * 4); };
            auto flush = [&]() {
#pragma unroll 1
                for (int ch = 0; ch < D / 16; ++ch) {
                    uint32_t w[16];
                    tmem_ld16(to + ch * 16, w);
                    if constexpr (S::kSumInTmem) {
                        uint32_t z[16];
                        if (flushed) tmem_ld16(tsum + ch * 16, z);
                        tmem_wait_ld(w);
                        if (flushed) {
                            tmem_wait_ld(z);
#pragma unroll
                            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__fmaf_rn(__uint_as_float(z[e]), since, __uint_as_float(w[e])));
                        }
                        tmem_st16(tsum + ch * 16, w);
                    } else {
                        float4 z[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) z[q] = flushed ? __ldcg(sum_at(ch * 4 + q)) : make_float4(0, 0, 0, 0);
                        tmem_wait_ld(w);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            z[q].x = __fmaf_rn(z[q].x, since, __uint_as_float(w[4 * q]));
                            z[q].y = __fmaf_rn(z[q].y, since, __uint_as_float(w[4 * q + 1]));
                            z[q].z = __fmaf_rn(z[q].z, since, __uint_as_float(w[4 * q + 2]));
                            z[q].w = __fmaf_rn(z[q].w, since, __uint_as_float(w[4 * q + 3]));
                            __stcg(sum_at(ch * 4 + q), z[q]);
                        }
                    }
                }
                flushed = true;
                since = 1.0f;
            };
            const bool part_of_it = tile < tiles;
            float m = -INFINITY, l = 0.0f, vl = kPreNoScale;  // vl: log2 of the reference value scale
            // The products of the step before are in O.  Waited for in every step,
            // before its own weights are handed over: a wait knows only the
            // parity of a phase, so none may be passed over.
            auto settled = [&]() {
                ok = wait(&pv_done[tile], (np - 1) & 1);
                tc_fence_after();
                return ok;
            };
            for (int k0 = 0; k0 < n && ok && part_of_it; k0 += S::kFlush) {
                if (k0 > 0) {
                    if (!settled()) break;
                    flush();
                }
                const int k1 = min(n, k0 + S::kFlush);
                for (int k = k0; k < k1 && ok; ++k, ++np) {
                    const int ring = (i + k) % kPreScaleRing;
                    const uint32_t ts = tmem + lane_base + tile * 2 * NT + (np & 1) * NT;
                    ok = wait(&sc_full[ring], ((i + k) / kPreScaleRing) & 1) && wait(&s_full[tile * 2 + (np & 1)], (np >> 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const int t0 = (cur.step + k) * NT;
                    const unsigned groups = valid[ring * 2];
                    const bool whole = t0 + NT <= seen_min && groups == (1u << G) - 1u;
                    const float2* sc = scales + ring * G;
                    // Largest score, group by group: the scale is applied to a group's
                    // maximum.  The loops over groups stay loops: unrolled, their code is
                    // larger than the schedulers' instruction caches.
                    float top = -INFINITY, lvmax = kPreNoScale;
                    auto largest = [&](auto masked) {
#pragma unroll 1
                        for (int g0 = 0; g0 < G; g0 += 2) {
                            uint32_t w[32];
                            tmem_ld32(ts + g0 * 16, w);
                            tmem_wait_ld32(w);
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                const int gr = g0 + b;
                                const float2 g2 = sc[gr];
                                const int left = masked ? (groups >> gr & 1 ? seen - t0 - gr * 16 : 0) : 16;
                                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                                for (int e = 0; e < 16; ++e)
                                    mx[e & 3] = fmaxf(mx[e & 3], !masked || e < left ? __uint_as_float(w[b * 16 + e]) : -INFINITY);
                                const float m4 = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                                top = fmaxf(top, masked && left <= 0 ? -INFINITY : m4 * (g2.x * qf));
                                lvmax = fmaxf(lvmax, g2.y);
                            }
                        }
                    };
                    if (whole) largest(std::false_type());
                    else largest(std::true_type());
                    // p <= 2^6 * 2^6 * 2^3 < 65504
                    const bool move = top > m + 6.0f, vmove = lvmax > vl + 3.0f;
                    if (__any_sync(0xffffffffu, move) || vmove) {
                        float f = 1.0f;
                        if (move) {
                            f = ex2(m - top);
                            l *= f;
                            m = top;
                        }
                        if (vmove) {
                            f *= ex2(vl - lvmax);
                            vl = lvmax;
                        }
                        since *= f;
                        if (k > k0) {  // step k0 begins O anew
                            if (!settled()) break;
#pragma unroll 1
                            for (int ch = 0; ch < D / 16; ++ch) {
                                uint32_t z[16];
                                tmem_ld16(to + ch * 16, z);
                                tmem_wait_ld(z);
#pragma unroll
                                for (int e = 0; e < 16; ++e) z[e] = __float_as_uint(__uint_as_float(z[e]) * f);
                                tmem_st16(to + ch * 16, z);
                            }
                        }
                    }
                    const float bias = m == -INFINITY ? 0.0f : 6.0f - m;
                    auto weigh = [&](auto masked) {
#pragma unroll 1
                        for (int g0 = 0; g0 < G; g0 += 2) {
                            uint32_t w[32];
                            tmem_ld32(ts + g0 * 16, w);
                            tmem_wait_ld32(w);
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                const int gr = g0 + b;
                                uint32_t ph[8], pl[8];
                                const float2 g2 = sc[gr];
                                const float lr0 = g2.y - vl, lr = lr0 < -40.0f ? -40.0f : lr0;  // a NaN stays
                                const float cf = g2.x * qf, bb = bias + lr, out = ex2(-lr);
                                const int left = masked ? (groups >> gr & 1 ? seen - t0 - gr * 16 : 0) : 16;
                                const uint64_t cf2 = pair(cf, cf), b2 = pair(bb, bb);
                                uint64_t part = 0;
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const float2 xx = unpair(fma2(pair(__uint_as_float(w[b * 16 + 2 * e]), __uint_as_float(w[b * 16 + 2 * e + 1])), cf2, b2));
                                    const float p0 = ex2(!masked || 2 * e < left ? xx.x : -INFINITY);
                                    const float p1 = ex2(!masked || 2 * e + 1 < left ? xx.y : -INFINITY);
                                    const uint64_t p = pair(p0, p1);
                                    part = add2(part, p);
                                    const __half2 hh = __floats2half2_rn(p0, p1);
                                    ph[e] = *reinterpret_cast<const uint32_t*>(&hh);
                                    const float2 f = __half22float2(hh);
                                    pl[e] = pack_f16(p0 - f.x, p1 - f.y);
                                }
                                const float2 s2 = unpair(part);
                                l = __fmaf_rn(s2.x + s2.y, out, l);
                                // Over the 16 columns of these tokens: hi, then lo.
                                tmem_st8(ts + gr * 16, ph);
                                tmem_st8(ts + gr * 16 + 8, pl);
                            }
                        }
                    };
                    if (whole) weigh(std::false_type());
                    else weigh(std::true_type());
                    tmem_wait_st();
                    if (k > 0 && !settled()) break;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_ready[tile * 2 + (np & 1)]);
                }
            }
            i += n;
            if (ok && part_of_it) {
                // ---- the segment's end ----
                ok = wait(&pv_done[tile], (np - 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const bool whole_unit = cur.step == 0 && n == cur.steps;
                const float vref = exp2f(vl);  // the smallest numbers too
                T* dst = (T*)a.out + (int64_t)(cur.q.row0 + (live ? j : 0)) * a.out_stride + col;
                auto write = [&](int e0, const float (&v)[8]) {
                    if (!live) return;
                    if (o16) {
                        constexpr int V = 16 / sizeof(T);
#pragma unroll
                        for (int b = 0; b < 8 / V; ++b) {
                            uint4 u;
                            T* t = reinterpret_cast<T*>(&u);
#pragma unroll
                            for (int q = 0; q < V; ++q) t[q] = (T)v[b * V + q];
                            *reinterpret_cast<uint4*>(dst + e0 + b * V) = u;
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 8; ++q) dst[e0 + q] = (T)v[q];
                    }
                };
                const float f = whole_unit ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;  // vref / l could be too small a number
#pragma unroll 1
                for (int ch = 0; ch < D / 32; ++ch) {
                    uint32_t w[32];
                    tmem_ld32(to + ch * 32, w);
                    if constexpr (S::kSumInTmem) {
                        uint32_t z[32];
                        if (flushed) tmem_ld32(tsum + ch * 32, z);
                        tmem_wait_ld32(w);
                        if (flushed) {
                            tmem_wait_ld32(z);
#pragma unroll
                            for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__fmaf_rn(__uint_as_float(z[e]), since, __uint_as_float(w[e])));
                        }
                    } else {
                        tmem_wait_ld32(w);
                        if (flushed) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const float4 z = __ldcg(sum_at(ch * 8 + q));
                                w[4 * q] = __float_as_uint(__fmaf_rn(z.x, since, __uint_as_float(w[4 * q])));
                                w[4 * q + 1] = __float_as_uint(__fmaf_rn(z.y, since, __uint_as_float(w[4 * q + 1])));
                                w[4 * q + 2] = __float_as_uint(__fmaf_rn(z.z, since, __uint_as_float(w[4 * q + 2])));
                                w[4 * q + 3] = __float_as_uint(__fmaf_rn(z.w, since, __uint_as_float(w[4 * q + 3])));
                            }
                        }
                    }
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = whole_unit && l == 0.0f ? 0.0f : __uint_as_float(w[b * 8 + e]) * f * vref;
                        if (whole_unit) {
                            write(ch * 32 + b * 8, v);
                        } else {  // [element / 4][row][4]
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                *reinterpret_cast<float4*>(piece + ((ch * 8 + b * 2 + q) * kPreRows + unit_row) * 4) =
                                    make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        }
                    }
                }
                tc_fence_before();
                if (!whole_unit) {
                    piece[kPreRows * D + unit_row] = m;
                    piece[kPreRows * D + kPreRows + unit_row] = l;
                    const unsigned u0 = x - cur.step, u1 = u0 + cur.steps;
                    const int first = (int)worker_of(u0), last = (int)worker_of(u1 - 1);
                    __threadfence();
                    __syncwarp();
                    int old = 0;
                    if (lane == 0) old = atomicAdd(counters + first * 8 + warp, 1);
                    old = __shfl_sync(0xffffffffu, old, 0);
                    if (old == last - first) {  // every piece of these 32 rows is there
                        if (lane == 0) counters[first * 8 + warp] = 0;
                        __threadfence();
                        auto at = [&](int b) { return pieces + ((size_t)b * 2 + (b == first ? 1 : 0)) * S::kPieceFloats; };
                        float mx = -INFINITY, sum = 0.0f;
                        for (int b = first; b <= last; ++b) mx = fmaxf(mx, __ldcg(at(b) + kPreRows * D + unit_row));
                        for (int b = first; b <= last; ++b) {
                            const float pm = __ldcg(at(b) + kPreRows * D + unit_row);
                            sum += __ldcg(at(b) + kPreRows * D + kPreRows + unit_row) * (pm == -INFINITY ? 0.0f : ex2(pm - mx));
                        }
                        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
                        for (int e0 = 0; e0 < D; e0 += 32) {
                            float v[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = 0.0f;
                            for (int b = first; b <= last; ++b) {
                                const float* pc = at(b);
                                const float pm = __ldcg(pc + kPreRows * D + unit_row);
                                const float h = pm == -INFINITY ? 0.0f : ex2(pm - mx);
#pragma unroll
                                for (int q = 0; q < 8; ++q) {
                                    const float4 u = __ldcg(reinterpret_cast<const float4*>(pc + ((e0 / 4 + q) * kPreRows + unit_row) * 4));
                                    v[4 * q] += u.x * h, v[4 * q + 1] += u.y * h, v[4 * q + 2] += u.z * h, v[4 * q + 3] += u.w * h;
                                }
                            }
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                float y[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) y[e] = sum == 0.0f ? 0.0f : v[b * 8 + e] * inv;
                                write(e0 + b * 8, y);
                            }
                        }
                    }
                }
            }
            x += n;
            cur.step += n;
            if (cur.step == cur.steps) {
                x += kPreUnitCost;
                if (x < hi) next_unit(cur);
            }
        }
    }
    // Everyone meets when all products and their arrivals are done, also where
    // a wait has given up.
    if (warp == 12 || warp == 13) {
        if (elect_one()) tc_commit(&drained);
        mbar_wait_bounded(&drained, 0, &unset, globaltimer_ns() + timeout_ns, kDevTimeoutDrain);
        if (unset) atomicCAS(err, 0, kDevTimeoutDrain);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <typename T, int FMT, int D>
cudaError_t kv8_prefill_prepare() {
    // The register split draws on what the launch has: more than that would wait forever.
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, kv8_prefill_kernel<T, FMT, D>);
    if (e != cudaSuccess) return e;
    if (attr.numRegs < PreShape<T, D>::kRegsLaunch) return cudaErrorInvalidKernelImage;
    return cudaFuncSetAttribute(kv8_prefill_kernel<T, FMT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                PreShape<T, D>::kSmem + (kPagesMaxSeqs + 1) * (int)sizeof(unsigned));
}

template <typename T, int FMT, int D>
cudaError_t launch_kv8_prefill(const Kv8& c, const Kv8Attention& a, int num_sms, void* ws, int* err, cudaStream_t st) {
    const int smem = PreShape<T, D>::kSmem + (a.n_seqs + 1) * (int)sizeof(unsigned);
    int* counters = (int*)ws;
    float* pieces = (float*)((uint8_t*)ws + kv8_prefill_counter_bytes(num_sms));
    return launch_ex(kv8_prefill_kernel<T, FMT, D>, dim3(num_sms), dim3(kPreThreads), smem, st, true, c, a, pieces, counters,
                     err, (uint64_t)2000000000ull);
}

}  // namespace lc
