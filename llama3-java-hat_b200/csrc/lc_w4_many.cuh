// lc_w4_many.cuh -- products of 4-bit weights with many rows (batches, prompts),
// on the tcgen05 tensor cores.
//
// Two kernels.  The first lays the rows of x out as f16 operands in the context's
// workspace: F16 rows as they are, F32 rows as hi + lo under a power-of-two row
// scale (2^-22), rows and columns that are not there as zeros.  The second has
// units of 256 rows of W and up to 128 rows of x (F32: 64),
//   D = A B   M 128 (twice), N up to 128, K one group (F32: A Bhi + A Blo)
// with A = (c - z) / 4, exact in f16, made from the codes.  A group's D is added,
// under the group's scale, to fp32 sums that an epilogue thread keeps in registers
// for its row of W, while the tensor cores fill the other D: so scales need no
// rounding into weights, and the tensor cores' own truncating sums run over 128
// columns at most.
//
// What bounds it: shared memory, while A lies there (units of more than 64 rows of
// x, whose Ds fill tensor memory): the products of a block of 128 columns read 128
// KB of it and the rest moves as much again, 2048 cycles where the tensor cores
// need 1024 (2048 F16 rows of 16384 x 2048, groups of 128: 208 us, 83 at the measured
// rate).  Up to 64 rows A is in tensor memory, a thread writing its row; making it
// takes the operand warps some 1300 cycles of a block (17 F16 rows of 128256 x 2048:
// 62 us, 22 at the measured copy's rate; with A in shared memory 73).  Groups of 32
// are bound by reading D, four times per block.
//
// Warps 0-7: epilogue, four for each 128 rows.  Warps 8-15: codes to operands,
// through rings of their own (cp.async).  Warp 16 issues the products, warp 17 the
// copies of x (bulk copies, whole stages).  Registers move to the epilogue.  With
// few units a cluster shares the columns; its CTAs add their sums through each
// other's shared memory.
#pragma once

#include <type_traits>

#include "lc_internal.h"
#include "lc_tcgen05.cuh"
#include "lc_w4.h"
#include "lc_w4_few.cuh"

namespace lc {

constexpr int kManyThreads = 20 * 32;
constexpr int kManyRows = 256;      // of W, of a unit
constexpr int kManyCols = 128;      // of D, for 128 rows of W
constexpr int many_most(bool split) { return split ? 64 : 128; }  // rows of x of a unit, at most
constexpr int kManyK = kW4Cols;     // columns of W of a stage: a block
constexpr int kManyStages = 2, kManyMaxRing = 5;  // stages of operands
constexpr int kManyACol = 256;  // tensor memory: Ds below, and A where it lies there
constexpr int kManyABytes = kManyRows * kManyK * 2;
constexpr int kManyRingBytes = 2 * kW4BlockBytes;  // of a warp: a block of two tiles
constexpr int kManySmem = 226 * 1024;
constexpr int kManyMaxCluster = 8;
// Registers after the split; their sum over the five warpgroups is the launch's.
// Units of 128 rows of x have sums of 128 registers.
template <bool BIG>
struct ManyRegs {
    static constexpr int kSum = BIG ? 168 : 136, kCodes = BIG ? 48 : 80, kRest = 48;
    static constexpr int kLaunch = (2 * kSum + 2 * kCodes + kRest + 4) / 5;
};

struct ManyPlan {
    int n;         // rows of x of a unit, a multiple of 16
    int x_tiles, w_tiles;
    int cluster;   // CTAs that share the columns of W, a power of two
    int cluster_log2;
    int sets;      // Ds of a block: one per group, or per two where they fit
    int ring;      // blocks of a warp's ring of codes
    const uint8_t* b;      // [x tile][block][hi, lo][n / 8][16 octets][8][16 bytes]
    const float* factor;   // [batch] what the rows of x were divided by
};

constexpr int kLayThreads = 512;

// A CTA lays out eight rows, with two warps each.
template <typename T>
__global__ void __launch_bounds__(kLayThreads) w4_lay_kernel(W4Product p, int cols, int blocks, ManyPlan plan, uint8_t* b, float* factor) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int R = 8, PARTS = kLayThreads / 32 / R;  // rows of a CTA, warps of a row
    constexpr int HOLD = 4;  // octets of columns that a lane keeps at a time
    __shared__ float tops[kLayThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % PARTS;
    griddep_wait();
    griddep_launch();
    const int groups = plan.n / 8, tile = blockIdx.x / groups, group = blockIdx.x % groups;
    const int r = group * R + warp / PARTS, row = tile * plan.n + r;
    const bool there = row < p.batch;
    const T* const x = (const T*)p.x + (there ? row * p.x_stride : 0);
    const bool vec = ((uintptr_t)p.x | (uintptr_t)(p.x_stride * sizeof(T))) % 16 == 0;
    const int octets = blocks * 16;
    auto eight = [&](int o, float (&v)[8]) {
        const int c = o * 8;
        if (there && vec && c + 8 <= cols) {
            if (SPLIT) {
                const float4 lo = *reinterpret_cast<const float4*>(x + c), hi = *reinterpret_cast<const float4*>(x + c + 4);
                v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
            } else {
                unpack_h8(*reinterpret_cast<const uint4*>(x + c), v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = there && c + i < cols ? (float)x[c + i] : 0.0f;
        }
    };
    float v[HOLD][8];
    auto load = [&](int base) {
#pragma unroll
        for (int h = 0; h < HOLD; ++h) {
            const int o = base + (h * PARTS + part) * 32 + lane;
            if (o < octets) eight(o, v[h]);
        }
    };
    constexpr int STEP = HOLD * PARTS * 32;
    float up = 1.0f;
    load(0);
    if (SPLIT) {
        float top = 0.0f;
        for (int base = 0; base < octets; base += STEP) {
            if (base) load(base);
#pragma unroll
            for (int h = 0; h < HOLD; ++h) {
                if (base + (h * PARTS + part) * 32 + lane >= octets) continue;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[h][i]));
            }
        }
        top = warp_max(top);
        if (lane == 0) tops[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PARTS; ++i) top = fmaxf(top, tops[warp / PARTS * PARTS + i]);
        const int e = split_row_exp(top);
        up = pow2f(e);
        if (there && part == 0 && lane == 0) factor[row] = pow2f(-e);
        if (octets > STEP) load(0);
    }
    constexpr int HALVES = SPLIT ? 2 : 1;
    uint8_t* const to = b + ((int64_t)tile * blocks * HALVES * groups + group) * 2048 + (r & 7) * 16;
    for (int base = 0; base < octets; base += STEP) {
        if (base) load(base);
#pragma unroll
        for (int h = 0; h < HOLD; ++h) {
            const int o = base + (h * PARTS + part) * 32 + lane;
            if (o >= octets) continue;
            if (SPLIT) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[h][i] *= up;
            }
            uint4 hi, lo;
            split_octet(v[h], hi, lo);
            uint8_t* const at = to + (int64_t)(o >> 4) * HALVES * groups * 2048 + (o & 15) * 128;
            *reinterpret_cast<uint4*>(at) = hi;
            if (SPLIT) *reinterpret_cast<uint4*>(at + groups * 2048) = lo;
        }
    }
}

LC_DEV uint64_t many_pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
LC_DEV uint64_t many_pair(uint32_t a, uint32_t b) { return (uint64_t)b << 32 | a; }
LC_DEV float2 many_two(uint64_t v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }
LC_DEV uint64_t many_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
LC_DEV void many_ld32(uint32_t taddr, uint32_t (&v)[32]) {
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
LC_DEV void many_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                   "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                   "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
LC_DEV void many_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
        "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
        "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
LC_DEV void many_mma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
LC_DEV bool many_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
LC_DEV void many_sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
LC_DEV uint32_t many_hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t v;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(a), "r"(b), "r"(c));
    return v;
}
// The eight codes of a word as f16 pairs c 2^-17: rows g, g + 8 of columns e = 0, 1,
// then of 2, 3.
LC_DEV void many_codes(uint32_t w, uint32_t (&a)[4]) {
    constexpr uint32_t kMask = 0x07800780u;
    a[0] = __funnelshift_l(w, w, 4) & kMask;
    a[1] = w & kMask;
    a[2] = __funnelshift_r(w, w, 4) & kMask;
    a[3] = __funnelshift_r(w, w, 8) & kMask;
}
LC_DEV void many_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// COLS: rows of x of a unit at most, 64 or 128 (without a residual, for which there
// are no registers).
template <typename T, int GROUP, bool ZEROS, int COLS>
__global__ void __launch_bounds__(kManyThreads, 1) w4_many_kernel(W4 w, W4Product p, ManyPlan plan, int* err, uint64_t timeout_ns) {
    constexpr bool SPLIT = sizeof(T) == 4;
    static_assert(COLS <= many_most(SPLIT), "");
    using R = ManyRegs<COLS == 128>;
    constexpr bool TA = COLS == 64;                // A in tensor memory
    constexpr int DCOLS = TA ? 64 : kManyCols;     // columns of a D for 128 rows of W
    constexpr int NG = kW4Cols / GROUP;
    constexpr int NS = kManyStages, HALVES = SPLIT ? 2 : 1;
    const uint32_t b_bytes = HALVES * plan.n * kManyK * 2;  // of a stage
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const sa = smem;                            // [stages][tile of 128 rows][row groups][octets][8][16]
    uint8_t* const sb = sa + (TA ? 0 : NS * kManyABytes);  // [stages][hi, lo][column groups][octets][8][16]
    uint8_t* const sc = sb + NS * b_bytes;               // [warps][ring][tile][half][lane][16]
    __shared__ __align__(8) uint64_t full[NS], empty[NS], d_full[2], d_free[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int unset;  // an error word of its own for the drain, which waits also after a failure
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cs = plan.cluster, units = plan.x_tiles * plan.w_tiles;
    uint32_t rank = 0;
    if (cs > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    if (tid == 0) {
        unset = 0;
        for (int i = 0; i < NS; ++i) mbar_init(&full[i], 8 + 1), mbar_init(&empty[i], 1);  // operand warps and the copy of x
        for (int i = 0; i < 2; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_free[i], 8);
        mbar_init(&drained, 1);
        fence_mbar_init();
    }
    if (warp == 16) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_launch();
    const uint32_t tmem = tmem_slot;
    // Units of this CTA: those of a range (neighbours share rows of x), or one of a cluster.
    const int ctas = gridDim.x / cs, id = blockIdx.x / cs;
    const int u0 = (int)((int64_t)units * id / ctas), u1 = (int)((int64_t)units * (id + 1) / ctas);
    const int block0 = (int)((int64_t)w.blocks * (int)rank / cs), block1 = (int)((int64_t)w.blocks * ((int)rank + 1) / cs);
    const int blocks = block1 - block0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // by whole warps, which go on together
        return (bool)__all_sync(0xffffffffu, mbar_try_wait(bar, parity) ||
                                                 mbar_wait_bounded(bar, parity, err, globaltimer_ns() + timeout_ns, kDevTimeoutGrid));
    };

    if (warp >= 8 && warp < 16) {
        // ---- codes to operands ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::kCodes));
        // Operands in shared memory: lane 8 t + g has rows g and g + 8 of a tile, so that
        // eight lanes write one core matrix; in tensor memory: lane 16 k + r has row r of
        // the warp's tile k.
        const int cw = warp - 8, g = lane & 7, t = lane >> 3;
        const uint32_t ring0 = smem_u32(sc) + cw * plan.ring * kManyRingBytes;
        // Where the lane puts the 16 bytes that it copies of a chunk, those of lane 4 g + t
        // of the layout.  For tensor memory rows are read by the lane, four times 16 bytes
        // next to each other: turned by g / 2, eight rows then lie in all banks.
        const uint32_t ring = ring0 + (TA ? 4 * g + ((t + (g >> 1)) & 3) : lane) * 16;
        int a_unit = u0, a_block = 0;
        auto tile_of = [&](int unit, int k) { return min((unit % plan.w_tiles) * (kManyRows / kW4Rows) + cw * 2 + k, w.tiles - 1); };
        const uint8_t* a_from[2];
        auto request = [&](int slot) {
            if (a_unit < u1) {
                if (a_block == 0) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        a_from[k] = w.codes + ((int64_t)tile_of(a_unit, k) * w.blocks + block0) * kW4BlockBytes + (4 * g + t) * 16;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    few_copy16(ring + slot * kManyRingBytes + k * 1024, a_from[k]);
                    few_copy16(ring + slot * kManyRingBytes + k * 1024 + 512, a_from[k] + 512);
                    a_from[k] += kW4BlockBytes;
                }
                if (++a_block == blocks) a_block = 0, ++a_unit;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // Zero points of the lane's rows: pairs (rows g, g + 8) of a block's groups, of
        // both tiles or of the lane's.
        constexpr int ZW = (NG + 1) / 2, ZT = TA ? 1 : 2;  // words, tiles
        uint32_t zero[ZT][ZW];
        auto load_zeros = [&](int unit, int block) {
            if constexpr (ZEROS) {
                if (unit >= u1) return;
#pragma unroll
                for (int k = 0; k < ZT; ++k) {
                    const uint8_t* z = w.zeros + (((int64_t)tile_of(unit, TA ? lane >> 4 : k) * w.blocks + block0 + block) * 8 + g) * NG * 2;
#pragma unroll
                    for (int i = 0; i < ZW; ++i) {
                        if constexpr (NG == 1) {
                            uint16_t v;
                            asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(z));
                            zero[k][i] = v;
                        } else {
                            asm volatile("ld.global.u32 %0, [%1];" : "=r"(zero[k][i]) : "l"(z + 4 * i));
                        }
                    }
                }
            }
        };
        auto quarter = [](uint32_t v) {  // -z / 4, twice
            const __half2 h = __half2half2(__float2half_rn(-0.25f * (float)(v & 255u)));
            return *reinterpret_cast<const uint32_t*>(&h);
        };
        constexpr uint32_t kUp = 0x78007800u;  // 2^15, twice: c 2^-17 2^15 - z / 4 is exact
        for (int i = 0; i < plan.ring - 1; ++i) request(i);
        load_zeros(u0, 0);
        int i = 0, slot = 0;
        for (int unit = u0; unit < u1 && ok; ++unit) {
            for (int block = 0; block < blocks && ok; ++block, ++i) {
                request(slot == 0 ? plan.ring - 1 : slot - 1);
                switch (plan.ring) {  // all but the newest ring - 1 have landed
                    case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
                    case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
                    case 4: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
                    default: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
                }
                uint32_t z[ZT][ZW];
#pragma unroll
                for (int k = 0; k < ZT; ++k)
#pragma unroll
                    for (int j = 0; j < ZW; ++j) z[k][j] = ZEROS ? zero[k][j] : 0x08080808u;
                if (block + 1 < blocks) load_zeros(unit, block + 1);
                else load_zeros(unit + 1, 0);
                const int st = i % NS;
                if constexpr (TA) {
                    __syncwarp();  // the copies of all lanes have landed
                    if (i >= NS) ok = wait(&empty[st], (i / NS - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();  // the products that read this stage's A come before what is written over it
                    const uint32_t held = ring0 + slot * kManyRingBytes + (lane >> 4) * 1024 + g * 64;
                    const int up = (lane >> 1) & 4;  // 4: rows g + 8, whose codes are 4 bits higher
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 64 columns
                        uint32_t v[32];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {  // octets e and 4 + e
                            const uint4 c = few_lds128(held + h * 512 + ((e + (g >> 1)) & 3) * 16);
                            const uint32_t ws[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int group = (2 * h + (j >> 1)) / (4 / NG);
                                const uint32_t zq = ZEROS ? quarter(z[0][group >> 1] >> (16 * (group & 1) + 2 * up)) : 0xc000c000u;
                                const uint32_t lo = __funnelshift_l(ws[j], ws[j], 4 - up) & 0x07800780u;
                                const uint32_t hi = __funnelshift_r(ws[j], ws[j], 4 + up) & 0x07800780u;
                                v[16 * (j >> 1) + 4 * e + 2 * (j & 1)] = many_hfma2(lo, kUp, zq);
                                v[16 * (j >> 1) + 4 * e + 2 * (j & 1) + 1] = many_hfma2(hi, kUp, zq);
                            }
                        }
                        many_st32(tmem + ((uint32_t)(cw & 3) << 21) + kManyACol + (st * 2 + (cw >> 2)) * 64 + h * 32, v);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                } else {
                    uint4 held[4];  // [tile][half]: read before anything is written, or each would wait for the one before
#pragma unroll
                    for (int k = 0; k < 4; ++k) held[k] = few_lds128(ring + slot * kManyRingBytes + k * 512);
                    if (i >= NS) ok = wait(&empty[st], (i / NS - 1) & 1);
                    if (!ok) break;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint4 c = held[k];
                        const int tl = cw * 2 + (k >> 1);
                        const uint32_t to = smem_u32(sa) + st * kManyABytes + (tl >> 3) * (kManyABytes / 2) + (tl & 7) * 4096 + (k & 1) * 1024 + t * 128 + g * 16;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {  // runs of eight columns
                            uint32_t a[4], b[4];
                            many_codes(q ? c.z : c.x, a);
                            many_codes(q ? c.w : c.y, b);
                            const int group = (2 * (k & 1) + q) / (4 / NG);
                            const uint32_t zq = z[(k >> 1) % ZT][group >> 1] >> (16 * (group & 1));
                            const uint32_t z0 = ZEROS ? quarter(zq) : 0xc000c000u, z1 = ZEROS ? quarter(zq >> 8) : 0xc000c000u;
                            many_sts128(to + q * 512, many_hfma2(a[0], kUp, z0), many_hfma2(a[2], kUp, z0), many_hfma2(b[0], kUp, z0), many_hfma2(b[2], kUp, z0));
                            many_sts128(to + 2048 + q * 512, many_hfma2(a[1], kUp, z1), many_hfma2(a[3], kUp, z1), many_hfma2(b[1], kUp, z1), many_hfma2(b[3], kUp, z1));
                        }
                    }
                    fence_async_shared();
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive(&full[st]);
                slot = slot == plan.ring - 1 ? 0 : slot + 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (cs > 1) many_cluster_sync(), many_cluster_sync();
    } else if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::kRest));
        if (warp == 16) {
            // ---- products ----
            // A wait costs the warp some 200 cycles and a commit 100, so a stage is a whole
            // block, its operands share a barrier, and as many groups as fit make one D.
            const uint32_t idesc = tc_idesc_f16_f32(128, plan.n);
            const uint64_t ad = tc_desc_kmajor(smem_u32(sa), 128, 2048), bd = tc_desc_kmajor(smem_u32(sb), 128, 2048);
            const uint32_t b_half = plan.n * kManyK * 2 / 16;
            constexpr int STEPS = GROUP / 16;  // products of a group
            auto issue = [&](auto sets) {
                constexpr int SETS = decltype(sets)::value, PER = NG / SETS, WIDE = DCOLS / PER;  // groups of a D, columns of one
                int i = 0, d = 0;  // stages and Ds so far
                for (int n = (u1 - u0) * blocks; i < n && ok; ++i) {
                    const int st = i % NS;
                    const uint64_t a0 = ad + st * (kManyABytes / 16), b0 = bd + st * HALVES * b_half;
                    ok = wait(&full[st], (i / NS) & 1);
#pragma unroll
                    for (int set = 0; set < SETS; ++set, ++d) {
                        if (ok && d >= 2) ok = wait(&d_free[d & 1], ((d >> 1) - 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t to = tmem + (d & 1) * 2 * DCOLS, ta = tmem + kManyACol + st * 128;
                        if (many_elect()) {
#pragma unroll
                            for (int k = set * PER * STEPS; k < (set + 1) * PER * STEPS; ++k) {
                                const uint32_t at = to + (k / STEPS - set * PER) * 2 * WIDE;
#pragma unroll
                                for (int h = 0; h < HALVES; ++h) {
                                    const uint64_t b = b0 + h * b_half + k * 16;
                                    if (TA) {
                                        many_mma_ta(at, ta + k * 8, b, idesc, k % STEPS != 0 || h);
                                        many_mma_ta(at + WIDE, ta + 64 + k * 8, b, idesc, k % STEPS != 0 || h);
                                    } else {
                                        tc_mma_f16(at, a0 + k * 16, b, idesc, k % STEPS != 0 || h);
                                        tc_mma_f16(at + WIDE, a0 + kManyABytes / 32 + k * 16, b, idesc, k % STEPS != 0 || h);
                                    }
                                }
                            }
                            tc_commit(&d_full[d & 1]);
                            if (set == SETS - 1) tc_commit(&empty[st]);
                        }
                        __syncwarp();
                    }
                }
            };
            if (plan.sets == 1) issue(std::integral_constant<int, 1>());
            else if (NG >= 2 && plan.sets == 2) issue(std::integral_constant<int, NG >= 2 ? 2 : 1>());
            else issue(std::integral_constant<int, NG>());
        } else if (warp == 17) {
            // ---- copies of x ----
            griddep_wait();
            const uint64_t policy = l2_policy_evict_last();
            int i = 0;
            for (int unit = u0; unit < u1 && ok; ++unit) {
                const uint8_t* from = plan.b + ((int64_t)(unit / plan.w_tiles) * w.blocks + block0) * b_bytes;
                for (int block = 0; block < blocks && ok; ++block, ++i, from += b_bytes) {
                    const int st = i % NS;
                    if (i >= NS) ok = wait(&empty[st], (i / NS - 1) & 1);
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&full[st], b_bytes);
                        bulk_g2s(sb + st * b_bytes, from, b_bytes, &full[st], policy);
                    }
                    __syncwarp();
                }
            }
            // The last copies land before the CTA may end.  Their stages are full once the
            // operand warps have come, too; after a failure these may not, and it takes
            // the limit.
            for (int k = i > NS ? i - NS : 0; k < i; ++k)
                mbar_wait_bounded(&full[k % NS], (k / NS) & 1, &unset, globaltimer_ns() + timeout_ns, kDevTimeoutDrain);
        }
        __syncwarp();
        if (cs > 1) many_cluster_sync(), many_cluster_sync();
    } else {
        // ---- sums ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R::kSum));
        griddep_wait();
        constexpr int PAIRS = COLS / 2;  // of rows of x
        const int row = warp * 32 + lane;   // of the unit
        const int per = NG / plan.sets, columns = DCOLS / per;  // groups of a D, columns of one
        const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + (warp >> 2) * columns;
        int d = 0;
        for (int unit = u0; unit < u1; ++unit) {
            const int wt = unit % plan.w_tiles, xt = unit / plan.w_tiles;
            const int64_t out = (int64_t)wt * kManyRows + row;
            const int tile = min(wt * (kManyRows / kW4Rows) + (row >> 4), w.tiles - 1);
            uint64_t total[PAIRS];
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) total[k] = 0;
            // Scales of a block: pairs (rows g, g + 8) of its groups.
            uint32_t sc_next[NG];
            auto load_scales = [&](int block) {
                const uint32_t* s = reinterpret_cast<const uint32_t*>(w.scales) + (((int64_t)tile * w.blocks + block) * 8 + (row & 7)) * NG;
                // Volatile: a load that the compiler may move goes to its use.
                if constexpr (NG == 4)
                    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(sc_next[0]), "=r"(sc_next[1]), "=r"(sc_next[2]), "=r"(sc_next[3]) : "l"(s));
                else if constexpr (NG == 2)
                    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(sc_next[0]), "=r"(sc_next[1]) : "l"(s));
                else
                    asm volatile("ld.global.u32 %0, [%1];" : "=r"(sc_next[0]) : "l"(s));
            };
            // They stream from HBM like the codes: asked for eight blocks ahead.
            auto prefetch_scales = [&](int block) {
                const uint32_t* s = reinterpret_cast<const uint32_t*>(w.scales) + (((int64_t)tile * w.blocks + block) * 8 + (row & 7)) * NG;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(s));
            };
            for (int block = block0 + 1; block < min(block0 + 8, block1); ++block) prefetch_scales(block);
            if (COLS == 64 && p.residual && (cs == 1 || rank == 0)) {  // to L2, while the sums are made
                constexpr int LINES = kManyRows * sizeof(T) / 128 + 1;
                const int64_t c0 = (int64_t)wt * kManyRows, wide = min((int64_t)kManyRows, w.rows - c0);
                for (int i = row; i < min(plan.n, p.batch - xt * plan.n) * LINES; i += kManyRows) {
                    const int64_t at = min((int64_t)(i % LINES) * (128 / (int)sizeof(T)), wide - 1);
                    asm volatile("prefetch.global.L2 [%0];" ::"l"((const T*)p.residual + (xt * plan.n + i / LINES) * p.residual_stride + c0 + at));
                }
            }
            load_scales(block0);
            for (int block = block0; block < block1 && ok; ++block) {
                uint32_t scale[NG];
#pragma unroll
                for (int k = 0; k < NG; ++k) scale[k] = row & 8 ? sc_next[k] >> 16 : sc_next[k] & 0xffffu;
                if (block + 1 < block1) load_scales(block + 1);
                if (block + 8 < block1) prefetch_scales(block + 8);
                // A load from tensor memory takes some 200 cycles whatever its size, so as much
                // as registers hold is asked for at once: 64 columns, of one group or of two,
                // or 32 where the sums take 128 registers.
                auto take = [&](int k) {  // tensor memory of group k, when it is there
                    const int in = k & (per - 1);
                    if (in == 0 && ok) {
                        ok = wait(&d_full[d & 1], (d >> 1) & 1);
                        tc_fence_after();
                    }
                    return from + (d & 1) * 2 * DCOLS + in * 2 * columns;
                };
                auto give = [&](int k) {
                    if ((k & (per - 1)) != per - 1) return;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&d_free[d & 1]);
                    ++d;
                };
                auto add = [&](int k, auto piece, const uint32_t (&v)[32]) {  // 32 columns
                    constexpr int C = decltype(piece)::value;
                    const float s = __half2float(__ushort_as_half((uint16_t)scale[k]));
                    const uint64_t s2 = many_pair(s, s);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        total[C * 16 + e] = many_fma(s2, many_pair(v[2 * e], v[2 * e + 1]), total[C * 16 + e]);
                };
                using P0 = std::integral_constant<int, 0>;
                using P1 = std::integral_constant<int, 1>;
                if (COLS == 64 && NG > 1 && plan.n <= 32) {  // two groups, of one D
#pragma unroll
                    for (int k = 0; k < NG; k += 2) {
                        const uint32_t at = take(k);
                        if (!ok) break;
                        uint32_t v[32], u[32];
                        many_ld32(at, v);
                        many_ld32(at + 2 * columns, u);
                        many_wait_ld(v);
                        many_wait_ld(u);
                        add(k, P0(), v);
                        if (NG > 1) add(k + (NG > 1), P0(), u);
                        give(k + 1);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < NG; ++k) {
                        const uint32_t at = take(k);
                        if (!ok) break;
                        auto pieces = [&](auto c) {
                            constexpr int C = decltype(c)::value;
                            using Next = std::integral_constant<int, (C + 1) * 32 < COLS ? C + 1 : 0>;
                            uint32_t v[32];
                            many_ld32(at + C * 32, v);
                            if (COLS == 64) {
                                uint32_t u[32];
                                many_ld32(at + Next::value * 32, u);
                                many_wait_ld(v);
                                many_wait_ld(u);
                                add(k, c, v);
                                add(k, Next(), u);
                            } else {
                                many_wait_ld(v);
                                add(k, c, v);
                                if (Next::value * 32 < plan.n) {
                                    many_ld32(at + Next::value * 32, v);
                                    many_wait_ld(v);
                                    add(k, Next(), v);
                                }
                            }
                        };
                        pieces(P0());
                        if constexpr (COLS == 128) {
                            if (plan.n > 64) pieces(std::integral_constant<int, 2>());
                        }
                        give(k);
                    }
                }
            }
            // Rows of x from the unit's first on, this thread's element of each.
            const int b0 = xt * plan.n, n = min(plan.n, p.batch - b0);
            const bool mine = ok && out < w.rows;
            T* const y = (T*)p.y + b0 * p.y_stride + out;
            const T* const res = COLS == 64 && p.residual ? (const T*)p.residual + b0 * p.residual_stride + out : nullptr;
            float factor[2] = {4.0f, 4.0f};  // of rows lane and lane + 32
            if (SPLIT) {
#pragma unroll
                for (int i = 0; i < 2; ++i) factor[i] = lane + 32 * i < n ? plan.factor[b0 + lane + 32 * i] : 0.0f;
            }
            // W values of rows r(0) .. r(W - 1): what is read comes before what is written.
            auto store = [&](auto width, auto row_of, const float* v) {
                constexpr int W = decltype(width)::value;
                float add[W];
                if (res) {
#pragma unroll
                    for (int i = 0; i < W; ++i) add[i] = mine && row_of(i) < n ? (float)res[row_of(i) * p.residual_stride] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int r = row_of(i);
                    float u = v[i] * 4.0f;
                    if (SPLIT) u *= __shfl_sync(0xffffffffu, r < 32 ? factor[0] : factor[1], r & 31);
                    if (res) u += add[i];
                    if (mine && r < n) y[r * p.y_stride] = (T)u;
                }
            };
            if (cs == 1) {
#pragma unroll
                for (int k = 0; k < PAIRS; k += 8) {
                    if (2 * k >= n) continue;
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 u = many_two(total[k + i]);
                        v[2 * i] = u.x, v[2 * i + 1] = u.y;
                    }
                    store(std::integral_constant<int, 16>(), [&](int i) { return 2 * k + i; }, v);
                }
            } else {
                // Row r of x belongs to CTA (r / 2) % cs: [sender][r / 2 / cs][r % 2][256] in
                // the stages, which nobody needs any more.
                many_cluster_sync();
                const int log2 = plan.cluster_log2, each = ((PAIRS + cs - 1) >> log2) * 2 * kManyRows;  // floats of a sender
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    if (2 * k >= plan.n) continue;
                    const float2 v = many_two(total[k]);
                    uint32_t to;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                 : "=r"(to)
                                 : "r"(smem_u32(smem) + (rank * each + (k >> log2) * 2 * kManyRows + row) * 4), "r"(k & (cs - 1)));
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v.x) : "memory");
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + kManyRows * 4), "f"(v.y) : "memory");
                }
                many_cluster_sync();
                const float* const sums = reinterpret_cast<const float*>(smem) + row;
                for (int k = rank; 2 * k < n; k += 2 * cs) {  // two pairs at a time
                    float v[4] = {};
                    for (int c = 0; c < cs; ++c) {
                        const float* from = sums + c * each + (k >> log2) * 2 * kManyRows;
                        v[0] += from[0], v[1] += from[kManyRows];
                        if (2 * (k + cs) < n) v[2] += from[2 * kManyRows], v[3] += from[3 * kManyRows];
                    }
                    store(std::integral_constant<int, 4>(), [&](int i) { return 2 * (k + (i >> 1) * cs) + (i & 1); }, v);
                }
            }
        }
    }
    // Everyone meets when all products and their arrivals are done, also where
    // a wait has given up.
    if (warp == 16) {
        if (many_elect()) tc_commit(&drained);
        mbar_wait_bounded(&drained, 0, &unset, globaltimer_ns() + timeout_ns, kDevTimeoutDrain);
        if (unset) atomicCAS(err, 0, kDevTimeoutDrain);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 16) tmem_dealloc(tmem, 512);
}

}  // namespace lc
