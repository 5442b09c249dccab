// lc_w4_few.cuh -- products of 4-bit weights with few rows (decode steps).
//
// A warp has 32 rows of W (two tiles, for which x is loaded once) and a part of
// the columns; m16n8k16 products take the weights as f16 numbers (c - z) 2^-6 from
// the words of the layout, exact as every product is: what a zero point takes away
// is gone before anything is rounded.  (Subnormal numbers c 2^-24 would take no
// rotation, but the tensor cores align products by the least normal exponent and
// lose what lies 2^-24 below it: errors of 2^-19 of the sum.)  x stands against them
// as columns: F16 rows as they are, F32 rows as hi and lo under a power-of-two scale
// of the row (of what the CTA has of it), exact to 2^-22.  The sums of a group are
// added under the group's scale to fp32 sums.
//
// Bound by HBM for large matrices, by latency for small ones.  Each warp streams
// its codes, scales and zero points through a ring of its own in shared memory
// (cp.async, no barrier); x lies there once for the CTA.  One, two, four or eight
// warps share a pair of tiles: fewer make fewer meetings, more make the pairs go
// round evenly.  Where a CTA's columns would not fit, or rows are too few to go
// round, a cluster shares them; its CTAs meet in each other's shared memory.  Sums
// are added in a fixed order.  128256 x 2048 for one row: 32.7 us, 21.4 at the
// measured copy's rate, with 152 instructions of a warp for 2048 codes, 72 of them
// for making weights of the codes, and 58 % of the issue slots used (one tile at a
// time and eight warps to a tile: 48 us; the zero points as -z sum x at the
// beginning of a group's sums, whose rounding then goes by the sizes of z x: 34.1).
// Four CTAs of an SM would hide more of their latency; registers are for two.
#pragma once

#include "lc_internal.h"
#include "lc_tcgen05.cuh"
#include "lc_w4.h"

namespace lc {

constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewDepth = 3;  // blocks of a warp's ring
constexpr int kFewMaxCluster = 8;
constexpr int kFewPitch = 24;  // floats between columns of 16 partial sums: no bank conflicts

struct FewPlan {
    int cluster;   // CTAs that share the columns
    int phases;    // parts of a CTA's columns that are taken one after the other
    int split;     // warps that share a pair of tiles
    int blocks;    // of a CTA's part of the columns, at most
    int clusters;
};

template <typename T, int GROUP, int NT>
struct FewShape {
    static constexpr int kRows = sizeof(T) == 4 ? 4 * NT : 8 * NT;  // of x
    static constexpr int kGroups = kW4Cols / GROUP;
    static constexpr int kScaleBytes = 16 * kGroups * 2, kZeroBytes = 16 * kGroups;  // of a tile's block
    static constexpr int kScaleAt = 2 * kW4BlockBytes, kZeroAt = kScaleAt + 2 * kScaleBytes;
    static constexpr int kSlot = kZeroAt + 2 * kZeroBytes;  // a block of two tiles
    static constexpr int kPartFloats = kFewWarps * 2 * kRows * kFewPitch;  // the warps' sums of one meeting
    // Elements of one CTA at a meeting of a cluster, in runs of 16.
    __host__ __device__ static int each(int cluster, int split) { return (kFewWarps / split * 2 * kRows + cluster - 1) / cluster * 16; }
    // rows: of x.  One column of zeros stands for all that are not there.
    static size_t smem(const FewPlan& plan, int rows) {
        const int columns = (sizeof(T) == 4 ? 2 : 1) * rows + 1;
        const size_t blocks = plan.blocks;  // before it is cut into phases a part can have millions
        return (size_t)kFewWarps * kFewDepth * kSlot + columns * (256 * blocks + 64) +
               (1 + kFewWarps) * kRows * 4 + kPartFloats * 4 +
               (plan.cluster > 1 ? 2 * plan.cluster * each(plan.cluster, plan.split) * 4 : 0);
    }
};

constexpr size_t kFewTwo = 113 * 1024, kFewOne = 226 * 1024;  // shared memory with which two CTAs, or one, fit an SM

// How the CTAs share the columns and the pairs of tiles, for `batch` rows of x.
template <typename S>
FewPlan few_plan(const W4& w, int batch, int num_sms) {
    const int pairs = (w.tiles + 1) / 2;
    FewPlan plan;
    auto set = [&](int cluster, int phases) {
        plan.cluster = cluster;
        plan.phases = phases;
        plan.blocks = (w.blocks + cluster * phases - 1) / (cluster * phases);
        // Two CTAs per SM; of clusters an eighth less, for they do not fill a GPC.
        const int most = cluster > 1 ? 2 * num_sms / cluster * 7 / 8 : 2 * num_sms;
        plan.clusters = pairs < most ? pairs : most;
        // Warps of a pair: few make few meetings, more make a CTA's pairs go round
        // evenly.  A meeting costs about as much as kMeet blocks.
        constexpr int kMeet = 2;
        const int mine = (pairs + plan.clusters - 1) / plan.clusters;
        int best = 0;
        for (int split = 1; split <= kFewWarps; split *= 2) {
            const int cost = (mine * split + kFewWarps - 1) / kFewWarps * ((plan.blocks + split - 1) / split + kMeet);
            if (!best || cost < best) best = cost, plan.split = split;
        }
    };
    // More CTAs for the columns while there are SMs without one and each warp has a
    // block, or while a CTA's part keeps a second CTA off the SMs that few pairs leave
    // idle (us with these clusters | without, F32 rows: 8 of 2048 x 8192 13 | 21, 5 of
    // 8192 x 4096 14 | 23; 5 of 4736 x 4096, whose pairs are as many as the SMs, 13 | 12).
    set(1, 1);
    while (plan.cluster < kFewMaxCluster &&
           ((w.blocks >= plan.cluster * kFewWarps && pairs * plan.cluster < num_sms) ||
            (w.blocks >= 2 * plan.cluster * kFewWarps && pairs * plan.cluster < 2 * num_sms && S::smem(plan, batch) > kFewTwo)))
        set(2 * plan.cluster, 1);
    while (S::smem(plan, batch) > kFewOne) set(plan.cluster, plan.phases + 1);
    return plan;
}

LC_DEV uint32_t few_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t v;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(a), "r"(b), "r"(c));
    return v;
}
// The eight weights of a word as f16 pairs (c - z) 2^-6, exact: rows g, g + 8 of
// columns e = 0, 1, then of 2, 3.  Two codes of each half lie where f16 numbers are
// linear in their bits, as c 2^-21 and c 2^-17.  z: -z 2^-6 of the rows.
LC_DEV void few_weights(uint32_t w, const uint32_t (&z)[2], uint32_t (&a)[4]) {
    const uint32_t v = __funnelshift_r(w, w, 8);
    a[0] = few_fma(w & 0x00780078u, 0x78007800u, z[0]);  // 2^15
    a[1] = few_fma(w & 0x07800780u, 0x68006800u, z[1]);  // 2^11
    a[2] = few_fma(v & 0x00780078u, 0x78007800u, z[0]);
    a[3] = few_fma(v & 0x07800780u, 0x68006800u, z[1]);
}
LC_DEV uint32_t few_zero(uint32_t z) {  // -z 2^-6, twice, of a byte up to 15
    uint32_t v;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"((z & 255u) * 0x00800080u), "r"(0xe800e800u));
    return v;
}
LC_DEV void few_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
LC_DEV void few_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
LC_DEV uint4 few_lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

template <typename T, int GROUP, bool ZEROS, int NT>
__global__ void __launch_bounds__(kFewThreads, 2) w4_few_kernel(W4 w, W4Product p, FewPlan plan) {
    using S = FewShape<T, GROUP, NT>;
    constexpr int NG = S::kGroups, ROWS = S::kRows;
    constexpr bool SPLIT = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int pitch = 256 * plan.blocks + 64, columns = (SPLIT ? 2 : 1) * p.batch;
    // Rings, x as f16 columns [columns + 1][pitch], factors [ROWS], largest sizes [warps][ROWS], parts and what a cluster's CTAs send.
    uint8_t* at = smem;
    const uint32_t ring = smem_u32(at) + warp * kFewDepth * S::kSlot;
    at += kFewWarps * kFewDepth * S::kSlot;
    uint8_t* const xcol = at;
    at += (columns + 1) * pitch;
    float* const factor = reinterpret_cast<float*>(at);
    float* const tops = factor + ROWS;
    float* const parts = tops + kFewWarps * ROWS;    // [warps][tile][ROWS][kFewPitch]
    float* const recv = parts + S::kPartFloats;      // [2][cluster][elements of one CTA]

    uint32_t rank = 0;
    const int cs = plan.cluster, id = blockIdx.x / cs;
    if (cs > 1) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    const int pairs = (w.tiles + 1) / 2, PB = kFewWarps / plan.split;  // PB: pairs between two meetings
    const int pair0 = (int)((int64_t)pairs * id / plan.clusters), pair1 = (int)((int64_t)pairs * (id + 1) / plan.clusters);
    const int shares = cs * plan.phases, mine_i = warp / plan.split, mine_k = warp % plan.split;
    auto cta0 = [&](int phase) { return (int)((int64_t)w.blocks * ((int)rank * plan.phases + phase) / shares); };
    auto part = [&](int phase, int k) {  // where the k-th warp of a pair begins
        const int c0 = cta0(phase), c1 = cta0(phase + 1);
        return c0 + (c1 - c0) * k / plan.split;
    };

    // What the warp reads, in order: meetings, phases, blocks.
    // Each lane copies 16 bytes of each half of both tiles' codes, and some 16 bytes
    // of their scales or zero points.
    constexpr int kMetaScales = 2 * S::kScaleBytes / 16, kMeta = kMetaScales + (ZEROS ? 2 * S::kZeroBytes / 16 : 0);
    const bool meta_zero = lane >= kMetaScales;
    const int meta_bytes = meta_zero ? S::kZeroBytes : S::kScaleBytes, meta_at = 16 * (meta_zero ? lane - kMetaScales : lane);
    const uint8_t* const meta_base = meta_zero ? w.zeros : (const uint8_t*)w.scales;
    int a_pair = pair0 + mine_i, a_phase = -1, a_left = 0;
    bool more = true;
    const uint8_t *a_code = nullptr, *a_meta = nullptr;
    int64_t a_second = 0;  // from the first tile's codes to the second's
    auto advance = [&] {   // to the next part that has blocks
        do {
            if (++a_phase == plan.phases) a_phase = 0, a_pair += PB;
            if (a_pair >= pair1) {
                more = false;
                return;
            }
            a_left = part(a_phase, mine_k + 1) - part(a_phase, mine_k);
        } while (!a_left);
        const int tile = 2 * a_pair;
        const bool two = tile + 1 < w.tiles;  // else the first stands for it
        const int64_t u = (int64_t)tile * w.blocks + part(a_phase, mine_k);
        a_code = w.codes + u * kW4BlockBytes + lane * 16;
        a_second = two ? (int64_t)w.blocks * kW4BlockBytes : 0;
        a_meta = meta_base + (u + (two && meta_at >= meta_bytes ? w.blocks : 0)) * meta_bytes + meta_at % meta_bytes;
    };
    auto request = [&](uint32_t to) {
        if (more) {
            few_copy16(to + lane * 16, a_code);
            few_copy16(to + 512 + lane * 16, a_code + 512);
            few_copy16(to + 1024 + lane * 16, a_code + a_second);
            few_copy16(to + 1536 + lane * 16, a_code + a_second + 512);
            if (lane < kMeta) few_copy16(to + S::kScaleAt + lane * 16, a_meta);
            a_code += kW4BlockBytes;
            a_meta += meta_bytes;
            if (--a_left == 0) advance();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    griddep_wait();
    griddep_launch();
    advance();
#pragma unroll
    for (int i = 0; i < kFewDepth - 1; ++i) request(ring + i * S::kSlot);

    // x of the columns [128 b0, 128 b1) as operands.  F32: columns 2 r and 2 r + 1
    // are hi and lo of row r.
    const T* const x = (const T*)p.x;
    const bool vec = ((uintptr_t)x | (uintptr_t)(p.x_stride * sizeof(T))) % (4 * sizeof(T)) == 0;
    auto four = [&](int r, int b, float (&v)[4]) {
        const int c = b * kW4Cols + lane * 4;
        const T* from = x + r * p.x_stride + c;
        if (vec && c + 4 <= w.cols) {
            if (SPLIT) {
                const float4 f = *reinterpret_cast<const float4*>(from);
                v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
            } else {
                const uint2 h = *reinterpret_cast<const uint2*>(from);
                const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
                v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = c + i < w.cols ? (float)from[i] : 0.0f;
        }
    };
    auto stage = [&](int b0, int b1) {  // by all warps
        for (int i = tid * 8; i < pitch; i += kFewThreads * 8) *reinterpret_cast<uint2*>(xcol + columns * pitch + i) = make_uint2(0, 0);
        const int n = b1 - b0;  // a warp has the blocks warp, warp + 8, ... of every row
        auto largest = [&](float top, const float (&u)[4]) {
            return fmaxf(fmaxf(top, fmaxf(fabsf(u[0]), fabsf(u[1]))), fmaxf(fabsf(u[2]), fabsf(u[3])));
        };
        auto put = [&](int r, int b, const float (&f)[4]) {
            const float up = SPLIT ? 1.0f / factor[r] : 1.0f;  // a power of two
            uint32_t h[2], l[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = f[2 * i] * up, c = f[2 * i + 1] * up;
                const __half2 hh = __floats2half2_rn(a, c);
                const float2 hf = __half22float2(hh);
                h[i] = *reinterpret_cast<const uint32_t*>(&hh);
                if (SPLIT) {
                    const __half2 ll = __floats2half2_rn(a - hf.x, c - hf.y);
                    l[i] = *reinterpret_cast<const uint32_t*>(&ll);
                }
            }
            uint8_t* const to = xcol + (SPLIT ? 2 * r : r) * pitch + b * 256 + lane * 8;
            *reinterpret_cast<uint2*>(to) = make_uint2(h[0], h[1]);
            if (SPLIT) *reinterpret_cast<uint2*>(to + pitch) = make_uint2(l[0], l[1]);
        };
        // Several rows are taken four at a time, whose loads are then under way together
        // (8 rows of 2048 x 8192: 17 against 14 us); one alone by two blocks.
        constexpr int TOGETHER = 4;
        const bool rows = p.batch > 1;
        if (SPLIT) {
            if (rows) {
                for (int r0 = 0; r0 < p.batch; r0 += TOGETHER) {
                    float top[TOGETHER] = {};
                    for (int b = warp; b < n; b += kFewWarps) {
                        float u[TOGETHER][4];
#pragma unroll
                        for (int i = 0; i < TOGETHER; ++i)
                            if (r0 + i < p.batch) four(r0 + i, b0 + b, u[i]);
#pragma unroll
                        for (int i = 0; i < TOGETHER; ++i)
                            if (r0 + i < p.batch) top[i] = largest(top[i], u[i]);
                    }
#pragma unroll
                    for (int i = 0; i < TOGETHER; ++i) {
                        if (r0 + i >= p.batch) continue;
                        const float m = warp_max(top[i]);
                        if (lane == 0) tops[warp * ROWS + r0 + i] = m;
                    }
                }
            } else {
                float top = 0.0f;
                for (int b = warp; b < n; b += 2 * kFewWarps) {
                    float u[4], v[4] = {};
                    four(0, b0 + b, u);
                    if (b + kFewWarps < n) four(0, b0 + b + kFewWarps, v);
                    top = largest(largest(top, u), v);
                }
                top = warp_max(top);
                if (lane == 0) tops[warp * ROWS] = top;
            }
            __syncthreads();
        }
        if (tid < ROWS) {
            float f = 1.0f;
            if (SPLIT) {
                float top = 0.0f;
                for (int k = 0; k < kFewWarps && tid < p.batch; ++k) top = fmaxf(top, tops[k * ROWS + tid]);
                f = pow2f(-split_row_exp(top));
            }
            factor[tid] = f;
        }
        if (SPLIT) __syncthreads();
        if (rows) {
            for (int r0 = 0; r0 < p.batch; r0 += TOGETHER) {
                for (int b = warp; b < n; b += kFewWarps) {
                    float f[TOGETHER][4];
#pragma unroll
                    for (int j = 0; j < TOGETHER; ++j)
                        if (r0 + j < p.batch) four(r0 + j, b0 + b, f[j]);
#pragma unroll
                    for (int j = 0; j < TOGETHER; ++j)
                        if (r0 + j < p.batch) put(r0 + j, b, f[j]);
                }
            }
        } else {
            for (int b = warp; b < n; b += kFewWarps) {
                float f[4];
                four(0, b0 + b, f);
                put(0, b, f);
            }
        }
        __syncthreads();
    };

    // Where the lane reads its columns of x.
    uint32_t xat[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xat[nt] = smem_u32(xcol) + min(8 * nt + g, columns) * pitch + t * 16;
    int slot = 0, buf = 0;
    bool staged = false;
    for (int first = pair0; first < pair1; first += PB, buf ^= 1) {
        const int n = min(PB, pair1 - first);
        constexpr int V = SPLIT ? 2 : 4;  // sums of a lane: rows g and g + 8, one or two rows of x
        float* const mine = parts + warp * (2 * ROWS * kFewPitch);
        for (int phase = 0; phase < plan.phases; ++phase) {
            const int c0 = cta0(phase);
            if (phase) __syncthreads();  // all have used the columns of the phase before
            if (!staged || plan.phases > 1) stage(c0, cta0(phase + 1));
            staged = true;
            if (mine_i < n) {
                const int b1 = part(phase, mine_k + 1) - c0;
                float total[2][NT][V] = {};
                for (int b = part(phase, mine_k) - c0; b < b1; ++b) {
                    const uint32_t from = ring + slot * S::kSlot;
                    request(ring + (slot == 0 ? kFewDepth - 1 : slot - 1) * S::kSlot);
                    asm volatile("cp.async.wait_group %0;" ::"n"(kFewDepth - 1) : "memory");
                    __syncwarp();
                    uint4 code[2][2];
                    uint32_t sc[2][NG], zp[2][(NG + 1) / 2];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        code[m][0] = few_lds128(from + m * 1024 + lane * 16);
                        code[m][1] = few_lds128(from + m * 1024 + 512 + lane * 16);
#pragma unroll
                        for (int k = 0; k < NG; ++k)
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(sc[m][k]) : "r"(from + S::kScaleAt + m * S::kScaleBytes + (g * NG + k) * 4));
                        if (ZEROS) {
#pragma unroll
                            for (int k = 0; k < (NG + 1) / 2; ++k) {
                                const uint32_t za = from + S::kZeroAt + m * S::kZeroBytes + (g * NG + 2 * k) * 2;
                                if (NG == 1) {
                                    uint16_t z;
                                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(z) : "r"(za));
                                    zp[m][k] = z;
                                } else {
                                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(zp[m][k]) : "r"(za));
                                }
                            }
                        }
                    }
                    float acc[2][NT][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {  // runs of 32 columns
                        const int k = q / (4 / NG);
                        if (q % (4 / NG) == 0) {
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) acc[m][nt][0] = acc[m][nt][1] = acc[m][nt][2] = acc[m][nt][3] = 0.0f;
                            }
                        }
                        uint4 xb[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) xb[nt] = few_lds128(xat[nt] + b * 256 + q * 64);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint4& c = code[m][q >> 1];
                            uint32_t a0[4], a1[4], z[2] = {0xb000b000u, 0xb000b000u};  // without zero points all are 8
                            if (ZEROS) {
                                const uint32_t both = zp[m][k >> 1] >> (16 * (k & 1));
                                z[0] = few_zero(both), z[1] = few_zero(both >> 8);
                            }
                            few_weights(q & 1 ? c.z : c.x, z, a0);
                            few_weights(q & 1 ? c.w : c.y, z, a1);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                few_mma(acc[m][nt], a0, xb[nt].x, xb[nt].y);
                                few_mma(acc[m][nt], a1, xb[nt].z, xb[nt].w);
                            }
                        }
                        if (q % (4 / NG) == 4 / NG - 1) {
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sc[m][k]));
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    float(&a)[4] = acc[m][nt];
                                    float(&v)[V] = total[m][nt];
                                    if (SPLIT) {
                                        v[0] = fmaf(s.x, a[0] + a[1], v[0]), v[1] = fmaf(s.y, a[2] + a[3], v[1]);
                                    } else {
                                        v[0] = fmaf(s.x, a[0], v[0]), v[1] = fmaf(s.x, a[1], v[1]);
                                        v[V - 2] = fmaf(s.y, a[2], v[V - 2]), v[V - 1] = fmaf(s.y, a[3], v[V - 1]);
                                    }
                                }
                            }
                        }
                    }
                    __syncwarp();  // all lanes have read the slot
                    slot = slot == kFewDepth - 1 ? 0 : slot + 1;
                }
#pragma unroll
                for (int m = 0; m < 2; ++m) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        auto give = [&](int r, float lo, float hi) {  // rows g and g + 8 for row r of x
                            float* const to = mine + (m * ROWS + r) * kFewPitch + g;
                            const float f = factor[r];
                            lo = lo * 64.0f * f, hi = hi * 64.0f * f;
                            to[0] = phase ? to[0] + lo : lo;
                            to[8] = phase ? to[8] + hi : hi;
                        };
                        if (SPLIT) {
                            give(nt * 4 + t, total[m][nt][0], total[m][nt][1]);
                        } else {
                            give(nt * 8 + 2 * t, total[m][nt][0], total[m][nt][V - 2]);
                            give(nt * 8 + 2 * t + 1, total[m][nt][1], total[m][nt][V - 1]);
                        }
                    }
                }
            }
        }
        __syncthreads();
        if (cs > 1 && first == pair0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all have begun
        // The warps' parts in order; a cluster's parts at the CTA that has the element.
        // Element e: row e % 16 of tile e / 16 / ROWS for row (e / 16) % ROWS of x.
        auto finish = [&](int e, float v) {
            const int r = (e >> 4) % ROWS;
            const int64_t out = ((int64_t)first * 2 + (e >> 4) / ROWS) * kW4Rows + (e & 15);
            if (r >= p.batch || out >= w.rows) return;
            if (p.residual) v += (float)((const T*)p.residual)[r * p.residual_stride + out];
            ((T*)p.y)[r * p.y_stride + out] = (T)v;
        };
        const int each = S::each(cs, plan.split);
        for (int e = tid; e < n * 32 * ROWS; e += kFewThreads) {
            constexpr int kPair = 2 * ROWS;  // runs of 16 of a pair
            const float* from = parts + ((e >> 4) / kPair * plan.split * kPair + (e >> 4) % kPair) * kFewPitch + (e & 15);
            float v = from[0];
            for (int k = 1; k < plan.split; ++k) v += from[k * kPair * kFewPitch];
            if (cs == 1) {
                finish(e, v);
            } else {
                uint32_t to;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                             : "=r"(to)
                             : "r"(smem_u32(recv + (buf * cs + (int)rank) * each + ((e >> 4) / cs) * 16 + (e & 15))), "r"((e >> 4) % cs));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
            }
        }
        if (cs > 1) {
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            for (int place = tid; place < each; place += kFewThreads) {
                const int e = ((place >> 4) * cs + (int)rank) * 16 + (place & 15);
                if (e >= n * 32 * ROWS) continue;
                float v = 0.0f;
                for (int k = 0; k < cs; ++k) v += recv[(buf * cs + k) * each + place];
                finish(e, v);
            }
        } else {
            __syncthreads();  // the parts have been read
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace lc
