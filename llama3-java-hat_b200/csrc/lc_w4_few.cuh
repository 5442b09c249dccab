// lc_w4_few.cuh -- products of 4-bit weights with few rows (decode steps).
//
// A warp has 16 rows of W and a part of the columns; m16n8k16 products take the
// codes as f16 numbers c 2^-17 straight from the words of the layout (exact, and so
// is every product; as c 2^-24, which takes five instructions instead of seven for
// eight codes, the tensor cores align products by the least normal exponent and
// lose what lies 2^-24 below it: errors 2^-19 of the sum) against x as columns: F16 rows as they are, F32 rows as two columns
// hi and lo under a power-of-two scale of the row (of what the warp has of it),
// exact to 2^-22.  The sums of a group begin at -z sum x, and are added under the
// group's scale to fp32 sums.
//
// Bound by HBM for large matrices, by latency for small ones.  Each warp streams
// its codes, scales and zero points through a ring of its own in shared memory
// (cp.async, no barrier), and makes the operands of its columns itself, so warps
// meet only where the eight parts of a tile are added.  Where a CTA's columns
// would not fit, or rows are too few to go round, a cluster shares them; its CTAs
// meet in each other's shared memory.  Sums are added in a fixed order.
#pragma once

#include "lc_internal.h"
#include "lc_tcgen05.cuh"
#include "lc_w4.h"

namespace lc {

constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewDepth = 4;  // blocks of a warp's ring
constexpr int kFewMaxCluster = 8;
constexpr int kFewPitch = 24;  // floats between columns of 16 partial sums: no bank conflicts

template <typename T, int GROUP, int NT>
struct FewShape {
    static constexpr int kRows = sizeof(T) == 4 ? 4 * NT : 8 * NT;  // of x
    static constexpr int kGroups = kW4Cols / GROUP;
    static constexpr int kScaleBytes = 16 * kGroups * 2, kZeroBytes = 16 * kGroups;
    static constexpr int kSlot = kW4BlockBytes + 128 + 64;
    static constexpr int kTiles = kRows >= 16 ? 1 : 16 / kRows;  // tiles between two meetings
    static constexpr int kElems = kTiles * kRows * 16;
    static constexpr int kPartBytes = 2 * kFewWarps * kTiles * kRows * kFewPitch * 4;
    static constexpr int kRecvBytes = 2 * (kElems + 16 * kFewMaxCluster) * 4;
    static int x_pitch(int blocks) { return 256 * blocks + 64; }
    static size_t smem(int blocks) {  // blocks: of a warp's part
        return (size_t)kFewWarps * (kFewDepth * kSlot + 8 * NT * x_pitch(blocks) + (blocks * kGroups + 1) * kRows * 4) + kPartBytes + kRecvBytes;
    }
};

struct FewPlan {
    int cluster, phases, blocks;  // CTAs that share the columns; parts of a warp one after the other; blocks of a part at most
    int clusters;
};

// The eight codes of a word as f16 pairs c 2^-17: rows g, g + 8 of columns e = 0, 1,
// then of 2, 3.
LC_DEV void few_codes(uint32_t w, uint32_t (&a)[4]) {
    constexpr uint32_t kMask = 0x07800780u;
    a[0] = __funnelshift_l(w, w, 4) & kMask;
    a[1] = w & kMask;
    a[2] = __funnelshift_r(w, w, 4) & kMask;
    a[3] = __funnelshift_r(w, w, 8) & kMask;
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
    constexpr int NG = S::kGroups, ROWS = S::kRows, TB = S::kTiles;
    constexpr bool SPLIT = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int pitch = 256 * plan.blocks + 64;
    // Of this warp: ring, x as f16 columns [8 NT][pitch], sums of x [groups][ROWS], factors [ROWS].
    uint8_t* at = smem;
    const uint32_t ring = smem_u32(at) + warp * kFewDepth * S::kSlot;
    at += kFewWarps * kFewDepth * S::kSlot;
    uint8_t* const xcol = at + warp * 8 * NT * pitch;
    at += kFewWarps * 8 * NT * pitch;
    float* const xsum = reinterpret_cast<float*>(at) + warp * (plan.blocks * NG + 1) * ROWS;
    float* const factor = xsum + plan.blocks * NG * ROWS;
    at += kFewWarps * (plan.blocks * NG + 1) * ROWS * 4;
    float* const parts = reinterpret_cast<float*>(at);  // [2][warps][TB][ROWS][kFewPitch]
    at += S::kPartBytes;
    float* const recv = reinterpret_cast<float*>(at);   // [2][cluster][elements of one CTA]

    uint32_t rank = 0;
    const int cs = plan.cluster, id = blockIdx.x / cs;
    if (cs > 1) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    const int tile0 = (int)((int64_t)w.tiles * id / plan.clusters), tile1 = (int)((int64_t)w.tiles * (id + 1) / plan.clusters);
    const int shares = cs * plan.phases * kFewWarps;
    auto part0 = [&](int phase) { return (int)((int64_t)w.blocks * (((int)rank * plan.phases + phase) * kFewWarps + warp) / shares); };
    auto part1 = [&](int phase) { return (int)((int64_t)w.blocks * (((int)rank * plan.phases + phase) * kFewWarps + warp + 1) / shares); };

    // What the warp reads, in order: batches of TB tiles, phases, tiles, blocks.
    struct Cursor {
        int batch, phase, i, block, end, n;  // n: tiles of the batch
    };
    auto open = [&](Cursor& c) {  // the first block at or behind (batch, phase, i = 0); false: none
        for (; c.batch < tile1; c.batch += TB, c.phase = 0) {
            for (; c.phase < plan.phases; ++c.phase) {
                c.block = part0(c.phase), c.end = part1(c.phase);
                c.n = min(TB, tile1 - c.batch);
                c.i = 0;
                if (c.block < c.end) return true;
            }
        }
        return false;
    };
    Cursor ahead = {tile0, 0, 0, 0, 0, 0};
    bool more = open(ahead);
    auto request = [&](int slot) {
        if (more) {
            const int64_t u = (int64_t)(ahead.batch + ahead.i) * w.blocks + ahead.block;
            const uint32_t to = ring + slot * S::kSlot;
            const uint8_t* from = w.codes + u * kW4BlockBytes + lane * 16;
            few_copy16(to + lane * 16, from);
            few_copy16(to + 512 + lane * 16, from + 512);
            if (lane < S::kScaleBytes / 16) few_copy16(to + 1024 + lane * 16, (const uint8_t*)w.scales + u * S::kScaleBytes + lane * 16);
            if (ZEROS && lane >= 16 && lane < 16 + S::kZeroBytes / 16)
                few_copy16(to + 1152 + (lane - 16) * 16, w.zeros + u * S::kZeroBytes + (lane - 16) * 16);
            if (++ahead.block == ahead.end) {
                if (++ahead.i < ahead.n) {
                    ahead.block = part0(ahead.phase);
                } else {
                    ++ahead.phase;
                    more = open(ahead);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    griddep_wait();
    griddep_launch();
#pragma unroll
    for (int i = 0; i < kFewDepth - 1; ++i) request(i);

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
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), b2 = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
                v[0] = a.x, v[1] = a.y, v[2] = b2.x, v[3] = b2.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = c + i < w.cols ? (float)from[i] : 0.0f;
        }
    };
    auto stage = [&](int b0, int b1) {
        constexpr float kSum = ZEROS ? -0x1p-17f : -0x1p-14f;  // without zero points all are 8
        __syncwarp();
        for (int r = 0; r < ROWS; ++r) {
            if (r >= p.batch) {
                for (int b = 0; b < b1 - b0; ++b) {
                    const uint2 none = make_uint2(0, 0);
                    *reinterpret_cast<uint2*>(xcol + (SPLIT ? 2 * r : r) * pitch + b * 256 + lane * 8) = none;
                    if (SPLIT) *reinterpret_cast<uint2*>(xcol + (2 * r + 1) * pitch + b * 256 + lane * 8) = none;
                    for (int i = lane; i < NG; i += 32) xsum[(b * NG + i) * ROWS + r] = 0.0f;
                }
                if (lane == 0) factor[r] = 0.0f;
                continue;
            }
            constexpr int HOLD = 4;  // blocks that are read once
            float v[HOLD][4], up = 1.0f;
            if (SPLIT) {
                float top = 0.0f;
                for (int b = b1 - 1; b >= b0; --b) {
                    float u[4];
                    if (b - b0 >= HOLD) {
                        four(r, b, u);
                        top = fmaxf(fmaxf(top, fmaxf(fabsf(u[0]), fabsf(u[1]))), fmaxf(fabsf(u[2]), fabsf(u[3])));
                    }
                }
#pragma unroll
                for (int b = 0; b < HOLD; ++b) {
                    if (b0 + b < b1) {
                        four(r, b0 + b, v[b]);
                        top = fmaxf(fmaxf(top, fmaxf(fabsf(v[b][0]), fabsf(v[b][1]))), fmaxf(fabsf(v[b][2]), fabsf(v[b][3])));
                    }
                }
                const int e = split_row_exp(warp_max(top));
                up = pow2f(e);
                if (lane == 0) factor[r] = pow2f(-e);
            } else {
#pragma unroll
                for (int b = 0; b < HOLD; ++b)
                    if (b0 + b < b1) four(r, b0 + b, v[b]);
                if (lane == 0) factor[r] = 1.0f;
            }
            auto put = [&](int b, float (&f)[4]) {
                uint32_t h[2], l[2];
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = f[2 * i] * up, c = f[2 * i + 1] * up;
                    const __half2 hh = __floats2half2_rn(a, c);
                    const float2 hf = __half22float2(hh);
                    h[i] = *reinterpret_cast<const uint32_t*>(&hh);
                    sum += hf.x + hf.y;
                    if (SPLIT) {
                        const __half2 ll = __floats2half2_rn(a - hf.x, c - hf.y);
                        const float2 lf = __half22float2(ll);
                        l[i] = *reinterpret_cast<const uint32_t*>(&ll);
                        sum += lf.x + lf.y;
                    }
                }
                uint8_t* const to = xcol + (SPLIT ? 2 * r : r) * pitch + b * 256 + lane * 8;
                *reinterpret_cast<uint2*>(to) = make_uint2(h[0], h[1]);
                if (SPLIT) *reinterpret_cast<uint2*>(to + pitch) = make_uint2(l[0], l[1]);
#pragma unroll
                for (int o = 1; o < GROUP / 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane % (GROUP / 4) == 0) xsum[(b * NG + lane / (GROUP / 4)) * ROWS + r] = sum * kSum;
            };
#pragma unroll
            for (int b = 0; b < HOLD; ++b)
                if (b0 + b < b1) put(b, v[b]);
            for (int b = HOLD; b < b1 - b0; ++b) {
                float u[4];
                four(r, b0 + b, u);
                put(b, u);
            }
        }
        __syncwarp();
    };

    int slot = 0, buf = 0;
    bool staged = false;
    for (int batch = tile0; batch < tile1; batch += TB, buf ^= 1) {
        const int n = min(TB, tile1 - batch);
        float* const mine = parts + ((buf * kFewWarps + warp) * TB) * ROWS * kFewPitch;
        for (int phase = 0; phase < plan.phases; ++phase) {
            const int b0 = part0(phase), b1 = part1(phase);
            if (!staged || plan.phases > 1) stage(b0, b1);
            staged = true;
            for (int i = 0; i < n; ++i) {
                constexpr int V = SPLIT ? 2 : 4;  // sums of a lane: rows g and g + 8, one or two rows of x
                float total[NT][V] = {};
                for (int b = b0; b < b1; ++b) {
                    request(slot == 0 ? kFewDepth - 1 : slot - 1);
                    asm volatile("cp.async.wait_group %0;" ::"n"(kFewDepth - 1) : "memory");
                    __syncwarp();
                    const uint32_t from = ring + slot * S::kSlot;
                    const uint32_t xat = smem_u32(xcol) + g * pitch + (b - b0) * 256 + t * 16;
                    const float* const xs = xsum + (b - b0) * NG * ROWS;
                    uint4 code[2] = {few_lds128(from + lane * 16), few_lds128(from + 512 + lane * 16)};
                    uint32_t sc[NG], zp[(NG + 1) / 2];
#pragma unroll
                    for (int k = 0; k < NG; ++k) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(sc[k]) : "r"(from + 1024 + (g * NG + k) * 4));
                    if (ZEROS) {
#pragma unroll
                        for (int k = 0; k < (NG + 1) / 2; ++k) {
                            if (NG == 1) {
                                uint16_t z;
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(z) : "r"(from + 1152 + g * 2));
                                zp[k] = z;
                            } else {
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(zp[k]) : "r"(from + 1152 + (g * NG + 2 * k) * 2));
                            }
                        }
                    }
                    float acc[NT][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {  // runs of 32 columns
                        if (q % (4 / NG) == 0) {
                            const int k = q / (4 / NG);
                            float z0 = 1.0f, z1 = 1.0f;
                            if (ZEROS) {
                                const uint32_t z = zp[k >> 1] >> (16 * (k & 1));
                                z0 = (float)(z & 255u), z1 = (float)((z >> 8) & 255u);
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (SPLIT) {
                                    const float a = xs[k * ROWS + nt * 4 + t];
                                    acc[nt][0] = z0 * a, acc[nt][1] = 0.0f, acc[nt][2] = z1 * a, acc[nt][3] = 0.0f;
                                } else {
                                    const float2 a = *reinterpret_cast<const float2*>(xs + k * ROWS + nt * 8 + 2 * t);
                                    acc[nt][0] = z0 * a.x, acc[nt][1] = z0 * a.y, acc[nt][2] = z1 * a.x, acc[nt][3] = z1 * a.y;
                                }
                            }
                        }
                        const uint4& c = code[q >> 1];
                        const uint32_t w0 = q & 1 ? c.z : c.x, w1 = q & 1 ? c.w : c.y;
                        uint32_t a0[4], a1[4];
                        few_codes(w0, a0);
                        few_codes(w1, a1);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint4 xb = few_lds128(xat + nt * 8 * pitch + q * 64);
                            few_mma(acc[nt], a0, xb.x, xb.y);
                            few_mma(acc[nt], a1, xb.z, xb.w);
                        }
                        if (q % (4 / NG) == 4 / NG - 1) {
                            const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sc[q / (4 / NG)]));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (SPLIT) {
                                    total[nt][0] = fmaf(s.x, acc[nt][0] + acc[nt][1], total[nt][0]);
                                    total[nt][1] = fmaf(s.y, acc[nt][2] + acc[nt][3], total[nt][1]);
                                } else {
                                    total[nt][0] = fmaf(s.x, acc[nt][0], total[nt][0]);
                                    total[nt][1] = fmaf(s.x, acc[nt][1], total[nt][1]);
                                    total[nt][V - 2] = fmaf(s.y, acc[nt][2], total[nt][V - 2]);
                                    total[nt][V - 1] = fmaf(s.y, acc[nt][3], total[nt][V - 1]);
                                }
                            }
                        }
                    }
                    __syncwarp();  // all lanes have read the slot
                    slot = slot == kFewDepth - 1 ? 0 : slot + 1;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    auto give = [&](int r, float lo, float hi) {  // rows g and g + 8 for row r of x
                        float* const to = mine + (i * ROWS + r) * kFewPitch + g;
                        const float f = factor[r];
                        lo = lo * 0x1p17f * f, hi = hi * 0x1p17f * f;
                        to[0] = phase ? to[0] + lo : lo;
                        to[8] = phase ? to[8] + hi : hi;
                    };
                    if (SPLIT) {
                        give(nt * 4 + t, total[nt][0], total[nt][1]);
                    } else {
                        give(nt * 8 + 2 * t, total[nt][0], total[nt][V - 2]);
                        give(nt * 8 + 2 * t + 1, total[nt][1], total[nt][V - 1]);
                    }
                }
            }
        }
        __syncthreads();
        if (cs > 1 && batch == tile0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all have begun
        // The warps' parts in order; a cluster's parts at the CTA that has the element.
        auto element = [&](int e, int& i, int& r, int& row) { row = e & 15, r = (e >> 4) % ROWS, i = (e >> 4) / ROWS; };
        auto finish = [&](int e, float v) {
            int i, r, row;
            element(e, i, r, row);
            const int64_t out = (int64_t)(batch + i) * kW4Rows + row;
            if (i >= n || r >= p.batch || out >= w.rows) return;
            if (p.residual) v += (float)((const T*)p.residual)[r * p.residual_stride + out];
            ((T*)p.y)[r * p.y_stride + out] = (T)v;
        };
        for (int e = tid; e < S::kElems; e += kFewThreads) {
            int i, r, row;
            element(e, i, r, row);
            if (i >= n) continue;
            const float* from = parts + (buf * kFewWarps * TB + i) * ROWS * kFewPitch + r * kFewPitch + row;
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < kFewWarps; ++k) v += from[k * TB * ROWS * kFewPitch];
            if (cs == 1) {
                finish(e, v);
            } else {
                // 16 neighbouring elements have one owner.
                const int owner = (e >> 4) % cs, place = ((e >> 4) / cs) * 16 + (e & 15);
                const int each = ((S::kElems / 16 + cs - 1) / cs) * 16;
                uint32_t to;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(recv + (buf * cs + (int)rank) * each + place)), "r"(owner));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
            }
        }
        if (cs > 1) {
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            const int each = ((S::kElems / 16 + cs - 1) / cs) * 16;
            for (int place = tid; place < each; place += kFewThreads) {
                const int e = ((place >> 4) * cs + (int)rank) * 16 + (place & 15);
                if (e >= S::kElems || (e >> 4) / ROWS >= n) continue;
                float v = 0.0f;
                for (int k = 0; k < cs; ++k) v += recv[(buf * cs + k) * each + place];
                finish(e, v);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace lc
