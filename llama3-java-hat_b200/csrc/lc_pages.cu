// lc_pages.cu -- block tables, slot maps and row positions of one serving
// step, from request lengths, without the host.
//
// Sequences that end (n_new < 0) push their pages on the free stack in
// sequence order; then growing sequences pop the pages they lack from its
// top, again in sequence order.  With prefix sums of the tokens, taken pages
// and returned pages over the sequences, every output is a closed form of the
// inputs, so the CTAs of one cluster share the work without talking: entry i
// of the stack after the pushes is free_list[i] for i < free_count, and past
// that the (i - free_count)-th returned page, read from the ended sequences'
// table rows, which no one writes.
//
// The work is a few dependent reads; latency bounds it.  One cluster (not
// more, so that a cluster barrier can separate all reads of lens and
// free_count from the writes of lens_out and free_count_out, which may be the
// same buffers) of 1 to 16 CTAs.
#include "lc_internal.h"
#include "lc_paged.h"

namespace lc {
namespace {

constexpr int kPagesThreads = 1024;
constexpr int kPerThread = kPagesMaxSeqs / kPagesThreads;

enum PagesStatus : int { kPagesOk = 0, kPagesShort = 1, kPagesRowFull = 2, kPagesCapacity = 3, kPagesBadLength = 4, kPagesBadCount = 5 };

LC_DEV void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The last index s in [lo, hi) with prefix[s] <= i.
LC_DEV int find_owner(const int* prefix, int lo, int hi, int i) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The owners of 32 neighbouring places i0 + lane (up to `last`), given that
// `lo` owns i0 or a place before it: by counting the few borders in between.
LC_DEV int find_owners(const int* prefix, int lo, int n, int i0, int lane, int last) {
    const int border = lo + 1 + lane <= n ? prefix[lo + 1 + lane] : 0x7fffffff;
    const unsigned inside = __ballot_sync(0xffffffffu, border <= last);
    if (inside == 0xffffffffu) return find_owner(prefix, lo, n, min(i0 + lane, last));
    int s = lo;
    for (int e = 0; e < __popc(inside); ++e) s += __shfl_sync(0xffffffffu, border, e) <= i0 + lane;
    return s;
}

__global__ void __launch_bounds__(kPagesThreads) pages_step_kernel(PagesStep p) {
    extern __shared__ int sm[];
    int* tok = sm;                       // [n + 1] tokens before sequence s
    int* take = tok + p.n_seqs + 1;      // [n + 1] pages taken before s
    int* give = take + p.n_seqs + 1;     // [n + 1] pages returned before s
    int* base = give + p.n_seqs + 1;     // [n] lens
    int* top = base + p.n_seqs;          // [n] stack entry of page 0, had it been taken: page pg lies at top - pg
    __shared__ long long warp_sum3[3][32];
    __shared__ unsigned long long bad;
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cta = blockIdx.x, ctas = gridDim.x;
    const int sh = p.page_shift, n = p.n_seqs;
    if (tid == 0) bad = ~0ull;
    __syncthreads();

    // Prefix sums: every thread takes kPerThread neighbouring sequences.
    long long mine[3] = {0, 0, 0};
    int add[kPerThread], len[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
        const int s = tid * kPerThread + k;
        add[k] = len[k] = 0;
        if (s >= n) continue;
        len[k] = p.lens[s];
        add[k] = p.n_new[s];
        const long long h = len[k], before = (h + (1 << sh) - 1) >> sh;
        const long long after = (h + (add[k] > 0 ? add[k] : 0) + (1 << sh) - 1) >> sh;
        if (h < 0) atomicMin(&bad, (0ull << 32) | (unsigned)s);
        else if (after > p.table_stride) atomicMin(&bad, (1ull << 32) | (unsigned)s);
        else if (add[k] < 0) mine[2] += before;
        else mine[0] += add[k], mine[1] += after - before;
    }
    long long sum[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        long long v = mine[q];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        sum[q] = v;
        if (lane == 31) warp_sum3[q][warp] = v;
    }
    const int count = *p.free_count;
    __syncthreads();
    long long total[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        const long long w = warp_sum3[q][lane];
        long long before = lane < warp ? w : 0, all = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        sum[q] += before - mine[q];  // exclusive
        total[q] = all;
    }
    // What is wrong, the gravest first; the same answer in every CTA.
    int code = kPagesOk;
    long long detail = 0;
    const unsigned long long wrong = bad;
    if (count < 0 || count > p.n_pages) code = kPagesBadCount, detail = count;
    else if (wrong != ~0ull) code = (wrong >> 32) ? kPagesRowFull : kPagesBadLength, detail = (int)(wrong & 0xffffffffu);
    else if (total[0] > p.capacity) code = kPagesCapacity, detail = total[0];
    else if (total[1] > count + total[2]) code = kPagesShort, detail = total[1] - count - total[2];
    else if (count + total[2] - total[1] > p.n_pages) code = kPagesBadCount, detail = count + total[2] - total[1];
    if (code == kPagesOk) {
#pragma unroll
        for (int k = 0; k < kPerThread; ++k) {
            const int s = tid * kPerThread + k;
            if (s > n) continue;
            tok[s] = (int)sum[0], take[s] = (int)sum[1], give[s] = (int)sum[2];
            if (s >= n) continue;
            base[s] = len[k];
            const int before = (int)(((long long)len[k] + (1 << sh) - 1) >> sh);
            top[s] = (int)(count + total[2]) - 1 - ((int)sum[1] - before);
            if (add[k] < 0) sum[2] += before;
            else sum[0] += add[k], sum[1] += (int)(((long long)len[k] + add[k] + (1 << sh) - 1) >> sh) - before;
        }
        if (n == kPagesMaxSeqs && tid == kPagesThreads - 1) tok[n] = (int)sum[0], take[n] = (int)sum[1], give[n] = (int)sum[2];
    }
    cluster_sync_all();  // every CTA has read lens and free_count (and its own prefix sums are in place)

    // Sequences of this thread: lens_out and q_start.
    if (cta == 0) {
#pragma unroll
        for (int k = 0; k < kPerThread; ++k) {
            const int s = tid * kPerThread + k;
            if (s < n) {
                p.lens_out[s] = code != kPagesOk ? len[k] : add[k] < 0 ? 0 : len[k] + add[k];
                p.q_start[s] = code != kPagesOk ? 0 : tok[s];
            }
        }
        if (tid == 0) {
            p.q_start[n] = code != kPagesOk ? 0 : tok[n];
            *p.free_count_out = code != kPagesOk ? count : (int)(count + total[2] - total[1]);
            p.status[0] = code;
            p.status[1] = (int)(detail > 0x7fffffff ? 0x7fffffff : detail);
        }
    }
    const int gtid = cta * kPagesThreads + tid, gthreads = ctas * kPagesThreads;
    const int tokens = code != kPagesOk ? 0 : (int)total[0];
    for (int i = tokens + gtid; i < p.capacity; i += gthreads) p.slots[i] = p.positions[i] = p.seq_ids[i] = -1;
    if (code != kPagesOk) return;

    const int held = count + (int)total[2], left = held - (int)total[1];
    auto stack = [&](int i) -> const int32_t* {  // where entry i of the free stack after the pushes lies
        if (i < count) return p.free_list + i;
        i -= count;
        const int s = find_owner(give, 0, n, i);
        return p.table + (long long)s * p.table_stride + (i - give[s]);
    };
    // Tokens: a range of neighbours per warp, 32 at a time, so that an owner is
    // searched once and followed from there (searched for every token, the
    // instructions of that took 30 us of 42 at 177,000 tokens).  Table reads
    // are trips to L2 or HBM: four rounds are under way together.
    const int warps = gthreads >> 5, span = ((tokens + warps - 1) / warps + 31) & ~31;
    const int begin = (gtid >> 5) * span, end = min(tokens, begin + span);
    int owner = begin < end ? find_owner(tok, 0, n, begin) : 0;
    for (int b0 = begin; b0 < end; b0 += 128) {
        int seq[4], pos[4], id[4];
        const int32_t* at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i0 = b0 + k * 32;
            at[k] = p.status;  // any place to read, where there is no token
            if (i0 >= end) continue;  // uniform over the warp
            const int i = min(i0 + lane, end - 1);
            const int s = seq[k] = find_owners(tok, owner, n, i0, lane, min(i0 + 31, end - 1));
            owner = __shfl_sync(0xffffffffu, s, 31);
            pos[k] = base[s] + i - tok[s];
            const int pg = pos[k] >> sh, first_new = (int)(((unsigned)base[s] + (1u << sh) - 1) >> sh);
            at[k] = pg < first_new ? p.table + (long long)s * p.table_stride + pg
                                   : stack(top[s] - pg);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) id[k] = *at[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = b0 + k * 32 + lane;
            if (i >= end) continue;
            p.slots[i] = (id[k] << sh) + (pos[k] & ((1 << sh) - 1));
            p.positions[i] = pos[k];
            p.seq_ids[i] = seq[k];
        }
    }
    // Taken pages into the table, returned pages that stay into the stack.
    for (int a = gtid; a < (int)total[1]; a += gthreads) {
        const int s = find_owner(take, 0, n, a);
        const int first_new = (int)(((long long)base[s] + (1 << sh) - 1) >> sh);
        p.table[(long long)s * p.table_stride + first_new + a - take[s]] = *stack(held - 1 - a);
    }
    for (int i = count + gtid; i < left; i += gthreads) p.free_list[i] = *stack(i);
}

}  // namespace

cudaError_t launch_pages_step(const PagesStep& p, cudaStream_t st) {
    const int smem = (5 * p.n_seqs + 3) * (int)sizeof(int);
    // 48 KB without asking is for these and the kernel's own static arrays
    // (under 1 KB) together.
    if (smem > 47 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(pages_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (5 * kPagesMaxSeqs + 3) * (int)sizeof(int));
        if (e != cudaSuccess) return e;
    }
    // One CTA handles 1024 tokens at a time; more CTAs only where there is a
    // second round of them.  A cluster of 16 is not portable to every device,
    // but to the one this library is built for.
    int ctas = 1;
    while (ctas < 16 && ctas * 2 * kPagesThreads <= p.capacity) ctas *= 2;
    if (ctas > 8) {
        const cudaError_t e = cudaFuncSetAttribute(pages_step_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPagesThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, pages_step_kernel, p);
}

}  // namespace lc
