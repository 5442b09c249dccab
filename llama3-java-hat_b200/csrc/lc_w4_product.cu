// lc_w4_product.cu -- y = x W^T (+ a residual) with 4-bit weights (lc_w4.h).
//
// y[b][r] = sum over groups of s[r][group] * sum over its columns of (c - z) x.
// The inner sums are of whole numbers times x; a group's scale is applied once.
#include "lc_internal.h"
#include "lc_w4.h"
#include "lc_w4_few.cuh"

#ifndef FEW_MEET
#define FEW_MEET 2
#endif
namespace lc {
namespace {

// Rows of x that one launch of the kernel for few rows takes.
constexpr int few_rows(int dtype) { return dtype == kRowF32 ? 8 : 16; }

template <typename T, int GROUP, bool ZEROS, int NT>
cudaError_t few_as(const W4& w, const W4Product& p, int num_sms, cudaStream_t st) {
    using S = FewShape<T, GROUP, NT>;
    constexpr size_t kTwo = 113 * 1024, kOne = 226 * 1024;  // shared memory with which two CTAs, or one, fit an SM
    const int pairs = (w.tiles + 1) / 2;
    FewPlan plan;
    auto set = [&](int cluster, int phases) {
        plan.cluster = cluster;
        plan.phases = phases;
        plan.blocks = (w.blocks + cluster * phases - 1) / (cluster * phases);
        const int most = 2 * num_sms / cluster;
        plan.clusters = pairs < most ? pairs : most;
        // Warps of a pair: few make few meetings, more make a CTA's pairs go round
        // evenly.  A meeting costs about as much as kMeet blocks.
        constexpr int kMeet = FEW_MEET;
        const int mine = (pairs + plan.clusters - 1) / plan.clusters;
        int best = 0;
        for (int split = 1; split <= kFewWarps; split *= 2) {
            const int cost = (mine * split + kFewWarps - 1) / kFewWarps * ((plan.blocks + split - 1) / split + kMeet);
            if (!best || cost < best) best = cost, plan.split = split;
        }
    };
    // More CTAs for the columns while a CTA's part would keep a second CTA off the
    // SM, or while there are SMs without one and each warp has two blocks to share.
    set(1, 1);
    while (plan.cluster < kFewMaxCluster && w.blocks >= 2 * plan.cluster * kFewWarps &&
           (S::smem(plan, p.batch) > kTwo || pairs * plan.cluster < num_sms))
        set(2 * plan.cluster, 1);
    while (S::smem(plan, p.batch) > kOne) set(plan.cluster, plan.phases + 1);
    auto* kernel = w4_few_kernel<T, GROUP, ZEROS, NT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kOne);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.clusters * plan.cluster));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = S::smem(plan, p.batch);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)plan.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, w, p, plan);
}

template <typename T, int GROUP, bool ZEROS>
cudaError_t few(const W4& w, const W4Product& p, int num_sms, cudaStream_t st) {
    const int tiles = (p.batch * (sizeof(T) == 4 ? 2 : 1) + 7) / 8;  // of eight columns
    return tiles <= 1   ? few_as<T, GROUP, ZEROS, 1>(w, p, num_sms, st)
                        : few_as<T, GROUP, ZEROS, 2>(w, p, num_sms, st);
}

template <typename T, int GROUP>
cudaError_t product(const W4& w, const W4Product& p, int num_sms, cudaStream_t st) {
    return w.zeros ? few<T, GROUP, true>(w, p, num_sms, st) : few<T, GROUP, false>(w, p, num_sms, st);
}

}  // namespace

cudaError_t launch_w4_product(const W4& w, const W4Product& all, int num_sms, cudaStream_t st) {
    const int elem = all.dtype == kRowF32 ? 4 : 2;
    for (int r = 0; r < all.batch; r += few_rows(all.dtype)) {
        W4Product p = all;
        p.batch = all.batch - r < few_rows(all.dtype) ? all.batch - r : few_rows(all.dtype);
        p.x = (const uint8_t*)all.x + r * all.x_stride * elem;
        p.y = (uint8_t*)all.y + r * all.y_stride * elem;
        if (all.residual) p.residual = (const uint8_t*)all.residual + r * all.residual_stride * elem;
        const bool f32 = p.dtype == kRowF32;
        const cudaError_t e = w.group == 32   ? (f32 ? product<float, 32>(w, p, num_sms, st) : product<__half, 32>(w, p, num_sms, st))
                              : w.group == 64 ? (f32 ? product<float, 64>(w, p, num_sms, st) : product<__half, 64>(w, p, num_sms, st))
                                              : (f32 ? product<float, 128>(w, p, num_sms, st) : product<__half, 128>(w, p, num_sms, st));
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace lc
