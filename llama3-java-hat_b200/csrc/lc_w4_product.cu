// lc_w4_product.cu -- y = x W^T (+ a residual) with 4-bit weights (lc_w4.h).
//
// y[b][r] = sum over groups of s[r][group] * sum over its columns of (c - z) x.
// The inner sums are of whole numbers times x; a group's scale is applied once, to
// them.  Two kernels: lc_w4_few.cuh and lc_w4_many.cuh.
#include "lc_internal.h"
#include "lc_w4.h"
#include "lc_w4_few.cuh"
#include "lc_w4_many.cuh"

namespace lc {
namespace {

// Rows of x that one launch of the kernel for few rows takes.
constexpr int few_rows(int dtype) { return dtype == kRowF32 ? 8 : 16; }

template <typename T, int GROUP, bool ZEROS, int NT>
cudaError_t few_as(const W4& w, const W4Product& p, int num_sms, cudaStream_t st) {
    const FewPlan plan = few_plan<FewShape<T, GROUP, NT>>(w, p.batch, num_sms);
    auto* kernel = w4_few_kernel<T, GROUP, ZEROS, NT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewOne);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.clusters * plan.cluster));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = FewShape<T, GROUP, NT>::smem(plan, p.batch);
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

// Rows of x that one pass through the workspace takes, whole units of them: 0 where
// not even one unit fits.
constexpr size_t kLayBytes = 32u << 20, kFactorBytes = 1u << 20;
int64_t many_rows(const W4& w, bool split) {
    const int64_t unit = many_most(split), fit = (int64_t)(kLayBytes / ((size_t)w.blocks * kW4Cols * (split ? 4 : 2))) / unit * unit;
    return fit < (int64_t)(kFactorBytes / 4) ? fit : (int64_t)(kFactorBytes / 4);
}

template <typename T, int GROUP, bool ZEROS>
cudaError_t many(const W4& w, const W4Product& p, int num_sms, void* ws, int* err, cudaStream_t st) {
    constexpr int HALVES = sizeof(T) == 4 ? 2 : 1;
    // Units of 128 rows for F16 prompts, whose products then set the pace, not the
    // codes: 2048 rows of 16384 x 2048, us in units of 128 | 64 rows: groups of 128 208
    // | 245, of 64 274 | 300, of 32 433 | 406; 386 rows of 5742 x 1024 21 | 27, 100 rows
    // of 16384 x 2048 24 | 20; with a residual 128 rows of it 47 | 27, for there are no
    // registers for it next to the sums (2048 rows with one: 285 in units of 64).
    constexpr bool CAN = sizeof(T) == 2 && GROUP >= 64;
    const int most = CAN && p.batch > 256 && !p.residual ? many_most(false) : 64;
    ManyPlan plan;
    plan.x_tiles = (p.batch + most - 1) / most;
    plan.n = ((p.batch + plan.x_tiles - 1) / plan.x_tiles + 15) / 16 * 16;
    plan.w_tiles = (w.rows + kManyRows - 1) / kManyRows;
    plan.b = (const uint8_t*)ws;
    plan.factor = (const float*)((uint8_t*)ws + kLayBytes);
    // Groups of a D share 64 columns of tensor memory (128 where A is not there) for
    // each 128 rows of W, 32 of them at least.
    constexpr int NG = kW4Cols / GROUP;
    const bool big = plan.n > 64;
    plan.sets = NG / (!big && plan.n <= 32 && NG >= 2 ? 2 : 1);
    const int spare = (kManySmem - kManyStages * ((big ? kManyABytes : 0) + HALVES * plan.n * kManyK * 2)) / (8 * kManyRingBytes);
    plan.ring = spare < kManyMaxRing ? spare : kManyMaxRing;
    // CTAs of a unit: what its CTAs and the units that come after one another take, in
    // blocks; a unit's beginning and end cost about four.
    const int64_t units = (int64_t)plan.x_tiles * plan.w_tiles;
    int64_t best = 0;
    for (int cs = 1; cs <= kManyMaxCluster && cs <= w.blocks; cs *= 2) {
        const int64_t cost = (units * cs + num_sms - 1) / num_sms * ((w.blocks + cs - 1) / cs + 4);
        if (!best || cost < best) best = cost, plan.cluster = cs;
    }
    for (plan.cluster_log2 = 0; 1 << plan.cluster_log2 < plan.cluster;) ++plan.cluster_log2;
    cudaError_t e = launch_ex(w4_lay_kernel<T>, dim3((unsigned)(plan.x_tiles * (plan.n / 8))), dim3(kLayThreads), 0, st, true, p, w.cols,
                              w.blocks, plan, (uint8_t*)ws, (float*)((uint8_t*)ws + kLayBytes));
    if (e != cudaSuccess) return e;
    auto* kernel = w4_many_kernel<T, GROUP, ZEROS, 64>;
    if constexpr (CAN) {
        if (big) kernel = w4_many_kernel<T, GROUP, ZEROS, many_most(false)>;
    }
    // The register split draws on what the launch has: more than that would wait forever.
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) return e;
    if (attr.numRegs < ManyRegs<true>::kLaunch || attr.numRegs < ManyRegs<false>::kLaunch) return cudaErrorInvalidKernelImage;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kManySmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    const int64_t ctas = plan.cluster > 1 ? units * plan.cluster : units < num_sms ? units : num_sms;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kManyThreads);
    cfg.dynamicSmemBytes = kManySmem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)plan.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, w, p, plan, err, (uint64_t)2000000000ull);
}

template <typename T, int GROUP, bool ZEROS>
cudaError_t product_as(const W4& w, const W4Product& all, int num_sms, void* ws, int* err, cudaStream_t st) {
    const int64_t step = ws ? many_rows(w, sizeof(T) == 4) : few_rows(all.dtype);
    for (int64_t r = 0; r < all.batch; r += step) {
        W4Product p = all;
        p.batch = (int)(all.batch - r < step ? all.batch - r : step);
        p.x = (const T*)all.x + r * all.x_stride;
        p.y = (T*)all.y + r * all.y_stride;
        if (all.residual) p.residual = (const T*)all.residual + r * all.residual_stride;
        const cudaError_t e = ws ? many<T, GROUP, ZEROS>(w, p, num_sms, ws, err, st) : few<T, GROUP, ZEROS>(w, p, num_sms, st);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <typename T, int GROUP>
cudaError_t product(const W4& w, const W4Product& p, int num_sms, void* ws, int* err, cudaStream_t st) {
    return w.zeros ? product_as<T, GROUP, true>(w, p, num_sms, ws, err, st) : product_as<T, GROUP, false>(w, p, num_sms, ws, err, st);
}
template <typename T>
cudaError_t product(const W4& w, const W4Product& p, int num_sms, void* ws, int* err, cudaStream_t st) {
    return w.group == 32   ? product<T, 32>(w, p, num_sms, ws, err, st)
           : w.group == 64 ? product<T, 64>(w, p, num_sms, ws, err, st)
                           : product<T, 128>(w, p, num_sms, ws, err, st);
}

}  // namespace

// Rows beyond one column tile of the kernel for few (4 F32 rows, 8 F16 rows) go
// through the tensor cores of the other where matrices have the rows to keep all SMs
// busy, and F16 rows of the smaller ones beyond 12.  us, few | many, groups of 128:
//   128256 x 2048  5 F32 46 | 62, 8 F32 60 | 62, 9 F16 68 | 59, 16 F16 77 | 60
//   16384 x 2048   5 F32 13 | 14, 8 F32 21 | 14, 9 F16 22 | 13, 16 F16 27 | 13
//   2048 x 8192    5 F32 11 | 26, 8 F32 13 | 27, 9 F16 12 | 20, 16 F16 29 | 19
//   2048 x 2048    5 F32  8 | 10, 8 F32  8 | 10, 9 F16  8 | 9,  16 F16  9 | 9
bool w4_product_uses_ws(const W4& w, const W4Product& p, int num_sms) {
    const bool f32 = p.dtype == kRowF32;
    if (p.batch <= few_rows(p.dtype) / 2 || many_rows(w, f32) == 0) return false;
    if (p.batch > (f32 ? 8 : 12)) return true;
    const int pairs = (w.tiles + 1) / 2;
    return !(pairs < num_sms || (f32 && pairs >= 8 * num_sms));
}
size_t w4_product_ws_bytes() { return kLayBytes + kFactorBytes; }

cudaError_t launch_w4_product(const W4& w, const W4Product& p, int num_sms, void* ws, int* err, cudaStream_t st) {
    return p.dtype == kRowF32 ? product<float>(w, p, num_sms, ws, err, st) : product<__half>(w, p, num_sms, ws, err, st);
}

}  // namespace lc
