// lc_kv8.cu -- writing rows into the 8-bit pages and reading them back.
//
// Append.  A unit is the runs (neighbouring rows with consecutive slots) of one
// page, for one kv head, keys or values.  With s the page's scale (0 when the
// run starts the page) the new scale is s' = max(s, max |x| / limit); the codes
// that the page holds below the run become round(c s / s') when s' > s, and the
// run's are round(x / s').  Each rounding is to the nearest code of the exact
// quotient, so a value is within half a code step of what was stored before,
// whatever order the tokens came in.  One warp per unit: no sums, and no
// order in which anything is added.
#include "lc_internal.h"
#include "lc_kv8.cuh"

namespace lc {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWindow = 32;  // rows whose slots one CTA looks at

template <typename T>
LC_DEV float row_value(const T* p) { return (float)*p; }
template <>
LC_DEV float row_value<__half>(const __half* p) { return __half2float(*p); }

template <typename T, int FMT>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(Kv8 c, Kv8Rows r) {
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sh = c.page_shift, page = 1 << sh, d = c.head_dim;
    const int64_t n_slots = (int64_t)c.n_pages << sh;
    const int row0 = blockIdx.x * kAppendWindow;
    // Lane i: is row row0 + i the first of its page's rows?  Rows without a
    // slot are passed over.
    const int my = row0 + lane;
    auto slot_of = [&](int i) {
        const int v = r.slots[i];
        return v >= 0 && v < n_slots ? v : -1;
    };
    int slot = -1;
    bool starts = false;
    if (my < r.rows) {
        slot = slot_of(my);
        if (slot >= 0) {
            int i = my - 1, prev = -1;
            while (i >= 0 && (prev = slot_of(i)) < 0) --i;
            starts = prev < 0 || (prev >> sh) != (slot >> sh);
        }
    }
    unsigned starters = __ballot_sync(0xffffffffu, starts);
    int n = 0;  // unit number within the CTA
    while (starters) {
        const int l = __ffs(starters) - 1;
        starters &= starters - 1;
        const int pg = __shfl_sync(0xffffffffu, slot, l) >> sh;
        for (int u = 0; u < 2 * c.n_kv; ++u, ++n) {
            if (n % (kAppendThreads / 32) != warp) continue;
            const int head = u >> 1;
            const T* rows = (const T*)((u & 1) ? r.v : r.k) + head * d;
            uint8_t* codes = ((u & 1) ? c.v : c.k) + ((((int64_t)pg * c.n_kv + head) << sh) * d);
            float* scale = ((u & 1) ? c.v_scale : c.k_scale) + (int64_t)pg * c.n_kv + head;
            float held = *scale;
            // The page's runs, one after the other: usually there is one.
            for (int row = row0 + l; row < r.rows;) {
                const int first = slot_of(row);
                if (first < 0) {
                    ++row;
                    continue;
                }
                if ((first >> sh) != pg) break;
                const int off = first & (page - 1);
                int len = 1;  // rows row .. row + len - 1, at most to the page's end
                for (;; len += 32) {
                    const int k = len + lane;
                    const bool ok = off + k < page && row + k < r.rows && r.slots[row + k] == first + k;
                    const unsigned m = __ballot_sync(0xffffffffu, ok);
                    if (m != 0xffffffffu) {
                        len += __ffs(~m) - 1;
                        break;
                    }
                }
                const T* x = rows + (int64_t)row * r.row_stride;
                float top = 0.0f;
                for (int i = lane; i < len * d; i += 32) {
                    const float v = fabsf(row_value(x + (int64_t)(i / d) * r.row_stride + i % d));
                    if (v < INFINITY) top = fmaxf(top, v);  // NaN and infinities do not set the scale
                }
                top = warp_max(top);
                const float old = off ? held : 0.0f;
                const float now = fmaxf(old, __fdiv_rn(top, kv8_limit(FMT)));
                if (now > old)
                    for (int i = lane; i < off * d; i += 32) codes[i] = (uint8_t)kv8_requant<FMT>(codes[i], old, now);
                for (int i = lane; i < len * d; i += 32)
                    codes[off * d + i] = (uint8_t)kv8_encode<FMT>(row_value(x + (int64_t)(i / d) * r.row_stride + i % d), now);
                held = now;
                row += len;
                __syncwarp();  // the next run rounds these codes anew
            }
            if (lane == 0) *scale = held;
        }
    }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, Kv8Rows r) {
    griddep_launch();
    griddep_wait();
    const int d = c.head_dim, width = c.n_kv * d, sh = c.page_shift;
    const int64_t n_slots = (int64_t)c.n_pages << sh;
    for (int row = blockIdx.x; row < r.rows; row += gridDim.x) {
        const int slot = r.slots[row];
        if (slot < 0 || slot >= n_slots) continue;
        const int64_t pg = slot >> sh;
        const int off = slot & ((1 << sh) - 1);
        for (int i = threadIdx.x; i < width; i += blockDim.x) {
            const int head = i / d, e = i - head * d;
            const int64_t at = (((pg * c.n_kv + head) << sh) + off) * d + e, st = pg * c.n_kv + head;
            ((T*)r.k)[(int64_t)row * r.row_stride + i] = (T)(kv8_decode<FMT>(c.k[at]) * c.k_scale[st]);
            ((T*)r.v)[(int64_t)row * r.row_stride + i] = (T)(kv8_decode<FMT>(c.v[at]) * c.v_scale[st]);
        }
    }
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st) {
    const dim3 grid((r.rows + kAppendWindow - 1) / kAppendWindow), block(kAppendThreads);
    if (r.dtype == kRowF32)
        return c.format == kKv8I8 ? launch_ex(kv8_append_kernel<float, kKv8I8>, grid, block, 0, st, true, c, r)
                                  : launch_ex(kv8_append_kernel<float, kKv8E4M3>, grid, block, 0, st, true, c, r);
    return c.format == kKv8I8 ? launch_ex(kv8_append_kernel<__half, kKv8I8>, grid, block, 0, st, true, c, r)
                              : launch_ex(kv8_append_kernel<__half, kKv8E4M3>, grid, block, 0, st, true, c, r);
}

cudaError_t launch_kv8_read(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st) {
    const dim3 grid(r.rows < num_sms * 8 ? r.rows : num_sms * 8), block(256);
    if (r.dtype == kRowF32)
        return c.format == kKv8I8 ? launch_ex(kv8_read_kernel<float, kKv8I8>, grid, block, 0, st, true, c, r)
                                  : launch_ex(kv8_read_kernel<float, kKv8E4M3>, grid, block, 0, st, true, c, r);
    return c.format == kKv8I8 ? launch_ex(kv8_read_kernel<__half, kKv8I8>, grid, block, 0, st, true, c, r)
                              : launch_ex(kv8_read_kernel<__half, kKv8E4M3>, grid, block, 0, st, true, c, r);
}

}  // namespace lc
