// lc_kv8_attention.cu -- causal grouped-query attention over the 8-bit pages.
//
// Query j of a sequence with n queries and a length of L stands at position
// L - n + j and sees positions 0..L - n + j; o = sum_t softmax(scale q.k_t) v_t
// with k_t, v_t = code * scale of the page and head.  A query that sees
// nothing gives zeros; rows behind the last sequence are left as they were.
#include "lc_internal.h"
#include "lc_kv8.cuh"

namespace lc {
namespace {

// One warp per (query row, head), the lanes over the head's elements, one
// position at a time with the running maximum and sum of the softmax.
template <typename T, int FMT>
__global__ void __launch_bounds__(128) kv8_attention_simple(Kv8 c, Kv8Attention a) {
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int row = (int)(unit / a.n_heads), head = (int)(unit % a.n_heads);
    if (row >= a.rows) return;
    int s = row, j = 0, nq = 1;
    if (a.q_start) {
        int lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before this row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.q_start[mid] <= row) lo = mid;
            else hi = mid;
        }
        s = lo;
        j = row - a.q_start[s];
        nq = a.q_start[s + 1] - a.q_start[s];
        if (j < 0 || j >= nq) return;
    } else if (row >= a.n_seqs) {
        return;
    }
    const int d = c.head_dim, sh = c.page_shift, kvh = head / (a.n_heads / c.n_kv), per = d / 32;
    const int64_t room = (int64_t)a.table_stride << sh;
    const int64_t len = a.kv_lens[s] < room ? a.kv_lens[s] : room;
    const int64_t seen = a.kv_lens[s] - nq + j + 1 < len ? a.kv_lens[s] - nq + j + 1 : len;
    const T* q = (const T*)a.q + (int64_t)row * a.q_stride + head * d + lane * per;
    float qv[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, sum = 0.0f;
    for (int e = 0; e < 4; ++e) qv[e] = e < per ? (float)q[e] * a.scale : 0.0f;
    for (int64_t t = 0; t < seen; ++t) {
        const int pg = a.table[(int64_t)s * a.table_stride + (t >> sh)];
        if (pg < 0 || pg >= c.n_pages) continue;
        const int64_t st = (int64_t)pg * c.n_kv + kvh, at = ((st << sh) + (t & ((1 << sh) - 1))) * d + lane * per;
        float x = 0.0f;
        for (int e = 0; e < 4; ++e)
            if (e < per) x += qv[e] * kv8_decode<FMT>(c.k[at + e]);
        x = warp_sum(x) * c.k_scale[st];
        const float mn = fmaxf(m, x), keep = expf(m - mn), p = expf(x - mn);
        sum = sum * keep + p;
        for (int e = 0; e < 4; ++e)
            if (e < per) o[e] = o[e] * keep + p * (kv8_decode<FMT>(c.v[at + e]) * c.v_scale[st]);
        m = mn;
    }
    T* out = (T*)a.out + (int64_t)row * a.out_stride + head * d + lane * per;
    for (int e = 0; e < 4; ++e)
        if (e < per) out[e] = (T)(sum > 0.0f ? o[e] / sum : 0.0f);
}

}  // namespace

cudaError_t launch_kv8_attention(const Kv8& c, const Kv8Attention& a, int num_sms, cudaStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.rows * a.n_heads + 3) / 4)), block(128);
    if (a.dtype == kRowF32)
        return c.format == kKv8I8 ? launch_ex(kv8_attention_simple<float, kKv8I8>, grid, block, 0, st, true, c, a)
                                  : launch_ex(kv8_attention_simple<float, kKv8E4M3>, grid, block, 0, st, true, c, a);
    return c.format == kKv8I8 ? launch_ex(kv8_attention_simple<__half, kKv8I8>, grid, block, 0, st, true, c, a)
                              : launch_ex(kv8_attention_simple<__half, kKv8E4M3>, grid, block, 0, st, true, c, a);
}

}  // namespace lc
