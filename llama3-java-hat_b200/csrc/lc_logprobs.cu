// lc_logprobs.cu -- log probabilities of given tokens with their ranks, the
// entropy and the best alternatives, from rows of logits.
//
// With m the largest logit of a row, t_i = scale (x_i - m) and S = sum e^t_i:
// log p_i = t_i - ln S and H = ln S - (sum t_i e^t_i) / S.  Tokens are ordered
// by logit, equal ones by index.
#include "lc_internal.h"
#include "lc_w4.h"

namespace lc {
namespace {

constexpr int kSimpleThreads = 256;

template <typename T>
LC_DEV float logit(const T* x, int i) {
    const float v = (float)x[i] + 0.0f;  // no negative zeros
    return v;
}
LC_DEV uint32_t ordered(float v) {  // NaN below -inf
    if (!(v == v)) v = -INFINITY;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
LC_DEV uint64_t order_key(float v, int i) { return (uint64_t)ordered(v) << 32 | (uint32_t)~i; }

LC_DEV double block_sum(double v, double* buf) {
    __syncthreads();
    buf[threadIdx.x] = v;
    __syncthreads();
    for (int o = kSimpleThreads / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) buf[threadIdx.x] += buf[threadIdx.x + o];
        __syncthreads();
    }
    return buf[0];
}
LC_DEV uint64_t block_max(uint64_t v, uint64_t* buf) {
    __syncthreads();
    buf[threadIdx.x] = v;
    __syncthreads();
    for (int o = kSimpleThreads / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) buf[threadIdx.x] = max(buf[threadIdx.x], buf[threadIdx.x + o]);
        __syncthreads();
    }
    return buf[0];
}

template <typename T>
__global__ void __launch_bounds__(kSimpleThreads) logprobs_simple_kernel(Logprobs p) {
    __shared__ double sums[kSimpleThreads];
    __shared__ uint64_t keys[kSimpleThreads];
    const int64_t row = blockIdx.x;
    const T* x = (const T*)p.x + row * p.stride;
    int token = p.tokens ? p.tokens[row] : -1;
    if (token >= p.vocab) token = -1;
    const uint64_t mine = token >= 0 ? order_key(logit(x, token), token) : ~0ull;
    uint64_t best = 0;
    double bad = 0, before = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kSimpleThreads) {
        const float v = logit(x, i);
        const uint64_t k = order_key(v, i);
        best = max(best, k);
        before += k > mine;
        bad += !(v < INFINITY);  // NaN or +inf
    }
    best = block_max(best, keys);
    before = block_sum(before, sums);
    bad = block_sum(bad, sums);
    const float high = logit(x, (int)~(uint32_t)best);
    const bool empty = high == -INFINITY;
    double total = 0, weighted = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kSimpleThreads) {
        const float t = empty ? -INFINITY : (logit(x, i) - high) * p.scale;
        const float e = expf(t);
        total += e;
        if (e > 0.0f) weighted += (double)e * t;
    }
    total = block_sum(total, sums);
    weighted = block_sum(weighted, sums);
    const double log_total = empty ? 0.0 : log(total);
    auto logp = [&](float v) { return bad > 0 ? NAN : empty ? -INFINITY : (float)((double)((v - high) * p.scale) - log_total); };
    if (threadIdx.x == 0) {
        if (p.token_logprobs) p.token_logprobs[row] = token >= 0 ? logp(logit(x, token)) : 0.0f;
        if (p.token_ranks) p.token_ranks[row] = token >= 0 ? (int)before : -1;
        if (p.entropy) p.entropy[row] = bad > 0 ? NAN : empty ? 0.0f : (float)(log_total - weighted / total);
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        uint64_t next = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kSimpleThreads) {
            const uint64_t key = order_key(logit(x, i), i);
            if (key < last) next = max(next, key);
        }
        last = block_max(next, keys);
        if (threadIdx.x == 0) {
            const int id = k < p.vocab ? (int)~(uint32_t)last : -1;
            if (p.top_ids) p.top_ids[row * p.top + k] = id;
            if (p.top_logprobs) p.top_logprobs[row * p.top + k] = id >= 0 ? logp(logit(x, id)) : bad > 0 ? NAN : -INFINITY;
        }
    }
}

}  // namespace

cudaError_t launch_logprobs(const Logprobs& p, int, cudaStream_t st) {
    if (p.dtype == kRowF32) logprobs_simple_kernel<float><<<p.rows, kSimpleThreads, 0, st>>>(p);
    else logprobs_simple_kernel<__half><<<p.rows, kSimpleThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace lc
