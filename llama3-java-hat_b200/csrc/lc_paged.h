// lc_paged.h -- host declarations of the paged 8-bit KV cache operators:
// rotary positions (lc_rope.cu), page bookkeeping (lc_pages.cu), quantised
// append and read (lc_kv8.cu) and attention over the pages
// (lc_kv8_attention.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lc {

enum RowType : int { kRowF32 = 0, kRowF16 = 1 };
enum Kv8Format : int { kKv8I8 = 0, kKv8E4M3 = 1 };

// ---- rotary positions ----
constexpr int kRopeMaxPairs = 256;  // head_dim <= 512
struct RopeTurns {
    double t[kRopeMaxPairs];  // turns (angle / 2 pi) per position of each rotated pair
};
struct RopeApply {
    const void* x;
    void* y;
    const int32_t* pos;
    int rows, heads, head_dim, rot_dim;
    int64_t x_stride, y_stride;  // elements
    float mult;                  // factor on cos and sin
    float sign;                  // -1: the transposed map
    bool half;                   // pairs (j, j + rot_dim / 2) instead of (2j, 2j + 1)
    int dtype;
};
cudaError_t launch_rope_apply(const RopeApply& a, const RopeTurns& turns, int num_sms, cudaStream_t st);

// ---- page bookkeeping ----
constexpr int kPagesMaxSeqs = 4096;
struct PagesStep {
    const int32_t* lens;
    const int32_t* n_new;
    int n_seqs, page_shift, table_stride, n_pages, capacity;
    int32_t* table;
    int32_t* free_list;
    const int32_t* free_count;
    int32_t *lens_out, *q_start, *slots, *positions, *seq_ids, *free_count_out, *status;
};
cudaError_t launch_pages_step(const PagesStep& p, cudaStream_t st);

// ---- 8-bit pages ----
struct Kv8 {
    uint8_t *k, *v;            // [n_pages][n_kv][page][d]
    float *k_scale, *v_scale;  // [n_pages][n_kv]
    int n_pages, page_shift, n_kv, head_dim, format;
};
struct Kv8Rows {
    void *k, *v;         // [rows][n_kv * d], row stride in elements
    int64_t row_stride;
    const int32_t* slots;
    int rows, dtype;
};
cudaError_t launch_kv8_append(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8& c, const Kv8Rows& r, int num_sms, cudaStream_t st);

struct Kv8Attention {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const int32_t* q_start;  // [n_seqs + 1]; null: row s is the one query of sequence s
    const int32_t* kv_lens;
    const int32_t* table;
    int table_stride, n_seqs, rows, max_q, n_heads, dtype;
    float scale;
};
// Workspace of one call at a time: its size depends on the device alone.
// prepare clears its counters and sets the kernels' attributes, once.
size_t kv8_attention_ws_bytes(int num_sms);
// Whether the call's line of work can be counted in 32 bits.
bool kv8_attention_fits(const Kv8& c, const Kv8Attention& a);
cudaError_t kv8_attention_prepare(void* ws, int num_sms, cudaStream_t st);
// Its counters to zero again, behind a call that gave up.
cudaError_t kv8_attention_clear(void* ws, int num_sms, cudaStream_t st);
cudaError_t launch_kv8_attention(const Kv8& c, const Kv8Attention& a, int num_sms, void* ws, int* err, cudaStream_t st);

}  // namespace lc
