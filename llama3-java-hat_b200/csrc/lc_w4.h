// lc_w4.h -- host declarations of the 4-bit weights (lc_w4.cu: quantising,
// packing and reading; lc_w4_product.cu: products) and of the log
// probabilities (lc_logprobs.cu).
//
// Layout.  Codes lie in tiles of 16 rows and blocks of 128 columns, [tiles]
// [blocks][1024 bytes]; 16 bytes of each 512 (a chunk of 64 columns) belong to
// lane 4 g + t of the warp that reads them: rows g and g + 8, and of each 32
// columns the eight from 8 t on.  Word j of the 16 bytes holds columns
// 32 (j / 2) + 8 t + 4 (j % 2) + e, e = 0..3, at bit {0, 16, 8, 24}[e] for row g
// and 4 bits higher for row g + 8, the whole word rotated left by 3.  So the word,
// and the word rotated by 8 bits, masked by 0x00780078 and 0x07800780, give the four
// registers that one m16n8k16 product takes from the lane, as pairs of f16 numbers
// c 2^-21 (row g) and c 2^-17 (row g + 8): f16 numbers below 2^-13 are linear in
// their bits, and an FMA makes c - z of them.  Each product lies within one group;
// and what the lane has of a row are runs of eight columns, 16 bytes of f16, which
// is what tcgen05 operands are made of.  The order of columns within a product does
// not matter as long as both operands have the same.
//
// Scales (f16) and zero points (bytes) of a block: [8 g][128 / group][2], the
// pair being rows g and g + 8.  Rows
// behind the last and groups without columns have scale 0; what codes stand behind
// the last column and row is of no consequence.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "lc_paged.h"

namespace lc {

constexpr int kW4Rows = 16;    // rows of a tile
constexpr int kW4Cols = 128;   // columns of a block
constexpr int kW4BlockBytes = 1024;
constexpr int kW4Turn = 3;  // bits by which words are rotated

struct W4 {
    uint8_t* codes;
    uint16_t* scales;
    uint8_t* zeros;  // null: 8
    int rows, cols, group;
    int tiles, blocks;
};
struct W4Product {
    const void* x;
    void* y;
    const void* residual;  // null: none
    int64_t x_stride, y_stride, residual_stride;  // elements
    int batch, dtype;
};
cudaError_t launch_w4_quantize(const W4& w, const void* values, int64_t stride, int dtype, int num_sms, cudaStream_t st);
cudaError_t launch_w4_pack(const W4& w, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int num_sms, cudaStream_t st);
cudaError_t launch_w4_read(const W4& w, void* values, int64_t stride, int dtype, int num_sms, cudaStream_t st);
// Whether the product goes through the workspace (ws of w4_product_ws_bytes; else null).
bool w4_product_uses_ws(const W4& w, const W4Product& p, int num_sms);
size_t w4_product_ws_bytes();
cudaError_t launch_w4_product(const W4& w, const W4Product& p, int num_sms, void* ws, int* err, cudaStream_t st);

constexpr int kLogprobsMaxTop = 32;
struct Logprobs {
    const void* x;
    int64_t stride;
    int dtype, rows, vocab, top;
    float scale;
    const int32_t* tokens;  // null: none
    float* token_logprobs;  // each output: null when not asked for
    int32_t* token_ranks;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
};
cudaError_t launch_logprobs(const Logprobs& p, int num_sms, cudaStream_t st);

}  // namespace lc
