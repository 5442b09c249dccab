// lc_kv8_attention.cu -- causal grouped-query attention over the 8-bit pages.
//
// Query j of a sequence with n queries and a length of L stands at position
// L - n + j and sees positions 0..L - n + j; o = sum_t softmax(scale q.k_t) v_t
// with k_t, v_t = code * scale of the page and head.  A query that sees
// nothing gives zeros; rows behind the last sequence are left as they were.
#include "lc_kv8_decode.cuh"
#include "lc_kv8_prefill.cuh"

namespace lc {
namespace {

// Calls f with the kernel's parameters as types: row type, code format, head size.
template <typename F>
cudaError_t by_shape(int dtype, int format, int head_dim, F&& f) {
    auto dim = [&](auto row, auto fmt) {
        return head_dim == 64 ? f(row, fmt, std::integral_constant<int, 64>()) : f(row, fmt, std::integral_constant<int, 128>());
    };
    auto codes = [&](auto row) {
        return format == kKv8I8 ? dim(row, std::integral_constant<int, kKv8I8>()) : dim(row, std::integral_constant<int, kKv8E4M3>());
    };
    return dtype == kRowF32 ? codes(float()) : codes(__half());
}

}  // namespace

// The two kernels' workspaces, one behind the other.
static size_t decode_ws(int num_sms) { return (kv8_decode_ws_bytes(num_sms) + 255) / 256 * 256; }

size_t kv8_attention_ws_bytes(int num_sms) { return decode_ws(num_sms) + kv8_prefill_ws_bytes(num_sms); }

cudaError_t kv8_attention_prepare(void* ws, int num_sms, cudaStream_t st) {
    for (int i = 0; i < 8; ++i) {
        const cudaError_t e = by_shape(i & 1, (i >> 1) & 1, i & 4 ? 128 : 64, [](auto row, auto fmt, auto d) {
            using T = decltype(row);
            cudaError_t e = kv8_decode_prepare<T, fmt.value, d.value, 1>();
            if (e == cudaSuccess) e = kv8_decode_prepare<T, fmt.value, d.value, 2>();
            return e != cudaSuccess ? e : kv8_prefill_prepare<T, fmt.value, d.value>();
        });
        if (e != cudaSuccess) return e;
    }
    return kv8_attention_clear(ws, num_sms, st);
}

cudaError_t kv8_attention_clear(void* ws, int num_sms, cudaStream_t st) {
    const cudaError_t e = cudaMemsetAsync(ws, 0, kv8_counter_bytes(num_sms), st);
    if (e != cudaSuccess) return e;
    return cudaMemsetAsync((uint8_t*)ws + decode_ws(num_sms), 0, kv8_prefill_counter_bytes(num_sms), st);
}

// Rows of a unit, by the rows that share a kv head's codes at most.  More rows
// share one reading of the codes; units of 8 instead of 4 cost registers and, in
// short sequences, idle warps.  us, 4 kv heads, head size 64 fp32 / 128 f16:
//   8 rows, units of 8 | 4:   1 x 131071 positions 34 | 36 / 52 | 61,
//                             64 x 1..8191 52 | 63 / 94 | 111, 64 x 1..500 19 | 16 / 27 | 23
//   16 rows, of 256 | 8:      160 | 48 / 176 | 79, 233 | 87 / 250 | 159, 48 | 22 / 51 | 34
//   32 rows, of 256 | 8:      159 | 76 / 175 | 136, 234 | 154 / 251 | 298, 48 | 28 / 51 | 51
//   64 rows, of 256 | 8:      160 | 132 / 176 | 252, (2 kv heads) 130 | 153 / 138 | 298, 33 | 28 / 35 | 51
// So up to 16 rows, at head size 64 up to 32, units of 8 would be the faster ones:
// their line of work in 32 bits is shorter by as much, and calls that fit now would not.
static int unit_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : kPreRows; }

bool kv8_attention_fits(const Kv8& c, const Kv8Attention& a) {
    const int group = a.n_heads / c.n_kv, unit = unit_rows((int64_t)group * a.max_q);
    const int64_t step = unit == kPreRows ? kPreTok : 2048 / c.head_dim, room = (int64_t)a.table_stride << c.page_shift;
    const double units = (double)c.n_kv * ((double)a.rows * group / unit + a.n_seqs);
    return units * (double)(room / step + 1 + kPreUnitCost) < 4294967296.0;
}

cudaError_t launch_kv8_attention(const Kv8& c, const Kv8Attention& a, int num_sms, void* ws, int* err, cudaStream_t st) {
    const int unit = unit_rows((int64_t)(a.n_heads / c.n_kv) * a.max_q);  // of the rows that share a kv head's codes, at most
    return by_shape(a.dtype, c.format, c.head_dim, [&](auto row, auto fmt, auto d) {
        using T = decltype(row);
        // Units of 4 rows where a sequence has no more, of 8 where it has (more
        // rows share one reading of the codes), and the tensor-core tiles of
        // 128 beyond.
        if (unit == 4) return launch_kv8_decode<T, fmt.value, d.value, 1>(c, a, num_sms, ws, st);
        if (unit == 8) return launch_kv8_decode<T, fmt.value, d.value, 2>(c, a, num_sms, ws, st);
        return launch_kv8_prefill<T, fmt.value, d.value>(c, a, num_sms, (uint8_t*)ws + decode_ws(num_sms), err, st);
    });
}

}  // namespace lc
