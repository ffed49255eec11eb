// Rows of a 4-bit KV cache.  One row holds one token's K (or V) of every kv head:
//
//   [num_kv_heads][head_size / 2]   codes, value 2i of a head in the low half of its byte i, value 2i + 1 in the high half
//   [num_kv_heads] {bf16 scale, bf16 zero}
//   padding to a multiple of 16 bytes (zeros)
//
// A value is code * scale + zero, codes 0..15.  zero is the smallest value of the head's row rounded to bf16 (exact
// for bf16 models), scale = bf16((largest - zero) / 15), code = floor((x - zero) / scale + 1/2) clamped to 0..15.  The
// scale is per head and token: what a code is multiplied with depends on the row alone, so attention can run its
// products on the bare codes and apply scale and zero to whole logits and weights.  bf16 for both, because its range
// is that of every model type; its 8 bits move a code's border by less than 1/17 of a step at the far end.
// A head's row whose values are all equal has scale 0.  One with a value that is not finite (or whose values are
// further apart than the largest float) has scale = zero = NaN and reads back as NaN, as it would have made every
// logit it meets NaN in a 16-bit cache.
#pragma once
#include <stdint.h>

namespace vtkv {

inline int64_t int4_row_bytes(int num_kv_heads, int head_size) {
  return ((int64_t)num_kv_heads * (head_size / 2 + 4) + 15) / 16 * 16;
}
inline bool int4_head_size(int d) { return d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 256; }

// csrc/vtkv_int4_rows.hip
int int4_write_rows(const void *key, const void *value, const int64_t *k_ptrs, const int64_t *v_ptrs,
                    const int64_t *slot_m, const int64_t *slot_ids, const int32_t *seq_lens,
                    const int32_t *cache_seq_lens, int batch, int max_seq_len, int num_heads, int head_size,
                    int64_t key_stride, int64_t value_stride, int src_dtype, void *stream);
// csrc/vtkv_int4_decode.hip
constexpr int kDecodeSpans = 256;  // workgroups of a launch at most: one per CU
int64_t int4_decode_workspace_bytes(int num_seqs, int num_heads, int head_size);
int int4_decode(void *out, const void *q, const int64_t *k_ptrs, const int64_t *v_ptrs, const int64_t *slot_ids,
                const int32_t *seq_lens, int num_seqs, int num_heads, int num_kv_heads, int head_size, int64_t q_stride,
                float scale, int max_seq_len, const float *alibi_slopes, int q_dtype, int out_dtype, void *workspace,
                int64_t workspace_bytes, void *stream);

}  // namespace vtkv
