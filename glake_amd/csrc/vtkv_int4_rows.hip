// Rows of a 4-bit cache written (quantised on the way into each sequence's range) and read back.
//
// A head's row takes a team of 16 lanes (32 for head size 256) with eight values each: one 16-byte load, minimum and
// maximum over the team, one division for the scale, eight codes packed into one 4-byte store.  grid (batch, max_seq_len),
// one workgroup per token with its K and V heads dealt to the teams.  The bytes of the 16-bit rows bound it (about 4/5
// of what moves), at decode-step sizes the launch itself.
#include "vtkv_common.h"
#include "vtkv_fp8.h"
#include "vtkv_int4.h"

namespace {

constexpr int kThreads = 256;

struct RowsParams {
  const char *key, *value;  // (read: where the values go)
  const int64_t *k_ptrs, *v_ptrs, *slot_m, *slot_ids;
  const int32_t *seq_lens, *cache_seq_lens;
  int max_seq_len, num_heads, head_size, row_bytes;
  int64_t key_stride, value_stride;  // elements
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// The token of this workgroup: false where there is none; else its row in the cache (per side) and in the tensors.
__device__ __forceinline__ bool token_of(const RowsParams &p, int64_t &src_row, int64_t &slot, int64_t &off) {
  const int b = blockIdx.x, t = blockIdx.y;
  if (p.max_seq_len != 1 && t >= p.seq_lens[b]) return false;
  off = p.slot_m[b];
  if (off < 0) return false;
  off += (int64_t)t * p.row_bytes;
  slot = p.slot_ids[b];
  src_row = p.max_seq_len == 1 ? (int64_t)b : (int64_t)p.cache_seq_lens[b] + t;
  return true;
}

template <bool F16>
__device__ __forceinline__ float widen(unsigned pair, int which) {
  const unsigned short h = (unsigned short)(which ? pair >> 16 : pair & 0xffffu);
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, h);
  return vtkv::bf16_bits_to_f32(h);
}

template <bool F16, bool ALIGNED, int TEAM>
__global__ void __launch_bounds__(kThreads) int4_write_kernel(RowsParams p) {
  int64_t src_row, slot, off;
  if (!token_of(p, src_row, slot, off)) return;
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int half = p.head_size / 2;
  const bool live = 8 * lane < p.head_size;
  for (int hr = team; hr < 2 * p.num_heads; hr += kThreads / TEAM) {
    const bool is_v = hr >= p.num_heads;
    const int head = is_v ? hr - p.num_heads : hr;
    const char *src = (is_v ? p.value + src_row * p.value_stride * 2 : p.key + src_row * p.key_stride * 2) +
                      ((int64_t)head * p.head_size + 8 * lane) * 2;
    char *row = reinterpret_cast<char *>(is_v ? p.v_ptrs[slot] : p.k_ptrs[slot]) + off;
    u32x4 raw = {0, 0, 0, 0};
    if (live) {
      if constexpr (ALIGNED) {
        raw = *reinterpret_cast<const u32x4 *>(src);
      } else {
        const uint16_t *e = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = (unsigned)e[2 * i] | (unsigned)e[2 * i + 1] << 16;
      }
    }
    float x[8], lo = INFINITY, hi = -INFINITY;
    bool odd = false;  // a value that is not finite
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = widen<F16>(raw[i >> 1], i & 1);
      odd |= (vtkv::f32_bits(x[i]) & 0x7f800000u) == 0x7f800000u;
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
    if (!live) lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int d = 1; d < TEAM; d <<= 1) {
      lo = fminf(lo, __shfl_xor(lo, d, TEAM));
      hi = fmaxf(hi, __shfl_xor(hi, d, TEAM));
    }
    const unsigned long long any = __ballot(odd);
    const unsigned long long mine = (any >> ((threadIdx.x & 63) / TEAM * TEAM)) & ((1ull << TEAM) - 1);
    unsigned zero16 = vtkv::f32_to_bf16_bits_rne(lo);
    const float zero = vtkv::bf16_bits_to_f32((uint16_t)zero16);
    const float range = hi - zero;
    unsigned scale16 = vtkv::f32_to_bf16_bits_rne(range / 15.0f);
    float scale = vtkv::bf16_bits_to_f32((uint16_t)scale16);
    if (scale < 1.17549435e-38f) scale = 0.f, scale16 = 0;  // (also a negative one: every value equal, zero rounded up)
    const bool bad = mine != 0 || (vtkv::f32_bits(range) & 0x7f800000u) == 0x7f800000u;
    const float inverse = scale > 0.f ? __builtin_amdgcn_rcpf(scale) : 0.f;
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // The quotient's nearest code first, then the exact remainder against half a step: a value on the border
      // between two codes takes the upper one, whatever the reciprocal's last bit is.  (16-bit values over a bf16
      // step meet that border in one of some hundred values.)
      const float d = x[i] - zero;
      float c = __builtin_rintf(d * inverse);
      const float rest = 2.f * __builtin_fmaf(-c, scale, d);
      c += rest >= scale ? 1.f : rest < -scale ? -1.f : 0.f;
      const int code = scale > 0.f && !bad ? (int)fminf(fmaxf(c, 0.f), 15.f) : 0;
      word |= (unsigned)code << (4 * i);
    }
    if (bad) scale16 = zero16 = 0x7fc0u;
    if (live) *reinterpret_cast<unsigned *>(row + head * half + 4 * lane) = word;
    if (lane == 0) *reinterpret_cast<unsigned *>(row + p.num_heads * half + 4 * head) = scale16 | zero16 << 16;
    if (head == p.num_heads - 1)
      for (int i = p.num_heads * (half + 4) + 4 * lane; i < p.row_bytes; i += 4 * TEAM)
        *reinterpret_cast<unsigned *>(row + i) = 0;
  }
}

template <int DT>
__global__ void __launch_bounds__(kThreads) int4_read_kernel(RowsParams p) {
  int64_t dst_row, slot, off;
  if (!token_of(p, dst_row, slot, off)) return;
  const int half = p.head_size / 2, words = p.head_size / 8;  // (a word: eight codes)
  for (int i = threadIdx.x; i < 2 * p.num_heads * words; i += kThreads) {
    const bool is_v = i >= p.num_heads * words;
    const int j = is_v ? i - p.num_heads * words : i;
    const int head = j / words, at = j % words;
    const char *row = reinterpret_cast<const char *>(is_v ? p.v_ptrs[slot] : p.k_ptrs[slot]) + off;
    const unsigned codes = *reinterpret_cast<const unsigned *>(row + head * half + 4 * at);
    const unsigned sz = *reinterpret_cast<const unsigned *>(row + p.num_heads * half + 4 * head);
    const float scale = vtkv::bits_f32(sz << 16), zero = vtkv::bits_f32(sz & 0xffff0000u);
    char *dst = const_cast<char *>(is_v ? p.value : p.key);
    const int64_t e0 = dst_row * (is_v ? p.value_stride : p.key_stride) + (int64_t)head * p.head_size + 8 * at;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // (code * scale has 12 significant bits: the one rounding to fp32 is the addition's)
      const float x = __builtin_fmaf((float)((codes >> (4 * e)) & 15u), scale, zero);
      if constexpr (DT == VTKV_F32) reinterpret_cast<float *>(dst)[e0 + e] = x;
      else if constexpr (DT == VTKV_BF16) reinterpret_cast<uint16_t *>(dst)[e0 + e] = vtkv::f32_to_bf16_bits_rne(x);
      else reinterpret_cast<_Float16 *>(dst)[e0 + e] = (_Float16)x;
    }
  }
}

int check_rows(const void *key, const void *value, const int64_t *k_ptrs, const int64_t *v_ptrs, const int64_t *slot_m,
               const int64_t *slot_ids, const int32_t *seq_lens, const int32_t *cache_seq_lens, int batch,
               int max_seq_len, int num_heads, int head_size, int64_t key_stride, int64_t value_stride) {
  VTKV_REQUIRE(key && value && k_ptrs && v_ptrs && slot_m && slot_ids, "null argument");
  VTKV_REQUIRE(batch >= 0 && max_seq_len >= 1 && num_heads > 0, "bad sizes");
  VTKV_REQUIRE(vtkv::int4_head_size(head_size), "a 4-bit cache takes head sizes 64, 80, 96, 112, 128 and 256, not %d", head_size);
  VTKV_REQUIRE(max_seq_len == 1 || (seq_lens && cache_seq_lens), "seq_lens and cache_seq_lens are needed when max_seq_len > 1");
  VTKV_REQUIRE(max_seq_len <= 65535, "max_seq_len %d exceeds the grid limit 65535", max_seq_len);
  VTKV_REQUIRE(num_heads <= 65536, "too many kv heads");
  const int64_t row = (int64_t)num_heads * head_size;
  VTKV_REQUIRE(key_stride >= row && value_stride >= row, "row stride smaller than a row");
  return VTKV_OK;
}

}  // namespace

namespace vtkv {

int int4_write_rows(const void *key, const void *value, const int64_t *k_ptrs, const int64_t *v_ptrs,
                    const int64_t *slot_m, const int64_t *slot_ids, const int32_t *seq_lens,
                    const int32_t *cache_seq_lens, int batch, int max_seq_len, int num_heads, int head_size,
                    int64_t key_stride, int64_t value_stride, int src_dtype, void *stream) {
  const int rc = check_rows(key, value, k_ptrs, v_ptrs, slot_m, slot_ids, seq_lens, cache_seq_lens, batch, max_seq_len,
                            num_heads, head_size, key_stride, value_stride);
  if (rc < 0) return rc;
  VTKV_REQUIRE(src_dtype == VTKV_BF16 || src_dtype == VTKV_F16, "a 4-bit cache takes bfloat16 and float16 keys and values");
  if (batch == 0) return VTKV_OK;
  const RowsParams p = {(const char *)key, (const char *)value, k_ptrs, v_ptrs, slot_m, slot_ids, seq_lens, cache_seq_lens,
                        max_seq_len, num_heads, head_size, (int)int4_row_bytes(num_heads, head_size), key_stride,
                        value_stride};
  const bool aligned = key_stride % 8 == 0 && value_stride % 8 == 0 && (uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0;
  const dim3 grid((unsigned)batch, (unsigned)max_seq_len);
  hipStream_t st = (hipStream_t)stream;
#define VTKV_INT4_WRITE(F, A)                                                                        \
  do {                                                                                               \
    if (head_size > 128)                                                                             \
      hipLaunchKernelGGL((int4_write_kernel<F, A, 32>), grid, dim3(kThreads), 0, st, p);             \
    else                                                                                             \
      hipLaunchKernelGGL((int4_write_kernel<F, A, 16>), grid, dim3(kThreads), 0, st, p);             \
  } while (0)
  const bool f16 = src_dtype == VTKV_F16;
  if (f16 && aligned) VTKV_INT4_WRITE(true, true);
  else if (f16) VTKV_INT4_WRITE(true, false);
  else if (aligned) VTKV_INT4_WRITE(false, true);
  else VTKV_INT4_WRITE(false, false);
#undef VTKV_INT4_WRITE
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

}  // namespace vtkv

extern "C" {

int64_t vtkv_kv_row_bytes(int num_kv_heads, int head_size, int kv_dtype) {
  if (num_kv_heads <= 0 || head_size <= 0) return 0;
  if (kv_dtype == VTKV_INT4) return vtkv::int4_head_size(head_size) ? vtkv::int4_row_bytes(num_kv_heads, head_size) : 0;
  return (int64_t)num_kv_heads * head_size * vtkv::elem_bytes(kv_dtype);
}

int vtkv_read_cached_rows(void *key, void *value, const int64_t *k_ptrs, const int64_t *v_ptrs, const int64_t *slot_m,
                          const int64_t *slot_ids, const int32_t *seq_lens, const int32_t *cache_seq_lens, int batch,
                          int max_seq_len, int num_heads, int head_size, int64_t key_stride, int64_t value_stride,
                          int dst_dtype, int kv_dtype, void *stream) {
  VTKV_REQUIRE(kv_dtype == VTKV_INT4, "read_cached_rows reads 4-bit caches");
  const int rc = check_rows(key, value, k_ptrs, v_ptrs, slot_m, slot_ids, seq_lens, cache_seq_lens, batch, max_seq_len,
                            num_heads, head_size, key_stride, value_stride);
  if (rc < 0) return rc;
  VTKV_REQUIRE(dst_dtype == VTKV_F32 || dst_dtype == VTKV_BF16 || dst_dtype == VTKV_F16, "the values go to F32, BF16 or F16");
  if (batch == 0) return VTKV_OK;
  const RowsParams p = {(const char *)key, (const char *)value, k_ptrs, v_ptrs, slot_m, slot_ids, seq_lens, cache_seq_lens,
                        max_seq_len, num_heads, head_size, (int)vtkv::int4_row_bytes(num_heads, head_size), key_stride,
                        value_stride};
  const dim3 grid((unsigned)batch, (unsigned)max_seq_len);
  hipStream_t st = (hipStream_t)stream;
  if (dst_dtype == VTKV_F32) hipLaunchKernelGGL(int4_read_kernel<VTKV_F32>, grid, dim3(kThreads), 0, st, p);
  else if (dst_dtype == VTKV_BF16) hipLaunchKernelGGL(int4_read_kernel<VTKV_BF16>, grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL(int4_read_kernel<VTKV_F16>, grid, dim3(kThreads), 0, st, p);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

}  // extern "C"
