// Rows of a 4-bit cache written (quantised on the way into each sequence's range) and read back.
//
// A head's row takes a team of 16 lanes (32 for head size 256) with eight values each: one 16-byte load, minimum and
// maximum over the team, one division for the scale, eight codes packed into one 4-byte store.  A workgroup takes four
// tokens, whose K and V heads its teams share out, four loads of a team in flight.
//   The bytes of the 16-bit rows bound it (about 4/5 of what moves), writing also the 30 instructions per value, at
// decode-step sizes the launch.  15 800 tokens of 8 kv heads of 128 (65 MB of 16-bit rows, 17 MB of 4-bit ones): written in
// 27 us, 3.0 TB/s, read back in 21 us, 3.9 TB/s; with one token per workgroup 42 and 32 us, with two 29 and 24, with eight
// as with four.
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

constexpr int kTokens = 4;  // of a workgroup, one behind the other
constexpr int kAhead = 4;   // head rows that a team asks for before it works on the first

// The tokens of this workgroup: how many, the first one's row in the tensors, and where its cache rows are.
struct Tokens {
  int rows;
  int64_t first;
  char *k, *v;
};
__device__ __forceinline__ Tokens tokens_of(const RowsParams &p) {
  const int b = blockIdx.x, t0 = blockIdx.y * kTokens;
  Tokens t;
  t.rows = p.max_seq_len == 1 ? 1 : min(kTokens, min(p.seq_lens[b], p.max_seq_len) - t0);
  const int64_t off = p.slot_m[b];
  if (off < 0) t.rows = 0;
  if (t.rows <= 0) return t;
  const int64_t slot = p.slot_ids[b], at = off + (int64_t)t0 * p.row_bytes;
  t.k = reinterpret_cast<char *>(p.k_ptrs[slot]) + at;
  t.v = reinterpret_cast<char *>(p.v_ptrs[slot]) + at;
  t.first = p.max_seq_len == 1 ? (int64_t)b : (int64_t)p.cache_seq_lens[b] + t0;
  return t;
}

// Item i of a workgroup: (token, K or V, head).
struct Item {
  int token, head;
  bool is_v;
};
__device__ __forceinline__ Item item_of(int i, int num_heads) {
  const int token = (int)((unsigned)i / (unsigned)(2 * num_heads)), hr = i - token * 2 * num_heads;
  return {token, hr >= num_heads ? hr - num_heads : hr, hr >= num_heads};
}

template <bool F16>
__device__ __forceinline__ float widen(unsigned pair, int which) {
  const unsigned short h = (unsigned short)(which ? pair >> 16 : pair & 0xffffu);
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, h);
  return vtkv::bf16_bits_to_f32(h);
}

// A value joined over each team's lanes, neighbours first.
template <int TEAM, typename Op>
__device__ __forceinline__ float over_team(float x, Op op) {
#define VTKV_JOIN(CTRL) \
  x = op(x, vtkv::bits_f32((unsigned)__builtin_amdgcn_update_dpp(0, (int)vtkv::f32_bits(x), CTRL, 0xf, 0xf, true)))
  VTKV_JOIN(0xb1);   // lanes 1 0 3 2 of each four
  VTKV_JOIN(0x4e);   // 2 3 0 1
  VTKV_JOIN(0x141);  // each eight mirrored
  VTKV_JOIN(0x140);  // each sixteen mirrored
#undef VTKV_JOIN
  if constexpr (TEAM == 32) x = op(x, __shfl_xor(x, 16, 32));
  return x;
}

template <bool F16, bool ALIGNED, int TEAM>
__global__ void __launch_bounds__(kThreads) int4_write_kernel(RowsParams p) {
  const Tokens t = tokens_of(p);
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int half = p.head_size / 2, items = max(t.rows, 0) * 2 * p.num_heads;
  const bool live = 8 * lane < p.head_size;
  constexpr int kTeams = kThreads / TEAM;
  for (int i0 = team; i0 < items; i0 += kTeams * kAhead) {
    u32x4 raws[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const Item it = item_of(min(i0 + a * kTeams, items - 1), p.num_heads);  // (past the end: the last one, not written)
      const int64_t src_row = t.first + it.token;
      const char *src = (it.is_v ? p.value + src_row * p.value_stride * 2 : p.key + src_row * p.key_stride * 2) +
                        ((int64_t)it.head * p.head_size + 8 * (live ? lane : 0)) * 2;
      if constexpr (ALIGNED) {
        raws[a] = *reinterpret_cast<const u32x4 *>(src);
      } else {
        const uint16_t *e = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) raws[a][i] = (unsigned)e[2 * i] | (unsigned)e[2 * i + 1] << 16;
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (i0 + a * kTeams >= items) break;
      const Item it = item_of(i0 + a * kTeams, p.num_heads);
      const int head = it.head;
      char *row = (it.is_v ? t.v : t.k) + (int64_t)it.token * p.row_bytes;
      const u32x4 raw = live ? raws[a] : (u32x4){0, 0, 0, 0};
      float x[8], lo = INFINITY, hi = -INFINITY, finite = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = widen<F16>(raw[i >> 1], i & 1);
        finite = __builtin_fmaf(x[i], 0.f, finite);  // (NaN from the first infinity or NaN on)
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
      }
      if (!live) lo = INFINITY, hi = -INFINITY;
      lo = over_team<TEAM>(lo, [](float u, float v) { return fminf(u, v); });
      hi = over_team<TEAM>(hi, [](float u, float v) { return fmaxf(u, v); });
      const unsigned long long any = __ballot(finite != 0.f);
      const unsigned long long mine = (any >> ((threadIdx.x & 63) / TEAM * TEAM)) & ((1ull << TEAM) - 1);
      unsigned zero16 = vtkv::f32_to_bf16_bits_rne(lo);
      const float zero = vtkv::bf16_bits_to_f32((uint16_t)zero16);
      const float range = hi - zero;
      unsigned scale16 = vtkv::f32_to_bf16_bits_rne(range / 15.0f);
      float scale = vtkv::bf16_bits_to_f32((uint16_t)scale16);
      const bool bad = mine != 0 || (vtkv::f32_bits(range) & 0x7f800000u) == 0x7f800000u;
      float half_step = 0.5f * scale, inverse = __builtin_amdgcn_rcpf(scale) * (1.f - 0x1p-20f);
      if (bad || scale < 1.17549435e-38f)  // (a negative one, too: every value equal, zero rounded up)
        scale = inverse = 0.f, scale16 = 0, half_step = INFINITY;
      unsigned word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // The quotient's code or the one below it (the reciprocal is cut by more than it can be too large), then the exact
        // remainder against half a step: a value on the border between two codes takes the upper one.  (16-bit values over a
        // bf16 step meet that border in one of some hundred values.)
        const float d = x[i] - zero, c = __builtin_floorf(__builtin_fmaf(d, inverse, 0.5f));
        const int code = (int)c + (__builtin_fmaf(-c, scale, d) >= half_step ? 1 : 0);
        word |= (unsigned)min(max(code, 0), 15) << (4 * i);
      }
      if (bad) scale16 = zero16 = 0x7fc0u;
      if (live) *reinterpret_cast<unsigned *>(row + head * half + 4 * lane) = word;
      if (lane == 0) *reinterpret_cast<unsigned *>(row + p.num_heads * half + 4 * head) = scale16 | zero16 << 16;
      if (head == p.num_heads - 1)
        for (int i = p.num_heads * (half + 4) + 4 * lane; i < p.row_bytes; i += 4 * TEAM)
          *reinterpret_cast<unsigned *>(row + i) = 0;
    }
  }
}

template <int DT, bool ALIGNED, int TEAM>
__global__ void __launch_bounds__(kThreads) int4_read_kernel(RowsParams p) {
  const Tokens t = tokens_of(p);
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int half = p.head_size / 2, items = max(t.rows, 0) * 2 * p.num_heads;
  if (8 * lane >= p.head_size) return;
  constexpr int kTeams = kThreads / TEAM;
  for (int i0 = team; i0 < items; i0 += kTeams * kAhead) {
    unsigned codes[kAhead], pairs[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const Item it = item_of(min(i0 + a * kTeams, items - 1), p.num_heads);
      const char *row = (it.is_v ? t.v : t.k) + (int64_t)it.token * p.row_bytes;
      codes[a] = *reinterpret_cast<const unsigned *>(row + it.head * half + 4 * lane);
      pairs[a] = *reinterpret_cast<const unsigned *>(row + p.num_heads * half + 4 * it.head);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (i0 + a * kTeams >= items) break;
      const Item it = item_of(i0 + a * kTeams, p.num_heads);
      const float scale = vtkv::bits_f32(pairs[a] << 16), zero = vtkv::bits_f32(pairs[a] & 0xffff0000u);
      char *dst = const_cast<char *>(it.is_v ? p.value : p.key);
      const int64_t e0 = (t.first + it.token) * (it.is_v ? p.value_stride : p.key_stride) + (int64_t)it.head * p.head_size + 8 * lane;
      constexpr int kElem = DT == VTKV_F32 ? 4 : 2;
      unsigned out[2 * kElem];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // (code * scale has 12 significant bits: the one rounding to fp32 is the addition's)
        const float x = __builtin_fmaf((float)((codes[a] >> (4 * e)) & 15u), scale, zero);
        if constexpr (DT == VTKV_F32) {
          out[e] = vtkv::f32_bits(x);
        } else {
          const unsigned h = DT == VTKV_BF16 ? (unsigned)vtkv::f32_to_bf16_bits_rne(x)
                                             : (unsigned)__builtin_bit_cast(unsigned short, (_Float16)x);
          out[e / 2] = e & 1 ? out[e / 2] | h << 16 : h;
        }
      }
      if constexpr (ALIGNED) {
#pragma unroll
        for (int w = 0; w < 2 * kElem; w += 4)
          *reinterpret_cast<u32x4 *>(dst + e0 * kElem + 4 * w) = (u32x4){out[w], out[w + 1], out[w + 2], out[w + 3]};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (DT == VTKV_F32) reinterpret_cast<unsigned *>(dst)[e0 + e] = out[e];
          else reinterpret_cast<uint16_t *>(dst)[e0 + e] = (uint16_t)(out[e / 2] >> (16 * (e & 1)));
        }
      }
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
  const dim3 grid((unsigned)batch, (unsigned)((max_seq_len + kTokens - 1) / kTokens));
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
  const dim3 grid((unsigned)batch, (unsigned)((max_seq_len + kTokens - 1) / kTokens));
  hipStream_t st = (hipStream_t)stream;
  const int esize = dst_dtype == VTKV_F32 ? 4 : 2;
  const bool aligned = key_stride * esize % 16 == 0 && value_stride * esize % 16 == 0 && (uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0;
  typedef void (*Kernel)(RowsParams);
  static const Kernel kernels[3][2][2] = {
      {{int4_read_kernel<VTKV_F32, false, 16>, int4_read_kernel<VTKV_F32, false, 32>},
       {int4_read_kernel<VTKV_F32, true, 16>, int4_read_kernel<VTKV_F32, true, 32>}},
      {{int4_read_kernel<VTKV_BF16, false, 16>, int4_read_kernel<VTKV_BF16, false, 32>},
       {int4_read_kernel<VTKV_BF16, true, 16>, int4_read_kernel<VTKV_BF16, true, 32>}},
      {{int4_read_kernel<VTKV_F16, false, 16>, int4_read_kernel<VTKV_F16, false, 32>},
       {int4_read_kernel<VTKV_F16, true, 16>, int4_read_kernel<VTKV_F16, true, 32>}}};
  const int type = dst_dtype == VTKV_F32 ? 0 : dst_dtype == VTKV_BF16 ? 1 : 2;
  hipLaunchKernelGGL(kernels[type][aligned][head_size > 128], grid, dim3(kThreads), 0, st, p);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

}  // extern "C"
