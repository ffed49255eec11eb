// Attention over a 4-bit cache, the simple form: one workgroup per (query row, kv head) walks over all rows that the
// query row sees, 256 at a time, with a running maximum and sum per query head (one pass).
//
// Lane r of the workgroup computes row r's logits: S = scale * (s_r (q . codes_r) + z_r sum(q)) straight from the
// codes.  Then lane d accumulates O_d = sum_r (p_r s_r) code_rd + sum_r p_r z_r.  All in fp32 on the vector unit.
#include "vtkv_attn_common.h"
#include "vtkv_common.h"
#include "vtkv_int4.h"

#include <cmath>

namespace {

using namespace vtkv_attn;

constexpr int kThreads = 256;
constexpr int kMaxGroup = 16;

struct Int4Params {
  const uint16_t *q;
  const int64_t *k_ptrs, *v_ptrs, *slot_ids;
  const int32_t *seq_lens;
  const int32_t *units;
  const float *alibi_slopes;
  void *out;
  int64_t q_stride;
  int num_heads, num_kv_heads, group, kv_split, group_real;  // (as the kernel sees them: see first_head_of)
  int head_size, row_bytes, unit_tokens, max_seq_len, out_f32, f16;
  float scale_log2;
};

__global__ void __launch_bounds__(kThreads) int4_attention_simple_kernel(Int4Params p) {
  __shared__ float sm_q[kMaxGroup][256];
  __shared__ float sm_p[kMaxGroup][kThreads];
  __shared__ float sm_zero[kThreads], sm_scale[kThreads], sm_alpha[kMaxGroup], sm_l[kMaxGroup], sm_m[kMaxGroup], sm_qsum[kMaxGroup];
  const int kvh = blockIdx.y, tid = threadIdx.x;
  int seq, qrow, len;
  if (p.units) {
    const int u = blockIdx.x / p.unit_tokens, t = blockIdx.x % p.unit_tokens;
    if (t >= p.units[4 * u + 2]) return;
    seq = p.units[4 * u];
    qrow = p.units[4 * u + 1] + t;
    len = p.units[4 * u + 3] + t + 1;
  } else {
    seq = qrow = blockIdx.x;
    len = p.seq_lens[seq];
  }
  len = min(len, p.max_seq_len);
  const int D = p.head_size, G = heads_of(p, kvh), head0 = first_head_of(p, kvh), real = real_kv_head(p, kvh);
  const int kv_real = p.num_kv_heads / p.kv_split;
  const int64_t slot = p.slot_ids[seq];
  const char *k_base = (const char *)(uintptr_t)p.k_ptrs[slot], *v_base = (const char *)(uintptr_t)p.v_ptrs[slot];
  const int code_off = real * (D / 2), sz_off = kv_real * (D / 2) + 4 * real;
  for (int i = tid; i < G * D; i += kThreads) {
    const uint16_t raw = p.q[(int64_t)qrow * p.q_stride + (int64_t)(head0 + i / D) * D + i % D];
    sm_q[i / D][i % D] = p.f16 ? (float)__builtin_bit_cast(_Float16, raw) : vtkv::bf16_bits_to_f32(raw);
  }
  if (tid < kMaxGroup) {
    sm_m[tid] = -INFINITY;
    sm_l[tid] = 0.f;
  }
  __syncthreads();
  if (tid < G) {
    float s = 0.f;
    for (int d = 0; d < D; ++d) s += sm_q[tid][d];
    sm_qsum[tid] = s;
  }
  __syncthreads();
  float o[kMaxGroup];
  for (int h = 0; h < kMaxGroup; ++h) o[h] = 0.f;
  for (int t0 = 0; t0 < len; t0 += kThreads) {
    const int row = t0 + tid;
    const bool valid = row < len;
    float acc[kMaxGroup];
    for (int h = 0; h < kMaxGroup; ++h) acc[h] = 0.f;
    float scale = 0.f, zero = 0.f;
    if (valid) {
      const char *kr = k_base + (int64_t)row * p.row_bytes;
      for (int w = 0; w < D / 8; ++w) {
        const unsigned c = *reinterpret_cast<const unsigned *>(kr + code_off + 4 * w);
        for (int e = 0; e < 8; ++e) {
          const float x = (float)((c >> (4 * e)) & 15u);
#pragma unroll
          for (int h = 0; h < kMaxGroup; ++h)
            if (h < G) acc[h] += x * sm_q[h][8 * w + e];
        }
      }
      const unsigned sz = *reinterpret_cast<const unsigned *>(kr + sz_off);
      scale = __builtin_bit_cast(float, sz << 16);
      zero = __builtin_bit_cast(float, sz & 0xffff0000u);
      const unsigned vz = *reinterpret_cast<const unsigned *>(v_base + (int64_t)row * p.row_bytes + sz_off);
      sm_scale[tid] = __builtin_bit_cast(float, vz << 16);
      sm_zero[tid] = __builtin_bit_cast(float, vz & 0xffff0000u);
    }
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h)
      if (h < G) {
        const float slope = p.alibi_slopes ? p.alibi_slopes[head0 + h] * kLog2e : 0.f;
        const float x = (scale * acc[h] + zero * sm_qsum[h]) * p.scale_log2 + slope * (float)(row - len + 1);
        sm_p[h][tid] = valid ? x : -INFINITY;
      }
    __syncthreads();
    const int wave = tid >> 6, lane = tid & 63;
    for (int h = wave; h < G; h += kThreads / 64) {
      float m = -INFINITY;
      for (int i = lane; i < kThreads; i += 64) m = fmaxf(m, sm_p[h][i]);
      for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
      const float m_old = sm_m[h], m_new = fmaxf(m_old, m);
      // (every logit so far -inf: the weights are exp2(-inf - 0) = 0)
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      float l = 0.f;
      for (int i = lane; i < kThreads; i += 64) {
        const float w = t0 + i < len ? __builtin_amdgcn_exp2f(sm_p[h][i] - ref) : 0.f;
        sm_p[h][i] = w;
        l += w;
      }
      for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
      const float alpha = __builtin_amdgcn_exp2f(m_old - ref);
      if (lane == 0) {
        sm_alpha[h] = alpha;
        sm_l[h] = sm_l[h] * alpha + l;
        sm_m[h] = m_new;
      }
    }
    __syncthreads();
    if (tid < D) {
      for (int h = 0; h < G; ++h) o[h] *= sm_alpha[h];
      const int rows = min(kThreads, len - t0);
      const char *vr = v_base + (int64_t)t0 * p.row_bytes + code_off + tid / 2;
      for (int r = 0; r < rows; ++r, vr += p.row_bytes) {
        const unsigned c = (*(const uint8_t *)vr >> (4 * (tid & 1))) & 15u;
        const float v = __builtin_fmaf((float)c, sm_scale[r], sm_zero[r]);
#pragma unroll
        for (int h = 0; h < kMaxGroup; ++h)
          if (h < G) o[h] += sm_p[h][r] * v;
      }
    }
    __syncthreads();
  }
  if (tid < D)
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h)
      if (h < G) {
        const float r = len > 0 ? o[h] / sm_l[h] : 0.f;
        const int64_t at = ((int64_t)qrow * p.num_heads + head0 + h) * D + tid;
        if (p.out_f32) reinterpret_cast<float *>(p.out)[at] = r;
        else reinterpret_cast<uint16_t *>(p.out)[at] = p.f16 ? f32_to_16<true>(r) : f32_to_16<false>(r);
      }
}

}  // namespace

namespace vtkv {

int int4_attention(void *out, const void *q, const int64_t *k_ptrs, const int64_t *v_ptrs, const int64_t *slot_ids,
                   const int32_t *seq_lens, const int32_t *units, int unit_tokens, int num_rows, int num_heads,
                   int num_kv_heads, int head_size, int64_t q_stride, float scale, int max_seq_len,
                   const float *alibi_slopes, int q_dtype, int out_dtype, void *workspace, int64_t workspace_bytes,
                   void *stream) {
  VTKV_REQUIRE(out && q && k_ptrs && v_ptrs && slot_ids && (seq_lens || units), "null argument");
  VTKV_REQUIRE(num_rows >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
               "num_heads %d must be a positive multiple of num_kv_heads %d", num_heads, num_kv_heads);
  VTKV_REQUIRE(int4_head_size(head_size), "head_size %d is not supported (64, 80, 96, 112, 128, 256)", head_size);
  VTKV_REQUIRE(q_dtype == VTKV_BF16 || q_dtype == VTKV_F16, "a 4-bit cache serves bfloat16 and float16 queries");
  VTKV_REQUIRE(out_dtype == q_dtype || out_dtype == VTKV_F32, "out_dtype must be q_dtype or F32");
  VTKV_REQUIRE(q_stride >= (int64_t)num_heads * head_size && q_stride % 8 == 0 && (uintptr_t)q % 16 == 0,
               "q rows must be 16-byte aligned and at least num_heads*head_size apart");
  VTKV_REQUIRE(max_seq_len > 0, "max_seq_len must be > 0");
  const int group_real = num_heads / num_kv_heads, split = vtkv_kv_split(group_real);
  VTKV_REQUIRE(num_kv_heads * split <= 65535, "too many kv heads");
  VTKV_REQUIRE(int4_row_bytes(num_kv_heads, head_size) < (4 << 20), "rows of 4 MiB and more are not supported");
  if (num_rows == 0) return VTKV_OK;
  if (!units)
    return int4_decode(out, q, k_ptrs, v_ptrs, slot_ids, seq_lens, num_rows, num_heads, num_kv_heads, head_size, q_stride,
                       scale, max_seq_len, alibi_slopes, q_dtype, out_dtype, workspace, workspace_bytes, stream);
  Int4Params p;
  p.q = (const uint16_t *)q;
  p.k_ptrs = k_ptrs;
  p.v_ptrs = v_ptrs;
  p.slot_ids = slot_ids;
  p.seq_lens = seq_lens;
  p.units = units;
  p.alibi_slopes = alibi_slopes;
  p.out = out;
  p.q_stride = q_stride;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads * split;
  p.group = (group_real + split - 1) / split;
  p.kv_split = split;
  p.group_real = group_real;
  p.head_size = head_size;
  p.row_bytes = (int)int4_row_bytes(num_kv_heads, head_size);
  p.unit_tokens = unit_tokens > 0 ? unit_tokens : 1;
  p.max_seq_len = max_seq_len;
  p.out_f32 = out_dtype == VTKV_F32;
  p.f16 = q_dtype == VTKV_F16;
  p.scale_log2 = scale * kLog2e;
  hipLaunchKernelGGL(int4_attention_simple_kernel, dim3((unsigned)num_rows, (unsigned)p.num_kv_heads), dim3(kThreads), 0,
                     (hipStream_t)stream, p);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

}  // namespace vtkv
