// A cache of a bounded number of rows: how much attention each cached row has drawn, and the eviction of the rows
// that drew least.
//
//  * weights[slot, kv head, row] += sum over the kv head's query heads of softmax_row(scale q . k [+ alibi]): one
//    workgroup per (sequence, kv head) reads K twice, first for the maximum and the sum of every query head, then for
//    the weights.
//  * evict: per (sequence, kv head) the last `recent` rows stay, and of the rows before them the `keep - recent` with
//    the largest weight (of equal ones those that come first).  The survivors that lie behind place keep - recent move
//    into the places of the evicted rows before it, in order, and the recent rows move behind them: no more rows move
//    than have to, and the recent rows, which the next steps append to, stay in the order of their tokens.
#include "vtkv_attn_common.h"
#include "vtkv_common.h"
#include "vtkv_int4.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace vtkv_attn;

constexpr int kWeightThreads = 256;
constexpr int kMaxGroup = 16;

struct WeightParams {
  float *weights;
  int64_t slot_stride, head_stride, num_slots;
  const uint16_t *q;  // (float32 models: float)
  const int64_t *k_ptrs, *slot_ids;
  const int32_t *seq_lens;
  const float *alibi_slopes;
  int64_t q_stride;
  int num_heads, num_kv_heads, head_size, row_bytes, max_seq_len, q_dtype, kv_dtype;
  float scale_log2;
};

__device__ __forceinline__ float load_elem(const char *p, int i, int dtype) {
  if (dtype == VTKV_F32) return reinterpret_cast<const float *>(p)[i];
  if (dtype == VTKV_BF16) return vtkv::bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
  if (dtype == VTKV_F16) return (float)reinterpret_cast<const _Float16 *>(p)[i];
  return vtkv::fp8_e4m3fn_decode(reinterpret_cast<const uint8_t *>(p)[i]);
}

__global__ void __launch_bounds__(kWeightThreads) attention_weights_simple_kernel(WeightParams p) {
  __shared__ float sm_q[kMaxGroup][256];
  __shared__ float sm_red[kMaxGroup][4];
  const int kvh = blockIdx.y, seq = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t slot = p.slot_ids[seq];
  const int len = min(p.seq_lens[seq], p.max_seq_len);
  if (len <= 0 || slot < 0 || slot >= p.num_slots) return;
  const int D = p.head_size, G = p.num_heads / p.num_kv_heads;
  const bool int4 = p.kv_dtype == VTKV_INT4;
  const char *k_base = (const char *)(uintptr_t)p.k_ptrs[slot];
  const int eb = p.kv_dtype == VTKV_F32 ? 4 : p.kv_dtype == VTKV_FP8_E4M3 ? 1 : 2;
  const int head_off = int4 ? kvh * (D / 2) : kvh * D * eb, sz_off = p.num_kv_heads * (D / 2) + 4 * kvh;
  float *w = p.weights + slot * p.slot_stride + kvh * p.head_stride;
  for (int h0 = 0; h0 < G; h0 += kMaxGroup) {
    const int n = min(kMaxGroup, G - h0);
    __syncthreads();
    for (int i = tid; i < n * D; i += kWeightThreads)
      sm_q[i / D][i % D] = load_elem((const char *)p.q + ((int64_t)seq * p.q_stride + (int64_t)(kvh * G + h0 + i / D) * D) *
                                                             (p.q_dtype == VTKV_F32 ? 4 : 2), i % D, p.q_dtype);
    __syncthreads();
    auto logits = [&](int row, float (&x)[kMaxGroup]) {
      float acc[kMaxGroup];
      for (int h = 0; h < kMaxGroup; ++h) acc[h] = 0.f;
      const char *kr = k_base + (int64_t)row * p.row_bytes;
      float scale = 1.f, zero = 0.f;
      if (int4) {
        const unsigned sz = *reinterpret_cast<const unsigned *>(kr + sz_off);
        scale = __builtin_bit_cast(float, sz << 16);
        zero = __builtin_bit_cast(float, sz & 0xffff0000u);
      }
      for (int d = 0; d < D; ++d) {
        const float k = int4 ? __builtin_fmaf((float)((((const uint8_t *)kr)[head_off + d / 2] >> (4 * (d & 1))) & 15), scale, zero)
                             : load_elem(kr + head_off, d, p.kv_dtype);
#pragma unroll
        for (int h = 0; h < kMaxGroup; ++h)
          if (h < n) acc[h] += k * sm_q[h][d];
      }
#pragma unroll
      for (int h = 0; h < kMaxGroup; ++h)
        if (h < n) {
          const float slope = p.alibi_slopes ? p.alibi_slopes[kvh * G + h0 + h] * kLog2e : 0.f;
          x[h] = acc[h] * p.scale_log2 + slope * (float)(row - len + 1);
        }
    };
    float m[kMaxGroup], l[kMaxGroup];
    for (int h = 0; h < kMaxGroup; ++h) m[h] = -INFINITY, l[h] = 0.f;
    for (int row = tid; row < len; row += kWeightThreads) {
      float x[kMaxGroup];
      logits(row, x);
#pragma unroll
      for (int h = 0; h < kMaxGroup; ++h)
        if (h < n) {
          const float m_new = fmaxf(m[h], x[h]);
          const float ref = m_new == -INFINITY ? 0.f : m_new;
          l[h] = l[h] * __builtin_amdgcn_exp2f(m[h] - ref) + __builtin_amdgcn_exp2f(x[h] - ref);
          m[h] = m_new;
        }
    }
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h)
      if (h < n) {
        float mm = m[h];
        for (int d = 32; d; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
        __syncthreads();
        if (lane == 0) sm_red[h][wave] = mm;
        __syncthreads();
        mm = fmaxf(fmaxf(sm_red[h][0], sm_red[h][1]), fmaxf(sm_red[h][2], sm_red[h][3]));
        if (mm == -INFINITY) mm = 0.f;
        float ll = l[h] * __builtin_amdgcn_exp2f(m[h] - mm);
        for (int d = 32; d; d >>= 1) ll += __shfl_xor(ll, d);
        __syncthreads();
        if (lane == 0) sm_red[h][wave] = ll;
        __syncthreads();
        m[h] = mm;
        l[h] = 1.f / (sm_red[h][0] + sm_red[h][1] + sm_red[h][2] + sm_red[h][3]);
      }
    for (int row = tid; row < len; row += kWeightThreads) {
      float x[kMaxGroup], sum = 0.f;
      logits(row, x);
#pragma unroll
      for (int h = 0; h < kMaxGroup; ++h)
        if (h < n) sum += __builtin_amdgcn_exp2f(x[h] - m[h]) * l[h];
      w[row] += sum;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;

struct EvictParams {
  const int64_t *k_ptrs, *v_ptrs, *slot_ids;
  float *weights;
  int64_t slot_stride, head_stride, num_slots;
  const int32_t *seq_lens;
  int32_t *new_seq_lens;
  int32_t *pairs;  // [num_seqs, num_kv_heads, 2, pair_cap]: places to fill, rows that fill them
  int pair_cap, keep, recent, max_seq_len;
  int num_kv_heads, row_bytes;
  int head_bytes, tail_off;  // bytes of one head in a row; 4-bit rows: where the (scale, zero) pairs start, else -1
};

// Larger weight <-> larger key; +0 and -0 are the same weight.
__device__ __forceinline__ unsigned weight_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int UNIT>
struct Unit;
template <>
struct Unit<16> {
  typedef unsigned T __attribute__((ext_vector_type(4)));
};
template <>
struct Unit<8> {
  typedef unsigned T __attribute__((ext_vector_type(2)));
};

template <int UNIT>
__global__ void __launch_bounds__(kEvictThreads) evict_simple_kernel(EvictParams p) {
  typedef typename Unit<UNIT>::T vec;
  __shared__ unsigned sm_hist[256];
  __shared__ unsigned sm_pick[2];
  __shared__ int sm_wave[kEvictWaves][3];
  const int kvh = blockIdx.y, seq = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int n = min(p.seq_lens[seq], p.max_seq_len);
  if (kvh == 0 && tid == 0) p.new_seq_lens[seq] = max(0, min(n, p.keep));
  const int64_t slot = p.slot_ids[seq];
  if (n <= p.keep || slot < 0 || slot >= p.num_slots) return;
  const int heavy = p.keep - p.recent, old = n - p.recent;  // old > heavy >= 0
  float *w = p.weights + slot * p.slot_stride + kvh * p.head_stride;
  int32_t *holes = p.pairs + ((int64_t)seq * p.num_kv_heads + kvh) * 2 * p.pair_cap, *movers = holes + p.pair_cap;

  // ---- the key of the last row that stays, a byte at a time from the top, and how many of its equals stay
  unsigned prefix = 0, rest = (unsigned)heavy;
  if (heavy > 0)
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) sm_hist[tid] = 0;
      __syncthreads();
      const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int i = tid; i < old; i += kEvictThreads) {
        const unsigned k = weight_key(w[i]);
        if ((k & mask) == prefix) atomicAdd(&sm_hist[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        unsigned left = rest;
        int d = 255;
        while (sm_hist[d] < left) left -= sm_hist[d--];
        sm_pick[0] = (unsigned)d;
        sm_pick[1] = left;
      }
      __syncthreads();
      prefix |= sm_pick[0] << shift;
      rest = sm_pick[1];
    }

  // ---- places and movers in order: each wave walks over its share of the old rows
  const int share = ((old + kEvictWaves - 1) / kEvictWaves + 63) / 64 * 64;
  const int begin = min(old, wave * share), end = min(old, begin + share);
  int before_eq = 0, before_hole = 0, before_mover = 0;
  for (int pass = 0; pass < 3; ++pass) {  // 0: equals per wave; 1: places and movers per wave; 2: the lists
    int eq = before_eq, hole = pass == 2 ? before_hole : 0, mover = pass == 2 ? before_mover : 0;
    for (int i0 = begin; i0 < end; i0 += 64) {
      const int i = i0 + lane;
      const unsigned k = i < end ? weight_key(w[i]) : 0u;
      const bool is_eq = i < end && heavy > 0 && k == prefix;
      const unsigned long long eqs = __ballot(is_eq), below = (1ull << lane) - 1;
      if (pass > 0) {
        const bool stays = i < end && heavy > 0 && (k > prefix || (is_eq && eq + __popcll(eqs & below) < (int)rest));
        const bool is_hole = i < end && !stays && i < heavy, is_mover = stays && i >= heavy;
        const unsigned long long hs = __ballot(is_hole), ms = __ballot(is_mover);
        if (pass == 2) {
          if (is_hole) holes[hole + __popcll(hs & below)] = i;
          if (is_mover) movers[mover + __popcll(ms & below)] = i;
        }
        hole += __popcll(hs);
        mover += __popcll(ms);
      }
      eq += __popcll(eqs);
    }
    if (pass == 2) break;
    __syncthreads();
    if (lane == 0) {
      sm_wave[wave][0] = eq;
      sm_wave[wave][1] = hole;
      sm_wave[wave][2] = mover;
    }
    __syncthreads();
    for (int v = 0; v < wave; ++v) {
      if (pass == 0) before_eq += sm_wave[v][0];
      before_hole += sm_wave[v][1];
      before_mover += sm_wave[v][2];
    }
  }
  int pairs = 0;
  __syncthreads();
  for (int v = 0; v < kEvictWaves; ++v) pairs += sm_wave[v][2];  // (as many movers as places)
  __syncthreads();

  // ---- the survivors into their places
  char *base[2] = {reinterpret_cast<char *>(p.k_ptrs[slot]), reinterpret_cast<char *>(p.v_ptrs[slot])};
  const int units = p.head_bytes / UNIT;
  const int64_t head_off = (int64_t)kvh * p.head_bytes;
  for (int j = tid; j < pairs * units * 2; j += kEvictThreads) {
    const int pair = j / (2 * units), u = j % (2 * units), side = u >= units;
    const int64_t off = head_off + (int64_t)(u - side * units) * UNIT;
    *reinterpret_cast<vec *>(base[side] + (int64_t)holes[pair] * p.row_bytes + off) =
        *reinterpret_cast<const vec *>(base[side] + (int64_t)movers[pair] * p.row_bytes + off);
  }
  for (int j = tid; j < pairs; j += kEvictThreads) {
    w[holes[j]] = w[movers[j]];
    if (p.tail_off >= 0)
      for (int side = 0; side < 2; ++side)
        *reinterpret_cast<unsigned *>(base[side] + (int64_t)holes[j] * p.row_bytes + p.tail_off + 4 * kvh) =
            *reinterpret_cast<const unsigned *>(base[side] + (int64_t)movers[j] * p.row_bytes + p.tail_off + 4 * kvh);
  }
  __syncthreads();
  // ---- the recent rows behind them, lowest first: a row moves down, so what a step overwrites has been read by it
  // or by a step before
  const int per_row = 2 * units, rows_step = std::max(1, kEvictThreads / per_row);
  for (int r0 = 0; r0 < p.recent; r0 += rows_step) {
    const int r = r0 + tid / per_row, u = tid % per_row, side = u >= units;
    const bool live = tid / per_row < rows_step && r < p.recent;
    const int64_t off = head_off + (int64_t)(u - side * units) * UNIT;
    vec v;
    unsigned tail = 0;
    float weight = 0.f;
    if (live) {
      v = *reinterpret_cast<const vec *>(base[side] + (int64_t)(old + r) * p.row_bytes + off);
      if (u == 0) weight = w[old + r];
      if (p.tail_off >= 0 && off == head_off)
        tail = *reinterpret_cast<const unsigned *>(base[side] + (int64_t)(old + r) * p.row_bytes + p.tail_off + 4 * kvh);
    }
    __syncthreads();
    if (live) {
      *reinterpret_cast<vec *>(base[side] + (int64_t)(heavy + r) * p.row_bytes + off) = v;
      if (u == 0) w[heavy + r] = weight;
      if (p.tail_off >= 0 && off == head_off)
        *reinterpret_cast<unsigned *>(base[side] + (int64_t)(heavy + r) * p.row_bytes + p.tail_off + 4 * kvh) = tail;
    }
    __syncthreads();
  }
  for (int i = p.keep + tid; i < n; i += kEvictThreads) w[i] = 0.f;
}

}  // namespace

extern "C" {

int64_t vtkv_accumulate_attention_weights_workspace_bytes(int num_seqs, int num_heads, int max_seq_len) {
  (void)num_seqs, (void)num_heads, (void)max_seq_len;
  return 0;
}

int vtkv_accumulate_attention_weights(float *weights, int64_t slot_stride, int64_t head_stride, int64_t num_slots,
                                      const void *q, const int64_t *k_ptrs, const int64_t *slot_ids,
                                      const int32_t *seq_lens, int num_seqs, int num_heads, int num_kv_heads,
                                      int head_size, int64_t q_stride, float scale, int max_seq_len,
                                      const float *alibi_slopes, int q_dtype, int kv_dtype, float k_scale,
                                      void *workspace, int64_t workspace_bytes, void *stream) {
  VTKV_REQUIRE(weights && q && k_ptrs && slot_ids && seq_lens, "null argument");
  VTKV_REQUIRE(num_seqs >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
               "num_heads %d must be a positive multiple of num_kv_heads %d", num_heads, num_kv_heads);
  VTKV_REQUIRE(vtkv::int4_head_size(head_size), "head_size %d is not supported (64, 80, 96, 112, 128, 256)", head_size);
  VTKV_REQUIRE(q_dtype == VTKV_BF16 || q_dtype == VTKV_F16, "q_dtype must be BF16 or F16");
  VTKV_REQUIRE(kv_dtype == q_dtype || kv_dtype == VTKV_FP8_E4M3 || kv_dtype == VTKV_INT4,
               "kv_dtype must be q_dtype, FP8_E4M3 or INT4");
  VTKV_REQUIRE(kv_dtype != VTKV_FP8_E4M3 || k_scale > 0.f, "fp8 scales must be positive");
  VTKV_REQUIRE(q_stride >= (int64_t)num_heads * head_size && q_stride % 8 == 0 && (uintptr_t)q % 16 == 0,
               "q rows must be 16-byte aligned and at least num_heads*head_size apart");
  VTKV_REQUIRE(max_seq_len > 0 && num_slots > 0, "max_seq_len and num_slots must be > 0");
  VTKV_REQUIRE(num_kv_heads <= 65535, "too many kv heads");
  if (num_seqs == 0) return VTKV_OK;
  WeightParams p;
  p.weights = weights;
  p.slot_stride = slot_stride;
  p.head_stride = head_stride;
  p.num_slots = num_slots;
  p.q = (const uint16_t *)q;
  p.k_ptrs = k_ptrs;
  p.slot_ids = slot_ids;
  p.seq_lens = seq_lens;
  p.alibi_slopes = alibi_slopes;
  p.q_stride = q_stride;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_size = head_size;
  p.row_bytes = (int)vtkv_kv_row_bytes(num_kv_heads, head_size, kv_dtype);
  p.max_seq_len = max_seq_len;
  p.q_dtype = q_dtype;
  p.kv_dtype = kv_dtype;
  p.scale_log2 = scale * kLog2e * (kv_dtype == VTKV_FP8_E4M3 ? k_scale : 1.f);
  hipLaunchKernelGGL(attention_weights_simple_kernel, dim3((unsigned)num_seqs, (unsigned)num_kv_heads), dim3(kWeightThreads),
                     0, (hipStream_t)stream, p);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

int64_t vtkv_evict_rows_workspace_bytes(int num_seqs, int num_kv_heads, int max_seq_len, int keep_rows, int recent_rows) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || keep_rows < 0 || recent_rows < 0 || recent_rows > keep_rows) return 0;
  const int64_t cap = std::max(0, std::min(keep_rows - recent_rows, max_seq_len - keep_rows));
  return (int64_t)num_seqs * num_kv_heads * 2 * cap * (int64_t)sizeof(int32_t);
}

int vtkv_evict_rows(const int64_t *k_ptrs, const int64_t *v_ptrs, float *weights, int64_t slot_stride,
                    int64_t head_stride, int64_t num_slots, const int64_t *slot_ids, const int32_t *seq_lens,
                    int32_t *new_seq_lens, int num_seqs, int num_kv_heads, int head_size, int kv_dtype, int keep_rows,
                    int recent_rows, int max_seq_len, void *workspace, int64_t workspace_bytes, void *stream) {
  VTKV_REQUIRE(k_ptrs && v_ptrs && weights && slot_ids && seq_lens && new_seq_lens, "null argument");
  VTKV_REQUIRE(num_seqs >= 0 && num_kv_heads > 0 && num_kv_heads <= 65535 && num_slots > 0, "bad sizes");
  VTKV_REQUIRE(vtkv::int4_head_size(head_size), "head_size %d is not supported (64, 80, 96, 112, 128, 256)", head_size);
  VTKV_REQUIRE(kv_dtype == VTKV_F32 || kv_dtype == VTKV_BF16 || kv_dtype == VTKV_F16 || kv_dtype == VTKV_FP8_E4M3 ||
                   kv_dtype == VTKV_INT4, "bad kv_dtype %d", kv_dtype);
  VTKV_REQUIRE(keep_rows > 0 && recent_rows >= 0 && recent_rows <= keep_rows,
               "keep_rows %d must be positive and recent_rows %d between 0 and keep_rows", keep_rows, recent_rows);
  VTKV_REQUIRE(max_seq_len > 0, "max_seq_len must be > 0");
  const int64_t need = vtkv_evict_rows_workspace_bytes(num_seqs, num_kv_heads, max_seq_len, keep_rows, recent_rows);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return vtkv::fail(VTKV_ENOMEM, "workspace of %lld bytes needed, got %lld", (long long)need, (long long)workspace_bytes);
  if (num_seqs == 0) return VTKV_OK;
  EvictParams p;
  p.k_ptrs = k_ptrs;
  p.v_ptrs = v_ptrs;
  p.slot_ids = slot_ids;
  p.weights = weights;
  p.slot_stride = slot_stride;
  p.head_stride = head_stride;
  p.num_slots = num_slots;
  p.seq_lens = seq_lens;
  p.new_seq_lens = new_seq_lens;
  p.pairs = (int32_t *)workspace;
  p.pair_cap = std::max(0, std::min(keep_rows - recent_rows, max_seq_len - keep_rows));
  p.keep = keep_rows;
  p.recent = recent_rows;
  p.max_seq_len = max_seq_len;
  p.num_kv_heads = num_kv_heads;
  p.row_bytes = (int)vtkv_kv_row_bytes(num_kv_heads, head_size, kv_dtype);
  const bool int4 = kv_dtype == VTKV_INT4;
  p.head_bytes = int4 ? head_size / 2 : head_size * vtkv::elem_bytes(kv_dtype);
  p.tail_off = int4 ? num_kv_heads * (head_size / 2) : -1;
  const dim3 grid((unsigned)num_seqs, (unsigned)num_kv_heads);
  hipStream_t st = (hipStream_t)stream;
  if (p.head_bytes % 16 == 0)
    hipLaunchKernelGGL(evict_simple_kernel<16>, grid, dim3(kEvictThreads), 0, st, p);
  else
    hipLaunchKernelGGL(evict_simple_kernel<8>, grid, dim3(kEvictThreads), 0, st, p);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

}  // extern "C"
