// Decode attention over a 4-bit cache for gfx950: one query token per sequence, split-K over spans of equal length.
//
// What it computes with.  A cached value is code * scale + zero with scale and zero of its row (per kv head), so
//
//   logit_r = s_r (q . c_r) + z_r sum(q)            o = sum_r (p_r s_r) c_r + sum_r p_r z_r
//
// and both products run on the matrix pipe with the bare codes as one operand, which never have to be scaled:
//
//  * K: two codes of a word masked in place (word & 0x000f000f, word & 0x00f000f0, the same of word >> 8) are the
//    fp16 numbers c * 2^-24 and c * 2^-20 (denormals, which the fp16 MFMA takes as they are): five instructions for
//    eight codes and no rounding.  The other factor 16 and the 2^24 go into q, which is brought to fp16 by a power of
//    two per head (its largest value near 2^14): exact for bf16 and fp16 queries.
//  * V: the codes of 16 rows come out of LDS transposed (ds_read_b64_tr_b4: lane d of a group gets column d of 16
//    rows); (word >> 4k & 0x000f000f) | 0x43004300 are the bf16 numbers 128 + c.  p s is carried as a bf16 head and a
//    bf16 tail (2^-17 relative); the 128 sum(p s) that come with the codes are subtracted from sum(p z) in fp32, with
//    the same head and tail, so that nothing but fp32 rounding remains of them.
//
// How it moves data.  HBM-bound: 2 rows of 68 bytes per token and kv head (head size 128).  A workgroup takes whole
// rows (or eight kv heads of them): a stage of 64 rows (512 / kv heads when there are fewer than eight) of K and V goes
// from global memory straight into LDS (16 bytes per lane, no registers), two stages deep, so that loads are always in
// flight while the other stage is computed; a row's bytes are fetched once whatever the heads per line.  Each wave
// serves one kv head and 64 rows of the stage.
//
// Group sizes below 16 leave columns of the 16-column tiles free.  A tile's columns are (part j, head): with up to four
// heads the four 16-row tiles of a wave's 64 rows share one tile of logits (J = 4), with up to eight in pairs (J = 2),
// so the softmax arithmetic is per logit that exists; P.V takes the same layout with zeros where a row is not the
// part's, and the parts are added up at the end of a span.
//
// The batch's rows in steps of 16 are cut into as many equal spans as workgroups run; a span that ends inside a
// sequence leaves a partial result in the workspace and a second kernel merges them.
#include "vtkv_attn_common.h"
#include "vtkv_common.h"
#include "vtkv_int4.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace vtkv_attn;

constexpr int kMaxBatch = 1024;   // sequences per launch
constexpr int kPtrTable = 256;    // base addresses held in LDS, of the first so many sequences
constexpr int kTileRows = 64;     // rows of a wave's tile
constexpr int kUnitRows = 16;     // rows by which spans are cut
constexpr int kLdsBytes = 160 * 1024;

constexpr int waves_of(int d) { return d > 128 ? 4 : 8; }
constexpr int loads_of(int d) { return d > 128 ? 9 : 5; }  // 16-byte loads per lane, stage and side at most

struct DecodeParams {
  const uint16_t *q;
  const int64_t *k_ptrs, *v_ptrs, *slot_ids;
  const int32_t *seq_lens;
  const float *alibi_slopes;
  void *out;
  float *part_o;    // [2 * grid][chunk heads][group][D]
  float *part_ml;   // the same without D, (maximum, sum) pairs
  int32_t *cum;     // [num_seqs + 1] units before a sequence
  int64_t q_stride;
  int num_seqs, num_heads, num_kv_heads, kv_split, group, group_real;  // (kv heads as the kernel sees them)
  int row_bytes, max_seq_len, out_f32;
  int chunk_heads, chunks, chunk_real, parts_per_real;  // kv heads of a workgroup; chunks per sequence; real kv heads of one
  int row_tiles;               // 64-row tiles per stage
  int stage_bytes;             // LDS of a stage: K, then V (or the results of its waves, merged when a part ends)
  int code_units, scale_units; // 16-byte pieces of a row in LDS
  int min_units;               // a span's units at least
  float scale_log2;
};

// The spans: unit u of the batch belongs to span u * active / total, each a contiguous range.
__device__ __forceinline__ int active_spans(const DecodeParams &p, int total, int grid) {
  return max(1, min(grid, total / p.min_units));
}
__device__ __forceinline__ int span_begin(int total, int active, int i) { return (int)((int64_t)total * i / active); }

__device__ __forceinline__ int real0_of(const DecodeParams &p, int chunk) {
  return p.kv_split == 1 ? chunk * p.chunk_heads : chunk / p.parts_per_real;
}
// kv head (as the kernel counts them) of place hs of a chunk, -1: none
__device__ __forceinline__ int head_of_chunk(const DecodeParams &p, int chunk, int hs) {
  if (p.kv_split == 1) return chunk * p.chunk_heads + hs;
  const int part = chunk % p.parts_per_real * p.chunk_heads + hs;
  return part < p.kv_split ? chunk / p.parts_per_real * p.kv_split + part : -1;
}

typedef __attribute__((address_space(3))) char *lptr;

// 16 bytes per lane from base + off to lds + 16 * lane (M0 holds lds; nothing else in these kernels uses M0).  Nothing the
// compiler counts: the caller waits (wait_loads).
__device__ __forceinline__ void load_to_lds(uint64_t base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
// Until at most n vector memory instructions are outstanding.  They retire in order, so the older ones are done.
__device__ __forceinline__ void wait_loads(int n) {
#define VTKV_WAIT(N)                                    \
  case N: asm volatile("s_waitcnt vmcnt(" #N ")" ::: "memory"); break;
  switch (n) {
    VTKV_WAIT(2) VTKV_WAIT(4) VTKV_WAIT(6) VTKV_WAIT(8) VTKV_WAIT(10) VTKV_WAIT(12) VTKV_WAIT(14) VTKV_WAIT(16) VTKV_WAIT(18)
    default: asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
#undef VTKV_WAIT
}
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A place in the batch's order (sequence, chunk, row), with the end of the part of it that this span holds.
struct Cursor {
  int b, chunk, row, end, left;  // left: units of the span behind this part
  __device__ __forceinline__ bool valid() const { return end > 0; }
};

template <int D, int J, bool F16>
__global__ void __launch_bounds__(waves_of(D) * 64) int4_decode_kernel(DecodeParams p) {
  constexpr int kWaves = waves_of(D), kThreads = kWaves * 64, kLoads = loads_of(D);
  constexpr int kWords = D / 8, kSteps = (kWords + 3) / 4;  // words of eight codes; MFMA steps over d
  constexpr int kDB = D / 16;
  constexpr int kHeads = 16 / J;  // columns of a part
  constexpr int kE = 4 / J;       // tiles of logits
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_tot[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int j = n / kHeads, h = n % kHeads;  // this lane's column: part and head
  const int B = p.num_seqs, C = p.chunks;
  const int units_row = p.code_units + p.scale_units, pitch = units_row * 16;
  const int stage_rows = p.row_tiles * kTileRows, side_bytes = stage_rows * pitch;
  int *s_cum = reinterpret_cast<int *>(smem + 2 * p.stage_bytes);
  uint64_t *s_ptr = reinterpret_cast<uint64_t *>(smem + 2 * p.stage_bytes + ((B + 1) * 4 + 15) / 16 * 16);

  // ---- units before every sequence, and the base addresses of the first ones
  {
    constexpr int kPer = (kMaxBatch + kThreads - 1) / kThreads;
    int local[kPer], sum = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int idx = tid * kPer + k;
      local[k] = sum;
      if (idx < B) {
        sum += (max(0, min(p.seq_lens[idx], p.max_seq_len)) + kUnitRows - 1) / kUnitRows;
      }
    }
    if (tid < min(B, kPtrTable)) {
      const int64_t slot = p.slot_ids[tid];
      s_ptr[2 * tid] = (uint64_t)p.k_ptrs[slot];
      s_ptr[2 * tid + 1] = (uint64_t)p.v_ptrs[slot];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(incl, d);
      if (lane >= d) incl += t;
    }
    if (lane == 63) s_tot[wave] = incl;
    __syncthreads();
    int excl = incl - sum, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) excl += s_tot[w];
      all += s_tot[w];
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (tid * kPer + k < B) s_cum[tid * kPer + k] = excl + local[k];
    if (tid == 0) s_cum[B] = all;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = tid; i <= B; i += kThreads) p.cum[i] = s_cum[i];
  }
  const int total = uniform(s_cum[B]) * C;
  const int active = active_spans(p, total, gridDim.x);
  if ((int)blockIdx.x >= active || total == 0) return;
  const int u_begin = span_begin(total, active, blockIdx.x), u_end = span_begin(total, active, blockIdx.x + 1);
  if (u_begin >= u_end) return;

  auto len_of = [&](int b) { return uniform(min(p.seq_lens[b], p.max_seq_len)); };
  // the part of sequence b, chunk c from unit k on, as far as `left` units go
  auto enter = [&](Cursor &c, int b, int chunk, int k, int left) {
    const int nb = uniform(s_cum[b + 1]) - uniform(s_cum[b]);
    const int take = min(left, nb - k);
    c.b = b;
    c.chunk = chunk;
    c.row = k * kUnitRows;
    c.end = min(len_of(b), (k + take) * kUnitRows);
    c.left = left - take;
  };
  auto step = [&](Cursor &c) {  // one stage on
    c.row += stage_rows;
    if (c.row < c.end) return;
    if (c.left == 0) {
      c.end = 0;
      return;
    }
    int b = c.b, chunk = c.chunk + 1;
    if (chunk == C) {
      chunk = 0;
      do ++b; while (uniform(s_cum[b + 1]) == uniform(s_cum[b]));  // (ends: `left` units are still to come)
    }
    enter(c, b, chunk, 0, c.left);
  };
  Cursor cc;
  {
    // the last sequence that begins at or before u_begin and has units
    int b = 0;
    for (int i0 = 0; i0 < B; i0 += 64) {
      const int i = i0 + lane;
      const bool before = i < B && (int64_t)s_cum[i] * C <= u_begin && s_cum[i + 1] > s_cum[i];
      const unsigned long long m = __builtin_amdgcn_ballot_w64(before);
      if (m) b = i0 + 63 - __builtin_clzll(m);
    }
    b = uniform(b);
    const int c0 = uniform(s_cum[b]), nb = uniform(s_cum[b + 1]) - c0;
    const int k = u_begin - c0 * C;
    enter(cc, b, k / nb, k % nb, u_end - u_begin);
  }

  // ---- stage loads: 16-byte piece i of a stage's side goes to LDS byte 16 i; lane l of load k of this wave takes
  // piece (wave + waves * k) * 64 + l
  const int pieces = stage_rows * units_row, num_loads = (pieces + 63) / 64;
  int ld_row[kLoads], ld_col[kLoads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int i = (wave + kWaves * k) * 64 + lane;
    ld_row[k] = i / units_row;
    ld_col[k] = i % units_row;
  }
  const int my_loads = wave < num_loads ? (num_loads - wave + kWaves - 1) / kWaves : 0;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr)smem;
  auto issue = [&](const Cursor &c, int buf) {
    uint64_t kb, vb;
    if (c.b < kPtrTable) {
      kb = s_ptr[2 * c.b];
      vb = s_ptr[2 * c.b + 1];
    } else {
      const int64_t slot = p.slot_ids[c.b];
      kb = (uint64_t)p.k_ptrs[slot];
      vb = (uint64_t)p.v_ptrs[slot];
    }
    const uint64_t from = (uint64_t)c.row * p.row_bytes;
    kb = ((uint64_t)uniform((int)(kb >> 32)) << 32 | (uint32_t)uniform((int)kb)) + from;
    vb = ((uint64_t)uniform((int)(vb >> 32)) << 32 | (uint32_t)uniform((int)vb)) + from;
    const int last = min(stage_rows, c.end - c.row) - 1;  // rows past the part's end: its last row again, never used
    const int real0 = real0_of(p, c.chunk);
    const int code0 = p.scale_units ? real0 * (D / 2) / 16 * 16 : 0;
    const int all_codes = p.num_kv_heads / p.kv_split * (D / 2);
    const int scale0 = min((all_codes + 4 * real0) / 16 * 16, p.row_bytes - 16 * p.scale_units) - 16 * p.code_units;
    const uint32_t dst = lds0 + buf * p.stage_bytes + wave * 1024;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      if (wave + kWaves * k >= num_loads) break;
      if ((wave + kWaves * k) * 64 + lane < pieces) {
        const uint32_t off = min(ld_row[k], last) * p.row_bytes + ld_col[k] * 16 + (ld_col[k] < p.code_units ? code0 : scale0);
        load_to_lds(kb, off, dst + k * kWaves * 1024);
        load_to_lds(vb, off, dst + k * kWaves * 1024 + side_bytes);
      }
    }
  };

  // ---- this wave's kv head and rows of the stage
  const int hs = wave % p.chunk_heads, rt = wave / p.chunk_heads;
  const bool has_tile = rt < p.row_tiles;
  const int word0 = kWords % 4 == 0 ? g * (kWords / 4) : g * (kWords / 4) + min(g, kWords % 4);
  const int words = kWords / 4 + (g < kWords % 4 ? 1 : 0);
  u32x4 qop[kSteps];
  float q_back, q_sum, slope;  // logit = s * acc * q_back + z * q_sum [+ slope * distance]
  int k_lane, v_lane, sz_lane, head = -1, len = 0;
  f32x4 acc[kDB];
  float m_run, l_run, corr;
  u32x4 raw[kSteps];
  auto load_q = [&](const Cursor &c) {
    const int v = has_tile ? head_of_chunk(p, c.chunk, hs) : -1;
    const int hv = v < 0 ? 0 : heads_of(p, v), h0 = v < 0 ? 0 : first_head_of(p, v);
    const uint16_t *row = p.q + (int64_t)c.b * p.q_stride + (int64_t)(h0 + min(h, max(hv - 1, 0))) * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      raw[s] = (u32x4){0, 0, 0, 0};
      if (s < words && h < hv) raw[s] = *reinterpret_cast<const u32x4 *>(row + 8 * (word0 + s));
    }
  };
  auto begin = [&](const Cursor &c) {
    head = has_tile ? head_of_chunk(p, c.chunk, hs) : -1;
    len = len_of(c.b);
    float top = 0.f, sum = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = unpack_16<F16>(raw[s][e >> 1], e & 1);
        top = fmaxf(top, fabsf(x));
        sum += x;
      }
    top = max_over_row_groups(top);
    sum = sum_over_row_groups(sum);
    const int expo = min(max((int)(__builtin_bit_cast(unsigned, top) >> 23), 14), 254);
    const float up = __builtin_bit_cast(float, (unsigned)(268 - expo) << 23);  // top * up in [2^14, 2^15)
    q_back = (1.f / up) * 16777216.f * p.scale_log2;
    q_sum = sum * p.scale_log2;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = unpack_16<F16>(raw[s][e >> 1], e & 1) * up;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = r & 1 ? 0.0625f : 1.f;
        qop[s][r] = pack_16x2<true>(x[r] * f, x[r + 4] * f);
      }
    }
    slope = 0.f;
    if (p.alibi_slopes && head >= 0 && h < heads_of(p, head)) slope = p.alibi_slopes[first_head_of(p, head) + h] * kLog2e;
    const int real = head >= 0 ? real_kv_head(p, head) : 0;
    const int real0 = real0_of(p, c.chunk);
    const int code_at = real * (D / 2) - (p.scale_units ? real0 * (D / 2) / 16 * 16 : 0);
    const int all_codes = p.num_kv_heads / p.kv_split * (D / 2);
    const int scale_at = p.scale_units ? p.code_units * 16 + all_codes + 4 * real -
                                             min((all_codes + 4 * real0) / 16 * 16, p.row_bytes - 16 * p.scale_units)
                                       : all_codes + 4 * real;
    // tile t's row of lane m as A operand: 16 t + 4 (m & 3) + m / 4; then a lane group's logits are rows = g mod 4,
    // the 16 rows whose codes its lanes bring together for P.V
    k_lane = (rt * kTileRows + 4 * (n & 3) + (n >> 2)) * pitch + code_at + 4 * word0;
    v_lane = side_bytes + (rt * kTileRows + 4 * n + g) * pitch + code_at;
    sz_lane = (rt * kTileRows + 16 * j + g) * pitch + scale_at;
#pragma unroll
    for (int d = 0; d < kDB; ++d) acc[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY;
    l_run = corr = 0.f;
  };

  auto compute = [&](const Cursor &c, int buf) {
    const int rows = min(kTileRows, c.end - c.row - rt * kTileRows);
    if (head < 0 || rows <= 0) return;
    const char *st = smem + buf * p.stage_bytes;
    f32x4 sa[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const char *at = st + k_lane + 16 * t * pitch;
      unsigned w[kSteps];
      if constexpr (D == 128 || D == 256) {
#pragma unroll
        for (int s = 0; s < kSteps; s += 4) {
          const u32x4 v = *reinterpret_cast<const u32x4 *>(at + 4 * s);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[s + i] = v[i];
        }
      } else if constexpr (D == 64) {
        const u32x2 v = *reinterpret_cast<const u32x2 *>(at);
        w[0] = v[0];
        w[1] = v[1];
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) w[s] = *reinterpret_cast<const unsigned *>(at + 4 * s);
      }
      sa[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const unsigned y = w[s] >> 8;
        const u32x4 a = {w[s] & 0x000f000fu, w[s] & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
        sa[t] = mfma_16x16x32<true>(a, qop[s], sa[t]);
      }
    }
    // x[e][i]: the lane's logit of row 16 (J e + j) + 4 i + g
    float x[kE][4];
    if constexpr (J == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[0][i] = j < 2 ? (j == 0 ? sa[0][i] : sa[1][i]) : (j == 2 ? sa[2][i] : sa[3][i]);
    } else if constexpr (J == 2) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e][i] = j == 0 ? sa[2 * e][i] : sa[2 * e + 1][i];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e][i] = sa[e][i];
    }
    const float ahead = (float)(c.row + rt * kTileRows + 16 * j + g - len + 1);
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned sz = *reinterpret_cast<const unsigned *>(st + sz_lane + (16 * J * e + 4 * i) * pitch);
        const float s = __builtin_bit_cast(float, sz << 16), z = __builtin_bit_cast(float, sz & 0xffff0000u);
        x[e][i] = __builtin_fmaf(s * x[e][i], q_back, z * q_sum) + slope * (ahead + (float)(16 * J * e + 4 * i));
      }
    if (rows < kTileRows) {
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * (J * e + j) + 4 * i + g >= rows) x[e][i] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, x[e][i]);
    // the reference point of a column follows its maximum only when that has grown by more than 8 (a factor 256 in
    // the weights): the rescale of the accumulators becomes rare
    if (__builtin_amdgcn_ballot_w64(top > m_run + 8.f) != 0) {
      const float t = max_over_row_groups(top);
      const float m_new = t > m_run + 8.f ? t : m_run;
      const float alpha = m_new == m_run ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      corr *= alpha;
      float a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __shfl(alpha, 4 * g + i);
#pragma unroll
      for (int d = 0; d < kDB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[d][i] *= a[i];
    }
    const float m_ref = m_run == -INFINITY ? 0.f : m_run;  // (nothing but masked rows so far)
    // heads and tails of p * s as A operands of P.V: word w's register r holds rows r and r + 4 of its eight
    u32x4 ph[2], pt[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) ph[w] = pt[w] = (u32x4){0, 0, 0, 0};
    float ps_sum = 0.f;
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned sz = *reinterpret_cast<const unsigned *>(st + side_bytes + sz_lane + (16 * J * e + 4 * i) * pitch);
        const float s = __builtin_bit_cast(float, sz << 16), z = __builtin_bit_cast(float, sz & 0xffff0000u);
        const float pr = __builtin_amdgcn_exp2f(x[e][i] - m_ref);
        l_run += pr;
        corr = __builtin_fmaf(pr, z, corr);
        const float ps = pr * s;
        const unsigned hi = vtkv::f32_to_bf16_bits_rne(ps);
        const float hf = __builtin_bit_cast(float, hi << 16);
        const unsigned lo = vtkv::f32_to_bf16_bits_rne(ps - hf);
        ps_sum += hf + __builtin_bit_cast(float, lo << 16);
        if constexpr (J == 1) {
          ph[e >> 1][i] |= e & 1 ? hi << 16 : hi;
          pt[e >> 1][i] |= e & 1 ? lo << 16 : lo;
        } else if constexpr (J == 2) {
          ph[e][i] = j ? hi << 16 : hi;
          pt[e][i] = j ? lo << 16 : lo;
        } else {
          const unsigned a = j & 1 ? hi << 16 : hi, b = j & 1 ? lo << 16 : lo;
          ph[0][i] = j < 2 ? a : 0u;
          pt[0][i] = j < 2 ? b : 0u;
          ph[1][i] = j < 2 ? 0u : a;
          pt[1][i] = j < 2 ? 0u : b;
        }
      }
    corr = __builtin_fmaf(-128.f, ps_sum, corr);
#pragma unroll
    for (int d = 0; d < kDB; ++d) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                                                    (__attribute__((address_space(3))) i32x2 *)(st + v_lane + 8 * d)));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        u32x4 b;
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = ((w[k] >> (4 * r)) & 0x000f000fu) | 0x43004300u;
        acc[d] = mfma_16x16x32<false>(ph[k], b, acc[d]);
        acc[d] = mfma_16x16x32<false>(pt[k], b, acc[d]);
      }
    }
  };

  // ---- the end of a part: o and the statistics over the row groups and the parts of a column
  auto fold = [&](float &m_tot, float &l_tot, float &c_tot) {
    const float l = sum_over_row_groups(l_run), c = sum_over_row_groups(corr);
    m_tot = m_run;
    if constexpr (J >= 2) m_tot = fmaxf(m_tot, __shfl_xor(m_tot, 8));
    if constexpr (J >= 4) m_tot = fmaxf(m_tot, __shfl_xor(m_tot, 4));
    const float f = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_tot);
    l_tot = l * f;
    c_tot = c * f;
    if constexpr (J >= 2) l_tot += __shfl_xor(l_tot, 8), c_tot += __shfl_xor(c_tot, 8);
    if constexpr (J >= 4) l_tot += __shfl_xor(l_tot, 4), c_tot += __shfl_xor(c_tot, 4);
    if constexpr (J > 1) {
      float a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __shfl(f, 4 * g + i);
#pragma unroll
      for (int d = 0; d < kDB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = acc[d][i] * a[i], v0, v1;
          if constexpr (J == 4) {
            v = sum_over_row_groups(v);
          } else {
            swap_rows32(v, v0, v1);
            v = v0 + v1;
          }
          acc[d][i] = v;
        }
    }
  };
  // the head whose results a lane holds in place i, and whether this lane stores block d of it
  auto head_at = [&](int i) { return J == 4 ? i : J == 2 ? 4 * (g & 1) + i : 4 * g + i; };
  auto stores = [&](int d) { return J == 4 ? (d & 3) == g : J == 2 ? (d & 1) == (g >> 1) : true; };
  // which result a part gives: -1: the sequence's own, whole; else its place among the partial ones
  auto place_of = [&](const Cursor &c, int first_row, bool first_part) {
    return first_row == 0 && c.end == len ? -1 : 2 * (int)blockIdx.x + (first_part ? 0 : 1);
  };
  auto put = [&](const Cursor &c, int v, int hh, int d, float o, float l) {  // one value of head hh of kv head v
    const int64_t at = ((int64_t)c.b * p.num_heads + first_head_of(p, v) + hh) * D + d;
    const float r = o / l;
    if (p.out_f32) reinterpret_cast<float *>(p.out)[at] = r;
    else reinterpret_cast<uint16_t *>(p.out)[at] = f32_to_16<F16>(r);
  };
  auto finish = [&](const Cursor &c, int first_row, bool first_part, int buf) {
    const int place = place_of(c, first_row, first_part);
    float m_tot, l_tot, c_tot;
    fold(m_tot, l_tot, c_tot);
    const int hv = head >= 0 ? heads_of(p, head) : 0;
    if (p.row_tiles == 1) {
      float lh[4], ch[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lh[i] = __shfl(l_tot, head_at(i));
        ch[i] = __shfl(c_tot, head_at(i));
      }
      const int64_t base = ((int64_t)place * p.chunk_heads + hs) * p.group;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int hh = head_at(i);
        if (hh >= hv) continue;
#pragma unroll
        for (int d = 0; d < kDB; ++d) {
          if (!stores(d)) continue;
          const float o = acc[d][i] + ch[i];
          if (place < 0) put(c, head, hh, 16 * d + n, o, lh[i]);
          else p.part_o[(base + hh) * D + 16 * d + n] = o;
        }
      }
      if (place >= 0 && g == 0 && n < kHeads && n < hv) {
        p.part_ml[(base + n) * 2] = m_tot;
        p.part_ml[(base + n) * 2 + 1] = l_tot;
      }
    } else {
      // several waves hold rows of one kv head: through the stage that has just been used up
      float *so = reinterpret_cast<float *>(smem + buf * p.stage_bytes);
      float *sml = so + p.chunk_heads * p.row_tiles * kHeads * D;
      float ch[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ch[i] = __shfl(c_tot, head_at(i));
      if (has_tile) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < kDB; ++d)
            if (stores(d)) so[(wave * kHeads + head_at(i)) * D + 16 * d + n] = acc[d][i] + ch[i];
        if (g == 0 && n < kHeads) {
          sml[(wave * kHeads + n) * 2] = m_tot;
          sml[(wave * kHeads + n) * 2 + 1] = l_tot;
        }
      }
      barrier();
      for (int idx = tid; idx < p.chunk_heads * kHeads * D; idx += kThreads) {
        const int d = idx % D, hh = idx / D % kHeads, place_h = idx / (D * kHeads);
        const int v = head_of_chunk(p, c.chunk, place_h);
        if (v < 0 || hh >= heads_of(p, v)) continue;
        float m = -INFINITY, l = 0.f, o = 0.f;
        for (int r = 0; r < p.row_tiles; ++r) m = fmaxf(m, sml[((r * p.chunk_heads + place_h) * kHeads + hh) * 2]);
        for (int r = 0; r < p.row_tiles; ++r) {
          const int w = (r * p.chunk_heads + place_h) * kHeads + hh;
          const float f = sml[w * 2] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sml[w * 2] - m);
          l += sml[w * 2 + 1] * f;
          o += so[w * D + d] * f;
        }
        const int64_t base = ((int64_t)place * p.chunk_heads + place_h) * p.group + hh;
        if (place < 0) {
          put(c, v, hh, d, o, l);
        } else {
          p.part_o[base * D + d] = o;
          if (d == 0) {
            p.part_ml[base * 2] = m;
            p.part_ml[base * 2 + 1] = l;
          }
        }
      }
      barrier();
    }
  };

  // ---- the pipeline: while stage s is computed, stage s + 1 is on its way
  Cursor lc = cc;
  load_q(cc);
  begin(cc);
  issue(lc, 0);
  step(lc);
  bool more = lc.valid();
  if (more) {
    issue(lc, 1);
    step(lc);
  }
  int first_row = cc.row;
  bool first_part = true;
  for (int buf = 0;; buf ^= 1) {
    wait_loads(more ? 2 * my_loads : 0);
    barrier();
    const Cursor now = cc;
    step(cc);
    const bool part_ends = now.row + stage_rows >= now.end;
    if (part_ends && cc.valid()) load_q(cc);
    compute(now, buf);
    barrier();
    if (part_ends) {
      finish(now, first_row, first_part, buf);
      if (!cc.valid()) return;
      first_part = false;
      begin(cc);
      first_row = cc.row;
    }
    more = lc.valid();
    if (more) {
      issue(lc, buf);
      step(lc);
    }
  }
}

// Merges the partial results of a (sequence, query head); writes zeros where there are no rows.
template <int D, bool F16>
__global__ void __launch_bounds__(256) int4_merge_kernel(DecodeParams p, int grid) {
  const int v = blockIdx.y, b = blockIdx.x, C = p.chunks;
  const int hv = heads_of(p, v), h0 = first_head_of(p, v);
  const int c0 = p.cum[b], nb = p.cum[b + 1] - c0, total = p.cum[p.num_seqs] * C;
  int chunk, hs;
  if (p.kv_split == 1) {
    chunk = v / p.chunk_heads;
    hs = v % p.chunk_heads;
  } else {
    const int part = v % p.kv_split;
    chunk = v / p.kv_split * p.parts_per_real + part / p.chunk_heads;
    hs = part % p.chunk_heads;
  }
  const int active = total ? active_spans(p, total, grid) : 1;
  const int u0 = c0 * C + chunk * nb, u1 = u0 + nb;
  // span of unit u: the last i with total * i / active <= u
  auto span_of = [&](int u) {
    int i = (int)(((int64_t)u * active) / total);
    while (i + 1 < active && span_begin(total, active, i + 1) <= u) ++i;
    return i;
  };
  const int i0 = nb ? span_of(u0) : 0, i1 = nb ? span_of(u1 - 1) : 0;
  if (nb && i0 == i1) return;
  for (int idx = threadIdx.x; idx < hv * D; idx += 256) {
    const int hh = idx / D, d = idx % D;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int i = i0; nb && i <= i1; ++i) {
      const int place = 2 * i + (span_begin(total, active, i) >= u0 ? 0 : 1);
      const int64_t base = ((int64_t)place * p.chunk_heads + hs) * p.group + hh;
      const float mi = p.part_ml[base * 2], li = p.part_ml[base * 2 + 1], oi = p.part_o[base * D + d];
      const float mn = fmaxf(m, mi);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn), fi = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - mn);
      l = l * f + li * fi;
      o = o * f + oi * fi;
      m = mn;
    }
    const float r = nb ? o / l : 0.f;
    const int64_t at = ((int64_t)b * p.num_heads + h0 + hh) * D + d;
    if (p.out_f32) reinterpret_cast<float *>(p.out)[at] = r;
    else reinterpret_cast<uint16_t *>(p.out)[at] = f32_to_16<F16>(r);
  }
}

template <int D>
int launch_decode(const DecodeParams &p, int j, bool f16, int grid, size_t lds, hipStream_t st) {
  typedef void (*Kernel)(DecodeParams);
  static const Kernel kernels[2][3] = {
      {int4_decode_kernel<D, 1, false>, int4_decode_kernel<D, 2, false>, int4_decode_kernel<D, 4, false>},
      {int4_decode_kernel<D, 1, true>, int4_decode_kernel<D, 2, true>, int4_decode_kernel<D, 4, true>}};
  Kernel k = kernels[f16][j == 4 ? 2 : j == 2 ? 1 : 0];
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(waves_of(D) * 64), lds, st, p);
  const dim3 mg((unsigned)p.num_seqs, (unsigned)p.num_kv_heads);
  if (f16)
    hipLaunchKernelGGL((int4_merge_kernel<D, true>), mg, dim3(256), 0, st, p, grid);
  else
    hipLaunchKernelGGL((int4_merge_kernel<D, false>), mg, dim3(256), 0, st, p, grid);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

int round_up(int x, int m) { return (x + m - 1) / m * m; }

// The shape of a launch: kv heads and row tiles per workgroup, its LDS.
int plan(DecodeParams &p, int d, int kv_real, int j, size_t &lds) {
  const int waves = waves_of(d);
  if (p.kv_split == 1) {
    int hc = waves;
    while (kv_real % hc) hc /= 2;
    p.chunk_heads = hc;
    p.chunk_real = hc;
    p.chunks = kv_real / hc;
    p.parts_per_real = 1;
  } else {
    int hc = 1;
    while (hc < p.kv_split && hc < waves) hc *= 2;
    p.chunk_heads = hc;
    p.chunk_real = 1;
    p.parts_per_real = (p.kv_split + hc - 1) / hc;
    p.chunks = kv_real * p.parts_per_real;
  }
  if (p.chunk_real == kv_real) {  // whole rows
    p.code_units = p.row_bytes / 16;
    p.scale_units = 0;
  } else {
    const int codes = p.chunk_real * (d / 2);
    p.code_units = codes % 16 == 0 ? codes / 16 : (codes + 8 + 15) / 16;  // (a start that is 8 bytes into a piece)
    p.scale_units = std::min(4 * p.chunk_real % 16 == 0 && kv_real * (d / 2) % 16 == 0 ? p.chunk_real / 4 : (4 * p.chunk_real + 12 + 15) / 16,
                             p.row_bytes / 16);
  }
  const int pitch = (p.code_units + p.scale_units) * 16;
  const int extra = round_up((p.num_seqs + 1) * 4, 16) + std::min(p.num_seqs, kPtrTable) * 16;
  p.row_tiles = waves / p.chunk_heads;
  for (;; --p.row_tiles) {
    // (a tile's results need less than its rows where every kv head has rows of its own, more where several parts of a
    // kv head read the same ones)
    const int results = p.row_tiles > 1 ? p.row_tiles * p.chunk_heads * (16 / j) * (4 * d + 8) : 0;
    p.stage_bytes = round_up(std::max(2 * p.row_tiles * kTileRows * pitch, results), 16);
    lds = (size_t)2 * p.stage_bytes + extra;
    if (lds + 256 <= kLdsBytes && p.row_tiles * pitch / 16 <= loads_of(d) * waves) break;
    VTKV_REQUIRE(p.row_tiles > 1, "rows of %d bytes leave no room for a stage", p.row_bytes);
  }
  p.min_units = 2 + 2 * p.row_tiles;
  return VTKV_OK;
}

}  // namespace

namespace vtkv {

int64_t int4_decode_workspace_bytes(int num_seqs, int num_heads, int head_size) {
  const int64_t heads = std::min<int64_t>(128, num_heads + num_heads / 16 + 16);
  return 2ll * kDecodeSpans * heads * (head_size + 2) * 4 + ((int64_t)std::min(num_seqs, kMaxBatch) + 1) * 4 + 64;
}

int int4_decode(void *out, const void *q, const int64_t *k_ptrs, const int64_t *v_ptrs, const int64_t *slot_ids,
                const int32_t *seq_lens, int num_seqs, int num_heads, int num_kv_heads, int head_size, int64_t q_stride,
                float scale, int max_seq_len, const float *alibi_slopes, int q_dtype, int out_dtype, void *workspace,
                int64_t workspace_bytes, void *stream) {
  const int group_real = num_heads / num_kv_heads, split = vtkv_kv_split(group_real);
  DecodeParams p;
  p.k_ptrs = k_ptrs;
  p.v_ptrs = v_ptrs;
  p.alibi_slopes = alibi_slopes;
  p.q_stride = q_stride;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads * split;
  p.kv_split = split;
  p.group_real = group_real;
  p.group = (group_real + split - 1) / split;
  p.row_bytes = (int)int4_row_bytes(num_kv_heads, head_size);
  p.max_seq_len = max_seq_len;
  p.out_f32 = out_dtype == VTKV_F32;
  p.scale_log2 = scale * kLog2e;
  const int j = p.group <= 4 ? 4 : p.group <= 8 ? 2 : 1;
  for (int at = 0; at < num_seqs; at += kMaxBatch) {
    p.num_seqs = std::min(kMaxBatch, num_seqs - at);
    p.q = (const uint16_t *)q + at * q_stride;
    p.slot_ids = slot_ids + at;
    p.seq_lens = seq_lens + at;
    p.out = (char *)out + (int64_t)at * num_heads * head_size * (p.out_f32 ? 4 : 2);
    size_t lds;
    const int planned = plan(p, head_size, num_kv_heads, j, lds);
    if (planned < 0) return planned;
    const int64_t cum_bytes = ((int64_t)p.num_seqs + 1 + 15) / 16 * 64;
    const int64_t per_span = 2ll * p.chunk_heads * p.group * (head_size + 2) * 4;
    const int64_t room = workspace ? (workspace_bytes - cum_bytes) / per_span : 0;
    if (room < 1 || (uintptr_t)workspace % 16 != 0)
      return fail(VTKV_ENOMEM, "a 16-byte aligned workspace of at least %lld bytes is needed, got %lld",
                  (long long)(cum_bytes + per_span), (long long)workspace_bytes);
    const int grid = (int)std::min<int64_t>(kDecodeSpans, room);
    p.cum = (int32_t *)workspace;
    p.part_o = (float *)((char *)workspace + cum_bytes);
    p.part_ml = p.part_o + 2ll * grid * p.chunk_heads * p.group * head_size;
    const bool f16 = q_dtype == VTKV_F16;
    hipStream_t st = (hipStream_t)stream;
    int rc;
    switch (head_size) {
      case 64: rc = launch_decode<64>(p, j, f16, grid, lds, st); break;
      case 80: rc = launch_decode<80>(p, j, f16, grid, lds, st); break;
      case 96: rc = launch_decode<96>(p, j, f16, grid, lds, st); break;
      case 112: rc = launch_decode<112>(p, j, f16, grid, lds, st); break;
      case 128: rc = launch_decode<128>(p, j, f16, grid, lds, st); break;
      default: rc = launch_decode<256>(p, j, f16, grid, lds, st); break;
    }
    if (rc < 0) return rc;
  }
  return VTKV_OK;
}

}  // namespace vtkv
