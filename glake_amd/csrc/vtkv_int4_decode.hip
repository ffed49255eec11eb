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
//    two per query head (its largest value near 2^14; how exact that is: vtkv_int4_query.h).
//  * V: the codes of 16 rows come out of LDS transposed (ds_read_b64_tr_b4: lane d of a group gets column d of 16
//    rows) and are masked the same way: as bf16 numbers they are c * 2^-133 and c * 2^-129, in the denormals and the
//    binade above them, where the bits count evenly.  p s comes with a factor of 2^60 (2^56 for the rows whose codes
//    stand 2^4 higher) and is carried as a bf16 head and a bf16 tail (2^-18 relative, rounded).  What p s is below 2^-57
//    loses bits (values of 1e-18 still come out within 1e-5 of their size, values of 1e-22 within 1e-2).  Scales of 2^60
//    and more, whose p s may leave the fp32 range, make the result of their query head NaN or infinite; the second kernel
//    computes such a result again, plainly (plain_attention).
//
// How it moves data.  HBM-bound: 2 rows of 68 bytes per token and kv head (head size 128).  A workgroup takes whole
// rows (or eight kv heads of them): a stage of 64 rows (512 / kv heads when there are fewer than eight) of K and V goes
// from global memory straight into LDS (16 bytes per lane, no registers), two stages deep, so that loads are always in
// flight while the other stage is computed; a row's bytes are fetched once whatever the heads per line.  Each wave
// serves one kv head and 32 rows of the stage; sixteen waves (four per SIMD) hide each other's chains of LDS reads, MFMAs
// and exponentials.  What the waves of a kv head hold is combined through LDS when a span's part of a sequence ends.
//
// Up to eight query heads per kv head leave half of the 16-column tiles free: then a tile's columns are (part j, head)
// and the two 16-row tiles of a wave share one tile of logits (J = 2), so the softmax arithmetic is per logit that
// exists; P.V takes the same layout with zeros where a row is not the part's, and the parts are added up at the end.
//
// The batch's rows in steps of 16 are cut into as many equal spans as workgroups run, where a sequence that begins counts
// as some steps more (part_units): a new part costs as much time as three stages, and without that count the workgroup
// with the most parts ends last (17 sequences of 3 to 2501 rows, 32 kv heads of 80 in four chunks: 53 us against 32 us when
// the end of a part took 4.5 us; two stages 35 us, four 32 us).  A span that ends inside a sequence leaves a partial
// result in the workspace and a second kernel merges them.
//
// What it takes (kernel and merge): 64 sequences of 512 to 4096 rows of 8 kv heads of 128, 4 query heads each (161 MB): 44 + 6
// us; four of 32768 to 131072 rows (371 MB): 80 + 5 us; 32 kv heads of 80 as above (60 MB): 31 + 4 us; one of 777 rows: 16 + 4
// us.  A stage takes 3.0 us with all workgroups at it (6.0 TB/s), the way to the first stage's rows 8.8 us, the end of a
// part 2.5 to 4 us.
#include "vtkv_attn_common.h"
#include "vtkv_common.h"
#include "vtkv_int4.h"
#include "vtkv_int4_query.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace vtkv_attn;

constexpr int kMaxBatch = 1024;   // sequences per launch
constexpr int kPtrTable = 256;    // base addresses held in LDS, of the first so many sequences
constexpr int kTileRows = 32;     // rows of a wave's tile
constexpr int kPrivate = 512;     // LDS of a wave: the scales and zeros of its tile's K rows, then of its V rows
constexpr int kUnitRows = 16;     // rows by which spans are cut
constexpr int kLdsBytes = 160 * 1024;

constexpr int waves_of(int d) { return d > 128 ? 8 : 16; }
constexpr int loads_of(int d) { return d > 128 ? 5 : 3; }  // 16-byte loads per lane, stage and side at most
// blocks of 16 columns of 16 rows that all waves' results go through LDS at a time: half of them (all, where two parts of a
// column are added up before)
constexpr int round_of(int d) { return (d / 16 + 1) / 2; }
constexpr int results_bytes(int d) { return waves_of(d) * (round_of(d) * 1024 + 192); }

struct DecodeParams {
  const uint16_t *q;
  const int64_t *k_ptrs, *v_ptrs, *slot_ids;
  const int32_t *seq_lens;
  const float *alibi_slopes;
  void *out;
  float *part_o;    // [2 * grid][chunk heads][group][D]
  float *part_ml;   // the same without D, (maximum, sum) pairs
  int32_t *spans;   // [num_seqs, chunks] pairs: the place of its first partial result, the last span that holds rows of it
  int64_t q_stride;
  int num_seqs, num_heads, num_kv_heads, kv_split, group, group_real;  // (kv heads as the kernel sees them)
  int row_bytes, max_seq_len, out_f32;
  int chunk_heads, chunks, chunk_real, parts_per_real;  // kv heads of a workgroup; chunks per sequence; real kv heads of one
  int row_tiles;               // tiles of rows per stage
  int stage_bytes;             // LDS of a stage: K, then V (or what its waves hold, combined when a part ends)
  int code_units, scale_units; // 16-byte pieces of a row in LDS
  int min_units;               // a span's units at least
  int part_units;              // what beginning a sequence counts
  float scale_log2;
};

// The spans: the batch's units are numbered through, part_units of each sequence (per chunk) that stand for no rows and
// then its rows' units; unit u belongs to span u * active / total, each a contiguous range.
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
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
// Until at most n vector memory instructions are outstanding.  They retire in order, so the older ones are done.
__device__ __forceinline__ void wait_loads(int n) {
#define VTKV_WAIT(N)                                    \
  case N: asm volatile("s_waitcnt vmcnt(" #N ")" ::: "memory"); break;
  switch (n) {
    VTKV_WAIT(2) VTKV_WAIT(4) VTKV_WAIT(6) VTKV_WAIT(8) VTKV_WAIT(10)
    default: asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
#undef VTKV_WAIT
}
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// x again, as a value the compiler knows nothing about: what is computed from it stays where it is used instead of being
// kept in registers across the loop
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
// The kernel's arguments again, for code between the loops: read from memory where they are used instead of being held in
// scalar registers (which run out: those that do not fit are kept in vector lanes, an instruction each time) all along.
__device__ __forceinline__ const DecodeParams &reload() {
  auto p = (const __attribute__((address_space(4))) DecodeParams *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const DecodeParams *)p;
}
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  return (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x);
}

// A place in the batch's order (sequence, chunk, row), with the end of the part of it that this span holds (0: past the
// span) and the units of the span behind that part.
struct Cursor {
  int b, chunk, row, end, left;
};

template <int D, int J, bool F16>
__global__ void __launch_bounds__(waves_of(D) * 64) int4_decode_kernel(DecodeParams p) {
  constexpr int kWaves = waves_of(D), kThreads = kWaves * 64, kLoads = loads_of(D);
  constexpr int kWords = D / 8, kSteps = (kWords + 3) / 4;  // words of eight codes; MFMA steps over d
  constexpr int kDB = D / 16, kPairs = (kDB + 1) / 2;       // blocks of 16 output columns
  constexpr int kRound = round_of(D);
  constexpr int kHeads = 16 / J;  // columns of a part
  constexpr int kE = 2 / J;       // tiles of logits
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_tot[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n = lane & 15;
  const int j = n / kHeads;  // this lane's column: part j, head n % kHeads
  const int B = p.num_seqs, C = p.chunks;
  const int units_row = p.code_units + p.scale_units, pitch = units_row * 16;
  const int stage_rows = p.row_tiles * kTileRows, side_bytes = stage_rows * pitch;
  int *s_cum = reinterpret_cast<int *>(smem + 2 * p.stage_bytes + kWaves * kPrivate);
  uint64_t *s_ptr = reinterpret_cast<uint64_t *>(smem + 2 * p.stage_bytes + kWaves * kPrivate + ((B + 1) * 4 + 15) / 16 * 16);

  // ---- units before every sequence, and the base addresses of the first ones
  {
    constexpr int kPer = (kMaxBatch + kThreads - 1) / kThreads;
    int local[kPer], sum = 0;
    const bool in_table = tid < min(B, kPtrTable);
    const int64_t slot = in_table ? p.slot_ids[tid] : 0;
    const int own_len = in_table ? min(p.seq_lens[tid], p.max_seq_len) : 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int idx = tid * kPer + k;
      local[k] = sum;
      if (idx < B) {
        const int rows = min(p.seq_lens[idx], p.max_seq_len);
        if (rows > 0) sum += (rows - 1) / kUnitRows + 1 + p.part_units;
      }
    }
    if (in_table) reinterpret_cast<int *>(s_ptr + 2 * kPtrTable)[tid] = own_len;
    if (own_len > 0) {  // (the slot of a sequence without rows is not followed: a padded entry may hold anything)
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
  }
  const int total = uniform(s_cum[B]) * C;
  const int active = active_spans(p, total, gridDim.x);
  if ((int)blockIdx.x >= active || total == 0) return;
  const int u_begin = span_begin(total, active, blockIdx.x), u_end = span_begin(total, active, blockIdx.x + 1);
  if (u_begin >= u_end) return;

  auto len_of = [&](int b) {
    if (b < kPtrTable) return uniform(reinterpret_cast<const int *>(s_ptr + 2 * kPtrTable)[b]);
    const DecodeParams &p = reload();
    return uniform(min(p.seq_lens[b], p.max_seq_len));
  };
  // the part of sequence b, chunk c from unit k on, as far as `left` units go (none, if they end before its rows begin)
  const int part_units = p.part_units;
  auto enter = [&](Cursor &c, int b, int chunk, int k, int left) {
    const int nb = uniform(s_cum[b + 1]) - uniform(s_cum[b]);
    const int take = min(left, nb - k);
    c.b = b;
    c.chunk = chunk;
    c.row = max(0, k - part_units) * kUnitRows;
    c.end = min(len_of(b), max(0, k + take - part_units) * kUnitRows);
    c.left = left - take;
  };
  auto step = [&](Cursor &c) {  // one stage on; true: into another part
    c.row += stage_rows;
    if (c.row < c.end) return false;
    if (c.left == 0) {
      c.end = 0;
      return true;
    }
    int b = c.b, chunk = c.chunk + 1;
    if (chunk == C) {
      chunk = 0;
      do ++b; while (uniform(s_cum[b + 1]) == uniform(s_cum[b]));  // (ends: `left` units are still to come)
    }
    enter(c, b, chunk, 0, c.left);
    return true;
  };
  Cursor cc;
  {
    // the last sequence that begins at or before u_begin and has units
    int b = 0;
    for (int i0 = 0; i0 < B; i0 += 64) {
      const int i = i0 + lane;
      const bool before = i < B && s_cum[i] * C <= u_begin && s_cum[i + 1] > s_cum[i];
      const unsigned long long m = __builtin_amdgcn_ballot_w64(before);
      if (m) b = i0 + 63 - __builtin_clzll(m);
    }
    b = uniform(b);
    const int c0 = uniform(s_cum[b]), nb = uniform(s_cum[b + 1]) - c0;
    const int k = u_begin - c0 * C;
    enter(cc, b, k / nb, k % nb, u_end - u_begin);
    if (cc.end == 0) return;
  }

  // ---- this wave's kv head and rows of the stage
  const int hs = wave % p.chunk_heads, rt = wave / p.chunk_heads;
  const bool has_tile = rt < p.row_tiles;
  // the words of a row that a lane group multiplies: the first, how many
  auto word0_of = [](int g) { return kWords % 4 == 0 ? g * (kWords / 4) : g * (kWords / 4) + min(g, kWords % 4); };
  auto words_of = [](int g) { return kWords / 4 + (g < kWords % 4 ? 1 : 0); };
  auto load_q = [&](const Cursor &c, u32x4 (&raw)[kSteps]) {
    const DecodeParams &p = reload();
    const int lane = opaque(tid & 63), g = lane >> 4, h = lane % kHeads, word0 = word0_of(g), words = words_of(g);
    const int v = has_tile ? head_of_chunk(p, c.chunk, hs) : -1;
    const int hv = v < 0 ? 0 : heads_of(p, v), h0 = v < 0 ? 0 : first_head_of(p, v);
    const uint16_t *row = p.q + (int64_t)c.b * p.q_stride + (int64_t)(h0 + min(h, max(hv - 1, 0))) * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      raw[s] = (u32x4){0, 0, 0, 0};
      if (s < words && h < hv) raw[s] = *reinterpret_cast<const u32x4 *>(row + 8 * (word0 + s));
    }
  };

  // ---- stage loads: 16-byte piece i of a stage's side goes to LDS byte 16 i; lane l of load k of this wave takes
  // piece (wave + waves * k) * 64 + l
  const int pieces = stage_rows * units_row, num_loads = (pieces + 63) / 64;
  const int my_loads = wave < num_loads ? (num_loads - wave + kWaves - 1) / kWaves : 0;
  // its row of the stage (10 bits) and where its piece begins in a row of the cursor's chunk (22: a row is below 4 MiB)
  unsigned ld_at[kLoads];
  uint64_t k_from, v_from;  // the cursor's first row
  auto aim = [&](const Cursor &c) {  // at the cursor's part
    const DecodeParams &p = reload();
    const int real0 = real0_of(p, c.chunk);
    const int code0 = p.scale_units ? real0 * (D / 2) / 16 * 16 : 0;
    const int all_codes = p.num_kv_heads / p.kv_split * (D / 2);
    const int scale0 = min((all_codes + 4 * real0) / 16 * 16, p.row_bytes - 16 * p.scale_units) - 16 * p.code_units;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = (wave + kWaves * k) * 64 + opaque(lane);
      const int row = i / units_row, col = i - row * units_row;
      ld_at[k] = (unsigned)row << 22 | (unsigned)(col * 16 + (col < p.code_units ? code0 : scale0));
    }
    uint64_t kb, vb;
    if (c.b < kPtrTable) {
      kb = s_ptr[2 * c.b];
      vb = s_ptr[2 * c.b + 1];
    } else {
      const int64_t slot = p.slot_ids[c.b];
      kb = (uint64_t)p.k_ptrs[slot];
      vb = (uint64_t)p.v_ptrs[slot];
    }
    k_from = uniform64(kb) + (uint64_t)c.row * p.row_bytes;
    v_from = uniform64(vb) + (uint64_t)c.row * p.row_bytes;
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr)smem + wave * 1024;
  const uint32_t stage_step = (uint32_t)stage_rows * p.row_bytes;
  auto issue = [&](const Cursor &c, int buf) {
    const int last = min(stage_rows, c.end - c.row) - 1;  // rows past the part's end: its last row again, never used
    const uint32_t dst = lds0 + buf * p.stage_bytes;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      if (wave + kWaves * k >= num_loads) break;
      const uint32_t off = __umul24(min((int)(ld_at[k] >> 22), last), p.row_bytes) + (ld_at[k] & 0x3fffffu);
      if ((wave + kWaves * k) * 64 + lane < pieces) {
        load_to_lds(k_from, off, dst + k * kWaves * 1024);
        load_to_lds(v_from, off, dst + k * kWaves * 1024 + side_bytes);
      }
    }
    k_from += stage_step;
    v_from += stage_step;
  };

  u32x4 qop[kSteps];
  float q_back, q_sum, slope;  // logit = (s * 2^24 scale) * (acc * q_back) + z * q_sum [+ slope * distance]
  float own_mul;               // what this lane multiplies its row's scale with: 2^24 scale (K), the power of two of P.V (V)
  int k_lane, v_lane, v_last, sz_lane, head = -1, len = 0;
  f32x4 acc[kDB];
  // a column's reference point, and how far a logit may be above it before it follows the maximum (-inf: no logit yet);
  // the sums of p and of p z
  float m_ref, lazy, l_run, z_run;
  auto begin = [&](const Cursor &c, const u32x4 (&raw)[kSteps]) {
    const DecodeParams &p = reload();
    const int lane = opaque(tid & 63), g = lane >> 4, n = lane & 15, h = n % kHeads, word0 = word0_of(g);
    head = has_tile ? head_of_chunk(p, c.chunk, hs) : -1;
    len = len_of(c.b);
    LargestQuery<F16> largest;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) largest.take(raw[s]);
    const QueryScale q_scale = query_scale(largest.value());
    q_back = q_scale.down;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      qop[s] = query_operand<F16>(raw[s], q_scale.up);
      __builtin_amdgcn_sched_barrier(0);
    }
    q_sum = query_sum(qop) * q_scale.down * p.scale_log2;
    __builtin_amdgcn_sched_barrier(0);  // (what follows must not take registers from what precedes)
    slope = 0.f;
    if (p.alibi_slopes && head >= 0 && h < heads_of(p, head)) slope = p.alibi_slopes[first_head_of(p, head) + h] * kLog2e;
    const int real0 = real0_of(p, c.chunk), real = head >= 0 ? real_kv_head(p, head) : real0;
    const int code_at = real * (D / 2) - (p.scale_units ? real0 * (D / 2) / 16 * 16 : 0);
    const int all_codes = p.num_kv_heads / p.kv_split * (D / 2);
    const int scale_at = p.scale_units ? p.code_units * 16 + all_codes + 4 * real -
                                             min((all_codes + 4 * real0) / 16 * 16, p.row_bytes - 16 * p.scale_units)
                                       : all_codes + 4 * real;
    // tile t's row of lane m as A operand: 16 t + 4 (m & 3) + m / 4; then a lane group's logits are rows = g mod 4: the 8
    // rows whose codes its lanes bring together for P.V, lanes 0..7 of the group from one block of 16 columns, lanes
    // 8..15 from the next (the odd last block: from the same)
    const int rt = has_tile ? wave / p.chunk_heads : 0;  // (a wave without a tile reads the first one and leaves it)
    k_lane = (rt * kTileRows + 4 * (n & 3) + (n >> 2)) * pitch + code_at + 4 * word0;
    v_lane = side_bytes + (rt * kTileRows + 4 * (n & 7) + g) * pitch + code_at + 8 * (n >> 3);
    v_last = v_lane - 8 * (n >> 3);
    sz_lane = (lane >> 5) * side_bytes + (rt * kTileRows + 4 * (lane & 7) + (lane >> 3 & 3)) * pitch + scale_at;
#pragma unroll
    for (int d = 0; d < kDB; ++d) acc[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // (this lane's row of the tile is 4 (lane & 7) + ..: its register of the P.V operands is odd where lane is)
    own_mul = lane < 32 ? 0x1p24f * p.scale_log2 : lane & 1 ? 0x1p56f : 0x1p60f;
    m_ref = 0.f;
    lazy = -INFINITY;
    l_run = z_run = 0.f;
  };
  // what a column's value is multiplied with, for the four columns whose results this lane holds
  auto rescale = [&](float f) {
    const int g = opaque(lane) >> 4;
    float a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __shfl(f, 4 * g + i);
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[d][i] *= a[i];
  };
  // v_perm selectors: the lower, the upper half of a register into the part's half, zero into the other (12: a zero byte)
  const unsigned half_sel[2] = {j == 0 ? 0x0c0c0100u : 0x01000c0cu, j == 0 ? 0x0c0c0302u : 0x03020c0cu};

  // A tile as its wave takes it out of LDS: K codes as MFMA operands need them, V codes transposed, one (scale, zero) pair
  // per lane.  It fits registers, so the stage's LDS is free for new loads as soon as every wave has read, not when it
  // has computed.
  struct Tile {
    unsigned kw[2][kSteps], pair;
    u32x2 vw[kPairs];
  };
  auto take = [&](int buf, Tile &tile) {
    auto &kw = tile.kw;
    const char *st = smem + buf * p.stage_bytes;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char *at = st + k_lane + 16 * t * pitch;
      if constexpr (D == 128 || D == 256) {
#pragma unroll
        for (int s = 0; s < kSteps; s += 4) {
          const u32x4 v = *reinterpret_cast<const u32x4 *>(at + 4 * s);
#pragma unroll
          for (int i = 0; i < 4; ++i) kw[t][s + i] = v[i];
        }
      } else if constexpr (D == 64) {
        const u32x2 v = *reinterpret_cast<const u32x2 *>(at);
        kw[t][0] = v[0];
        kw[t][1] = v[1];
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) kw[t][s] = *reinterpret_cast<const unsigned *>(at + 4 * s);
      }
    }
    tile.pair = *reinterpret_cast<const unsigned *>(st + sz_lane);
#pragma unroll
    for (int dp = 0; dp < kPairs; ++dp) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      tile.vw[dp] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2 *)(
                                             st + (kDB % 2 == 1 && 2 * dp + 1 == kDB ? v_last : v_lane) + 16 * dp)));
    }
  };
  auto compute = [&](const Cursor &c, const Tile &tile) {
    const int rows = min(kTileRows, c.end - c.row - rt * kTileRows);
    if (head < 0 || rows <= 0) return;
    f32x4 sa[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) sa[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const unsigned w = tile.kw[t][s], y = w >> 8;
        const u32x4 a = {w & 0x000f000fu, w & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
        sa[t] = mfma_16x16x32<true>(a, qop[s], sa[t]);
      }
    // The scales and zeros change lanes through the wave's own LDS (whose operations keep their order): row 16 t + 4 i + g
    // is held by lane 8 g + 4 t + i (K), 32 lanes on (V); each lane prepares its row's for all columns.
    const int at_lane = opaque(lane);
    char *own = smem + 2 * p.stage_bytes + wave * kPrivate;
    {
      float *at = reinterpret_cast<float *>(own + 8 * (at_lane & 32) + 4 * (at_lane & 31));
      at[0] = __builtin_bit_cast(float, tile.pair << 16) * own_mul;
      at[32] = __builtin_bit_cast(float, tile.pair & 0xffff0000u);
    }
    own += 32 * (at_lane >> 4) + (J == 2 ? 16 * (at_lane >> 3 & 1) : 0);
    f32x4 k_s[kE], k_z[kE], v_s[kE], v_z[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      k_s[e] = *reinterpret_cast<const f32x4 *>(own + 16 * e);
      k_z[e] = *reinterpret_cast<const f32x4 *>(own + 128 + 16 * e);
    }
    auto values = [&]() {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        v_s[e] = *reinterpret_cast<const f32x4 *>(own + 256 + 16 * e);
        v_z[e] = *reinterpret_cast<const f32x4 *>(own + 384 + 16 * e);
      }
    };
    if constexpr (J == 2) values();
    __builtin_amdgcn_sched_barrier(0);
    // x[e][i]: how far the lane's logit of row 16 (J e + j) + 4 i + g is above the reference point
    float x[kE][4], a[kE][4], top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[e][i] = (J == 2 ? (j == 0 ? sa[0][i] : sa[1][i]) : sa[e][i]) * q_back;
    {
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[e][i] = __builtin_fmaf(k_s[e][i], a[e][i], __builtin_fmaf(k_z[e][i], q_sum, -m_ref));
      if (p.alibi_slopes) {
        const float ahead = (float)(c.row + rt * kTileRows + 16 * (J == 2 ? at_lane >> 3 & 1 : 0) + (at_lane >> 4) - len + 1);
#pragma unroll
        for (int e = 0; e < kE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[e][i] = __builtin_fmaf(slope, ahead + (float)(16 * J * e + 4 * i), x[e][i]);
      }
      if (rows < kTileRows) {
        const int row = 16 * (J == 2 ? at_lane >> 3 & 1 : 0) + (at_lane >> 4);
#pragma unroll
        for (int e = 0; e < kE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * J * e + 4 * i + row >= rows) x[e][i] = -INFINITY;
      }
      top = -INFINITY;
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[e][i]);
    }
    // The reference point of a column follows its maximum only when that has grown by more than 8 (a factor 256 in
    // the weights): the rescale of the accumulators becomes rare.  (The logits follow by the same number, so that the
    // largest is 0 exactly however large it was.)
    if (__builtin_amdgcn_ballot_w64(top > lazy) != 0) {
      const float t = max_over_row_groups(top);
      const bool moves = t > lazy;  // (its first logit, where lazy is -inf)
      const float alpha = moves ? (lazy == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-t)) : 1.f;
      if (moves) {
        m_ref += t;
        lazy = 8.f;
      }
      l_run *= alpha;
      z_run *= alpha;
      rescale(alpha);
      const float up = moves ? t : 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e][i] -= up;
    }
    if constexpr (J == 1) {  // (twice the logits: registers are short until they are done)
      __builtin_amdgcn_sched_barrier(0);
      values();
    }
    // heads and tails of p * s as A operands of P.V: register r holds rows r and r + 4 of the group's eight (J = 2: the
    // lane's half of it, the other zero).  Both are rounded to nearest: a head cut off instead leaves a tail of one sign, whose
    // own cut then adds up over the rows (1.5e-4 of the results' root mean square at 4096 rows, against the codes' part being
    // nearly cancelled by the zeros').
    u32x4 ph, pt;
    float ps[kE][4];
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float pr = __builtin_amdgcn_exp2f(x[e][i]);
        l_run += pr;
        z_run = __builtin_fmaf(pr, v_z[e][i], z_run);
        ps[e][i] = pr * v_s[e][i];
      }
    // what the two 16-bit values of a register leave of the numbers they stand for
    auto left = [](float a, float b, unsigned h) {
      return pack_bf16x2(a - __builtin_bit_cast(float, h << 16), b - __builtin_bit_cast(float, h & 0xffff0000u));
    };
    if constexpr (J == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ph[i] = pack_bf16x2(ps[0][i], ps[1][i]);
        pt[i] = left(ps[0][i], ps[1][i], ph[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const unsigned h = pack_bf16x2(ps[0][i], ps[0][i + 1]), t = left(ps[0][i], ps[0][i + 1], h);
        ph[i] = __builtin_amdgcn_perm(0u, h, half_sel[0]);
        ph[i + 1] = __builtin_amdgcn_perm(0u, h, half_sel[1]);
        pt[i] = __builtin_amdgcn_perm(0u, t, half_sel[0]);
        pt[i + 1] = __builtin_amdgcn_perm(0u, t, half_sel[1]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < kDB; ++d) {
      const unsigned w = tile.vw[d / 2][d & 1], y = w >> 8;
      const u32x4 b = {w & 0x000f000fu, w & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
      acc[d] = mfma_16x16x32<false>(ph, b, acc[d]);
      acc[d] = mfma_16x16x32<false>(pt, b, acc[d]);
    }
  };

  // ---- the end of a part: the waves of a kv head (row tiles, and the parts of a column) first agree on the maximum, bring
  // their sums to it and add up the parts in registers, then the tiles through the stage that has been used up: each of
  // the head's waves adds up some blocks of columns and stores them: the result, or this span's share of one
  auto finish = [&](const Cursor &c, int first_row, bool first_part, int buf) {
    const DecodeParams &p = reload();
    const int tid = opaque(threadIdx.x), lane = tid & 63, g = lane >> 4, n = lane & 15;
    constexpr int kVals = J == 2 ? 2 : 4, kPer = kRound * J;  // rows of a block per lane; blocks of columns of a round
    l_run = sum_over_row_groups(l_run);
    z_run = sum_over_row_groups(z_run);
    float *so = reinterpret_cast<float *>(smem + buf * p.stage_bytes), *sml = so + kWaves * kRound * 256;
    if (g == 0) {
      sml[(wave * 16 + n) * 3] = lazy == -INFINITY ? -INFINITY : m_ref;
      sml[(wave * 16 + n) * 3 + 1] = l_run;
      sml[(wave * 16 + n) * 3 + 2] = z_run;
    }
    const bool whole = first_row == 0 && c.end == len;
    const int place = 2 * (int)blockIdx.x + (first_part ? 0 : 1);
    if (tid == 0) {
      int32_t *span = p.spans + 2 * ((int64_t)c.b * C + c.chunk);
      if (first_row == 0) span[0] = place;
      if (c.end == len) span[1] = blockIdx.x;
    }
    barrier();
    // the tiles of the kv head are waves hs, hs + chunk_heads, ...; this lane: query head n % kHeads
    const int tiles = p.row_tiles, tile_step = p.chunk_heads;
    float m = -INFINITY, l = 0.f, cr = 0.f;
    const float *ml0 = sml + (hs * 16 + n % kHeads) * 3;
#pragma unroll 1
    for (int t = 0; t < tiles; ++t)
#pragma unroll
      for (int q = 0; q < J; ++q) m = fmaxf(m, ml0[(t * tile_step * 16 + q * kHeads) * 3]);
#pragma unroll 1
    for (int t = 0; t < tiles; ++t)
#pragma unroll
      for (int q = 0; q < J; ++q) {
        const float *ml = ml0 + (t * tile_step * 16 + q * kHeads) * 3;
        const float f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m);
        l = __builtin_fmaf(ml[1], f, l);
        cr = __builtin_fmaf(ml[2], f, cr);
      }
    rescale(lazy == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - m) * 0x1p73f);  // (133 - 60 binades)
    const int hv = head < 0 ? 0 : heads_of(p, head);
    const int64_t part = ((int64_t)place * p.chunk_heads + hs) * p.group;
    if (!whole && rt == 0 && lane < hv)  // (hv <= kHeads)
      *reinterpret_cast<u32x2 *>(p.part_ml + (part + lane) * 2) = (u32x2){__builtin_bit_cast(unsigned, m), __builtin_bit_cast(unsigned, l)};
    // the rows (query heads) that this lane holds of a block, and what they take
    auto row_of = [&](int k) { return J == 2 ? 4 * (g & 1) + 2 * k + (lane >> 5) : 4 * g + k; };
    const float factor = whole ? 1.f / l : 1.f;
    float add[kVals], mul[kVals];
#pragma unroll
    for (int k = 0; k < kVals; ++k) {
      add[k] = __shfl(cr, row_of(k));
      mul[k] = __shfl(factor, row_of(k));
    }
    typedef float Vals __attribute__((ext_vector_type(kVals)));
#pragma unroll
    for (int d0 = 0; d0 < kDB; d0 += kPer) {
      if (d0 > 0) barrier();
#pragma unroll
      for (int d = d0; d < kDB && d < d0 + kPer; ++d) {
        Vals x;
        if constexpr (J == 2) {
          // rows r and r + 8, which are 32 lanes apart, added up: the lower lanes get those of acc[..][2 k], the upper those of
          // acc[..][2 k + 1]
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float lower = acc[d][2 * k], upper = acc[d][2 * k + 1];
            const auto y = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, lower),
                                                            __builtin_bit_cast(unsigned, upper), false, false);
            const unsigned y0 = y[0], y1 = y[1];
            x[k] = __builtin_bit_cast(float, y0) + __builtin_bit_cast(float, y1);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = acc[d][k];
        }
        *reinterpret_cast<Vals *>(so + ((wave * kPer + d - d0) * 64 + lane) * kVals) = x;
      }
      barrier();
      if (head >= 0) {
#pragma unroll 1
        for (int d = d0 + rt; d < min(kDB, d0 + kPer); d += tiles) {
          const float *from = so + ((hs * kPer + d - d0) * 64 + lane) * kVals;
          Vals o = *reinterpret_cast<const Vals *>(from);
#pragma unroll 1
          for (int t = 1; t < tiles; ++t) o += *reinterpret_cast<const Vals *>(from + t * tile_step * kPer * 64 * kVals);
#pragma unroll
          for (int k = 0; k < kVals; ++k) {
            const int row = row_of(k);
            if (row >= hv) continue;
            const float x = (o[k] + add[k]) * mul[k];
            const int64_t at = ((int64_t)c.b * p.num_heads + first_head_of(p, head) + row) * D + 16 * d + n;
            if (!whole) p.part_o[(part + row) * D + 16 * d + n] = x;
            else if (p.out_f32) reinterpret_cast<float *>(p.out)[at] = x;
            else reinterpret_cast<uint16_t *>(p.out)[at] = f32_to_16<F16>(x);
          }
        }
      }
    }
    barrier();
  };

  // ---- the pipeline: while a stage is computed, the next one is on its way
  Cursor lc = cc, now = cc;
  int ahead = 0, first_row = cc.row;  // stages asked for and not yet computed
  bool fresh = true, first_part = true, any = false, aimed = false;
  auto ask = [&](int next, int most) {  // for stages from the one that is computed next on
    for (; ahead < most && lc.end > 0; ++ahead) {
      if (!aimed) aim(lc);
      issue(lc, next ^ ahead);
      aimed = !step(lc);
    }
  };
  for (int buf = 0;; buf ^= 1) {
    if (fresh && any) {
      finish(now, first_row, first_part, buf ^ 1);
      if (cc.end == 0) return;
      first_part = false;
      first_row = cc.row;
    }
    // a part's first stage is asked for before its q, its second after: the wait for q is a wait for all that was asked
    // for before
#pragma unroll 1
    for (int most = fresh ? 1 : 2;; ++most) {
      ask(buf, most);
      if (most == 2) break;
      u32x4 raw[kSteps];
      load_q(cc, raw);
      begin(cc, raw);
    }
    wait_loads(ahead == 2 ? 2 * my_loads : 0);
    barrier();
    now = cc;
    fresh = step(cc);
    Tile tile;
    take(buf, tile);
    barrier();
    --ahead;
    // (the last stage of a part is left to its results)
    if (!fresh) ask(buf ^ 1, 2);
    compute(now, tile);
    any = true;
  }
}

// Attention of one query head over the values themselves, in fp32 on the vector unit by a workgroup of 256 threads: for
// results that the kernel above could not hold (and for those that are not finite whichever way they are computed).  A thread
// takes whole rows for their logits, then, 256 rows at a time, a dim for the sum of the values, whose weights are normalised
// first: it stays as small as the values are.  Where a logit or a V row is not a number the result is none either, and known
// after the logits.  (One sequence of 131072 rows, 32 query heads over 8 kv heads of
// 128: 12 ms, 1.3 ms where it ends after the logits; ordinary values take 0.1 ms.)
template <int D, bool F16>
__device__ void plain_attention(const DecodeParams &p, int b, int head, int len) {
  __shared__ float s_q[D], s_p[256], s_top[256];
  const int tid = threadIdx.x, real = head / p.group_real, kv_real = p.num_kv_heads / p.kv_split;
  const int64_t slot = p.slot_ids[b];
  const char *const k_rows = (const char *)(uintptr_t)p.k_ptrs[slot], *const v_rows = (const char *)(uintptr_t)p.v_ptrs[slot];
  const int codes_at = real * (D / 2), pair_at = kv_real * (D / 2) + 4 * real;
  const float slope = p.alibi_slopes ? p.alibi_slopes[head] * kLog2e : 0.f;
  if (tid < D) s_q[tid] = unpack_16<F16>(p.q[(int64_t)b * p.q_stride + (int64_t)head * D + tid], 0) * p.scale_log2;
  __syncthreads();
  auto logit = [&](int r) {
    const char *row = k_rows + (int64_t)r * p.row_bytes;
    const unsigned *codes = reinterpret_cast<const unsigned *>(row + codes_at);
    const unsigned pair = *reinterpret_cast<const unsigned *>(row + pair_at);
    const float s = __builtin_bit_cast(float, pair << 16), z = __builtin_bit_cast(float, pair & 0xffff0000u);
    float x = 0.f;
#pragma unroll 4
    for (int w = 0; w < D / 8; ++w)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x = __builtin_fmaf(s_q[8 * w + i], __builtin_fmaf((float)(codes[w] >> (4 * i) & 15u), s, z), x);
    return __builtin_fmaf(slope, (float)(r - len + 1), x);
  };
  // ---- maximum and sum
  float m = -INFINITY, l = 0.f;
  bool none = false;
#pragma unroll 1
  for (int r = tid; r < len; r += 256) {
    const unsigned pair = *reinterpret_cast<const unsigned *>(v_rows + (int64_t)r * p.row_bytes + pair_at);
    const float x = logit(r), top = fmaxf(m, x);
    none |= (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u || x != x || x == INFINITY;
    l = l * (m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top)) + (x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - top));
    m = top;
  }
  none = __syncthreads_or(none);
  s_top[tid] = m;
  __syncthreads();
  float all = -INFINITY;
  for (int i = 0; i < 256; ++i) all = fmaxf(all, s_top[i]);
  s_p[tid] = m == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - all);
  __syncthreads();
  float sum = 0.f;
  for (int i = 0; i < 256; ++i) sum += s_p[i];
  const float inv = 1.f / sum;
  // ---- the values
  float o = none ? __builtin_nanf("") : 0.f;
#pragma unroll 1
  for (int r0 = 0; r0 < len && !none; r0 += 256) {
    __syncthreads();
    if (r0 + tid < len) s_p[tid] = __builtin_amdgcn_exp2f(logit(r0 + tid) - all) * inv;
    __syncthreads();
    if (tid < D) {
      const char *row = v_rows + (int64_t)r0 * p.row_bytes;
#pragma unroll 8
      for (int i = 0; i < min(256, len - r0); ++i, row += p.row_bytes) {
        const unsigned pair = *reinterpret_cast<const unsigned *>(row + pair_at), code = (unsigned char)row[codes_at + tid / 2] >> (4 * (tid & 1)) & 15u;
        o = __builtin_fmaf(s_p[i], __builtin_fmaf((float)code, __builtin_bit_cast(float, pair << 16), __builtin_bit_cast(float, pair & 0xffff0000u)), o);
      }
    }
  }
  if (tid < D) {
    const int64_t at = ((int64_t)b * p.num_heads + head) * D + tid;
    if (p.out_f32) reinterpret_cast<float *>(p.out)[at] = o;
    else reinterpret_cast<uint16_t *>(p.out)[at] = f32_to_16<F16>(o);
  }
}

// Merges the partial results of a (sequence, query head); writes zeros where there are no rows.  The partial results are
// dealt to groups of D / 4 lanes with four values each.  A result that is not finite is computed again.
template <int D, bool F16>
__global__ void __launch_bounds__(256) int4_merge_kernel(DecodeParams p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes, kUnroll = 4;
  __shared__ float s_o[kGroups][D], s_m[kGroups], s_l[kGroups];
  const int b = blockIdx.x, head = blockIdx.y;
  const int real = head / p.group_real, in_real = head % p.group_real;
  int hh = in_real, hs = real % p.chunk_heads, chunk = real / p.chunk_heads;
  if (p.kv_split > 1) {
    const int part = in_real / p.group;
    hh = in_real % p.group;
    hs = part % p.chunk_heads;
    chunk = real * p.parts_per_real + part / p.chunk_heads;
  }
  const int len = min(p.seq_lens[b], p.max_seq_len);
  const int32_t *span = p.spans + 2 * ((int64_t)b * p.chunks + chunk);
  const int first = len > 0 ? span[0] : 0, i0 = first / 2, i1 = len > 0 ? span[1] : -1;
  if (i0 == i1) {  // one span held all rows and has written the result
    bool lost = false;
    if (threadIdx.x < D) {
      const int64_t at = ((int64_t)b * p.num_heads + head) * D + threadIdx.x;
      if (p.out_f32) lost = (reinterpret_cast<const unsigned *>(p.out)[at] & 0x7f800000u) == 0x7f800000u;
      else lost = (~reinterpret_cast<const uint16_t *>(p.out)[at] & (F16 ? 0x7c00u : 0x7f80u)) == 0;
    }
    if (__syncthreads_or(lost)) plain_attention<D, F16>(p, b, head, len);
    return;
  }
  const int grp = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int i = i0 + grp; grp < kGroups && i <= i1; i += kGroups * kUnroll) {
    float mi[kUnroll], li[kUnroll];
    f32x4 oi[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int at = min(i + k * kGroups, i1);
      const int place = at == i0 ? first : 2 * at;
      const int64_t base = ((int64_t)place * p.chunk_heads + hs) * p.group + hh;
      mi[k] = i + k * kGroups <= i1 ? p.part_ml[base * 2] : -INFINITY;
      li[k] = p.part_ml[base * 2 + 1];
      oi[k] = *reinterpret_cast<const f32x4 *>(p.part_o + base * D + d);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) mn = fmaxf(mn, mi[k]);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    l *= f;
    o *= f;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const float fi = mi[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi[k] - mn);
      l += li[k] * fi;
      o += oi[k] * fi;
    }
    m = mn;
  }
  if (grp < kGroups) {
    *reinterpret_cast<f32x4 *>(&s_o[grp][d]) = o;
    if (d == 0) {
      s_m[grp] = m;
      s_l[grp] = l;
    }
  }
  __syncthreads();
  bool lost = false;
  if (threadIdx.x < D) {
    float mm = -INFINITY, ll = 0.f, oo = 0.f;
    for (int k = 0; k < kGroups; ++k) mm = fmaxf(mm, s_m[k]);
    for (int k = 0; k < kGroups; ++k) {
      const float f = s_m[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[k] - mm);
      ll += s_l[k] * f;
      oo += s_o[k][threadIdx.x] * f;
    }
    const float r = len > 0 ? oo / ll : 0.f;
    const int64_t at = ((int64_t)b * p.num_heads + head) * D + threadIdx.x;
    if (p.out_f32) reinterpret_cast<float *>(p.out)[at] = r;
    else reinterpret_cast<uint16_t *>(p.out)[at] = f32_to_16<F16>(r);
    lost = (__builtin_bit_cast(unsigned, r) & 0x7f800000u) == 0x7f800000u;
  }
  if (__syncthreads_or(lost)) plain_attention<D, F16>(p, b, head, len);
}

template <int D>
int launch_decode(const DecodeParams &p, int j, bool f16, int grid, size_t lds, hipStream_t st) {
  typedef void (*Kernel)(DecodeParams);
  static const Kernel kernels[2][2] = {{int4_decode_kernel<D, 1, false>, int4_decode_kernel<D, 2, false>},
                                       {int4_decode_kernel<D, 1, true>, int4_decode_kernel<D, 2, true>}};
  hipLaunchKernelGGL(kernels[f16][j == 2], dim3((unsigned)grid), dim3(waves_of(D) * 64), lds, st, p);
  const dim3 mg((unsigned)p.num_seqs, (unsigned)p.num_heads);
  if (f16)
    hipLaunchKernelGGL((int4_merge_kernel<D, true>), mg, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((int4_merge_kernel<D, false>), mg, dim3(256), 0, st, p);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

int round_up(int x, int m) { return (x + m - 1) / m * m; }

// The shape of a launch: kv heads and row tiles per workgroup, its LDS.
int plan(DecodeParams &p, int d, int kv_real, size_t &lds) {
  const int waves = waves_of(d), most = waves / 2;  // (at least two row tiles: 64 rows of a stage)
  if (p.kv_split == 1) {
    int hc = most;
    while (kv_real % hc) hc /= 2;
    p.chunk_heads = hc;
    p.chunk_real = hc;
    p.chunks = kv_real / hc;
    p.parts_per_real = 1;
  } else {
    int hc = 1;
    while (hc < p.kv_split && hc < most) hc *= 2;
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
  const int extra = waves * kPrivate + round_up((p.num_seqs + 1) * 4, 16) + kPtrTable * 20;
  p.row_tiles = waves / p.chunk_heads;
  for (;; --p.row_tiles) {
    // (the results of a round need less than the rows where every kv head has rows of its own, more where several parts
    // of a kv head read the same ones)
    p.stage_bytes = round_up(std::max(2 * p.row_tiles * kTileRows * pitch, results_bytes(d)), 16);
    lds = (size_t)2 * p.stage_bytes + extra;
    if (lds + 256 <= kLdsBytes && (p.row_tiles * kTileRows * pitch / 16 + 63) / 64 <= loads_of(d) * waves) break;
    VTKV_REQUIRE(p.row_tiles > 1, "rows of %d bytes leave no room for a stage", p.row_bytes);
  }
  p.min_units = std::max(4, p.row_tiles);
  p.part_units = 3 * p.row_tiles * kTileRows / kUnitRows;
  return VTKV_OK;
}

}  // namespace

namespace vtkv {

int64_t int4_decode_workspace_bytes(int num_seqs, int num_heads, int head_size) {
  const int64_t heads = std::min<int64_t>(128, num_heads + num_heads / 16 + 16);
  return 2ll * kDecodeSpans * heads * (head_size + 2) * 4 + (int64_t)std::min(num_seqs, kMaxBatch) * num_heads * 8 + 64;
}

int int4_decode(void *out, const void *q, const int64_t *k_ptrs, const int64_t *v_ptrs, const int64_t *slot_ids,
                const int32_t *seq_lens, int num_seqs, int num_heads, int num_kv_heads, int head_size, int64_t q_stride,
                float scale, int max_seq_len, const float *alibi_slopes, int q_dtype, int out_dtype, void *workspace,
                int64_t workspace_bytes, void *stream) {
  VTKV_REQUIRE(out && q && k_ptrs && v_ptrs && slot_ids && seq_lens, "null argument");
  VTKV_REQUIRE(num_seqs >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
               "num_heads %d must be a positive multiple of num_kv_heads %d", num_heads, num_kv_heads);
  VTKV_REQUIRE(int4_head_size(head_size), "head_size %d is not supported (64, 80, 96, 112, 128, 256)", head_size);
  VTKV_REQUIRE(q_dtype == VTKV_BF16 || q_dtype == VTKV_F16, "a 4-bit cache serves bfloat16 and float16 queries");
  VTKV_REQUIRE(out_dtype == q_dtype || out_dtype == VTKV_F32, "out_dtype must be q_dtype or F32");
  VTKV_REQUIRE(q_stride >= (int64_t)num_heads * head_size && q_stride % 8 == 0 && (uintptr_t)q % 16 == 0 &&
                   (uintptr_t)out % 16 == 0,
               "q and out must be 16-byte aligned, q rows at least num_heads*head_size apart");
  VTKV_REQUIRE(max_seq_len > 0, "max_seq_len must be > 0");
  VTKV_REQUIRE(num_heads <= 65535, "too many query heads");
  VTKV_REQUIRE(int4_row_bytes(num_kv_heads, head_size) < (4 << 20), "rows of 4 MiB and more are not supported");
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
  const int j = p.group <= 8 ? 2 : 1;
  for (int at = 0; at < num_seqs; at += p.num_seqs) {
    p.num_seqs = std::min(kMaxBatch, num_seqs - at);
    p.q = (const uint16_t *)q + at * q_stride;
    p.slot_ids = slot_ids + at;
    p.seq_lens = seq_lens + at;
    p.out = (char *)out + (int64_t)at * num_heads * head_size * (p.out_f32 ? 4 : 2);
    size_t lds;
    const int planned = plan(p, head_size, num_kv_heads, lds);
    if (planned < 0) return planned;
    // (a launch numbers its units with 32 bits)
    const int64_t most = 0x7fffffff / ((((int64_t)max_seq_len - 1) / kUnitRows + 1 + p.part_units) * p.chunks);
    VTKV_REQUIRE(most > 0, "max_seq_len %d is too large for %d kv heads", max_seq_len, num_kv_heads);
    p.num_seqs = (int)std::min<int64_t>(p.num_seqs, most);
    const int64_t table = ((int64_t)p.num_seqs * p.chunks * 8 + 63) / 64 * 64;
    const int64_t per_span = 2ll * p.chunk_heads * p.group * (head_size + 2) * 4;
    const int64_t room = workspace ? (workspace_bytes - table) / per_span : 0;
    if (room < 1 || (uintptr_t)workspace % 16 != 0)
      return fail(VTKV_ENOMEM, "a 16-byte aligned workspace of at least %lld bytes is needed, got %lld",
                  (long long)(table + per_span), (long long)workspace_bytes);
    const int grid = (int)std::min<int64_t>(kDecodeSpans, room);
    p.spans = (int32_t *)workspace;
    p.part_o = (float *)((char *)workspace + table);
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
