// A cache of a bounded number of rows: how much attention each cached row has drawn, and the eviction of the rows
// that drew least.
//
//  * weights[slot, kv head, row] += sum over the kv head's query heads of softmax_row(scale q . k [+ alibi]): K is read
//    once.  The first kernel writes the logits (fp32, 4 bytes per query head and row against 256 bytes of K per kv head at
//    head size 128) and every 64 rows' maximum and sum, the second turns them into weights.  Bound by the K rows.
//  * evict: per (sequence, kv head) the last `recent` rows stay, and of the rows before them the `keep - recent` with
//    the largest weight (of equal ones those that come first).  The survivors that lie behind place keep - recent move
//    into the places of the evicted rows before it, in order, and the recent rows move behind them: no more rows move
//    than have to, and the recent rows, which the next steps append to, stay in the order of their tokens.
#include "vtkv_attn_common.h"
#include "vtkv_common.h"
#include "vtkv_int4.h"
#include "vtkv_int4_query.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace vtkv_attn;

constexpr int kTileRows = 64;  // rows of a wave of the logit kernel, whose maximum and sum are kept
constexpr int kSumThreads = 512;
constexpr int kSumRows = 4 * kSumThreads;  // rows of a workgroup of the second kernel
constexpr int64_t kMostScratch = 256ll << 20;  // a larger batch runs as consecutive parts through the same scratch

struct WeightParams {
  float *weights;
  int64_t slot_stride, head_stride, num_slots;
  const uint16_t *q;
  const int64_t *k_ptrs, *slot_ids;
  const int32_t *seq_lens;
  const float *alibi_slopes;
  float *logits;  // [num_seqs, num_heads, pitch], log2 units
  float *stats;   // [num_seqs, num_heads, pitch / 64, 2]: maximum, sum of 2^(logit - maximum)
  int64_t q_stride;
  int num_heads, num_kv_heads, kv_split, group, group_real;  // (kv heads as the kernel sees them: see first_head_of)
  int row_bytes, max_seq_len, pitch;
  int heads_wg;   // waves of a workgroup that take neighbouring kv heads of the same rows
  float scale_log2;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(1))) u32x4 *gvec4;
typedef const __attribute__((address_space(1))) unsigned *gvec1;

// 16 bytes per lane from base + off to lds + 16 * lane (M0 holds lds).  Nothing the compiler counts: the caller waits.
__device__ __forceinline__ void load_to_lds(uint64_t base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "memory");
}

// A maximum as one instruction (fmaxf() first quiets operands that the compiler cannot prove canonical).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The value of the lane eight places on in its sixteen.
__device__ __forceinline__ float other_part(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
}

// KV: 0: 16-bit rows of the model's type, 1: e4m3fn codes, 2: 4-bit rows.  A wave takes up to kTiles tiles of 64 rows
// of one kv head one after the other; while a tile is multiplied, the next one is on its way.  The workgroup's waves take
// kv heads next to each other of the same rows, since a head's part of a row is short (64 sequences of 512 to 4096 rows,
// 32 query heads over 8 kv heads of 128 bf16 elements: 68 us that way, K at 4.5 TB/s; four waves along the rows of one head: 82 us).
//  * 16-bit and fp8 rows go into the wave's own LDS as whole head rows (a load instruction covers whole cache lines; lane m
//    of an MFMA operand holds one row, so loads into registers would take 64 bytes of sixteen rows each: 88 us against 82),
//    from there into registers, which frees the LDS for the next tile.  Rows of a power of two of 16-byte pieces have their
//    pieces exchanged by row so that operand reads meet all banks.  Two tiles per wave: 68 us, one 78, four 74, eight 71.
//  * 4-bit codes go straight into operand registers and are multiplied as fp16 denormals, q carrying the rest, and a row's
//    scale and zero applied to its logits (as in vtkv_int4_decode.hip).  27 us for 24
//    sequences of 1024 to 8192 rows and 64 query heads over 8 kv heads, one tile per wave or two.
constexpr int kTiles = 2;

// J = 2: up to eight query heads per kv head: a lane's column is (part j, head), and of two 16-row tiles it keeps the logits
// of the j-th, so that what follows the products is done once per logit (J = 1 for the 24 sequences above: 29 us instead of 27).
template <int D, int KV, bool F16, int J>
__global__ void __launch_bounds__(KV == 2 ? 512 : 256) attention_logits_kernel(WeightParams p) {
  constexpr bool I4 = KV == 2, FP8 = KV == 1;
  constexpr int kWords = D / 8;                                                // 4-bit rows: words of eight codes
  constexpr int kHeadBytes = I4 ? D / 2 : FP8 ? D : 2 * D;
  constexpr int kRowPieces = kHeadBytes / 16;                                  // (not 4-bit) 16-byte pieces of a head's row
  constexpr bool kSwizzle = !I4 && (kRowPieces & (kRowPieces - 1)) == 0;
  constexpr int kPieces = I4 ? 1 : (kRowPieces + 3) / 4;                       // of them that a lane multiplies
  constexpr int kSteps = FP8 ? 2 * kPieces : (kWords + 3) / 4;                 // MFMA steps over d
  __shared__ __attribute__((aligned(16))) char s_rows[I4 ? 1 : 4][I4 ? 16 : kTileRows * kHeadBytes];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), waves = blockDim.x >> 6;
  constexpr int kHeads = 16 / J, kE = 4 / J;
  const int g = lane >> 4, n = lane & 15, j = n / kHeads, h = n % kHeads;
  const int b = blockIdx.z, groups = (p.num_kv_heads + p.heads_wg - 1) / p.heads_wg;
  const int v = blockIdx.x % groups * p.heads_wg + wave % p.heads_wg;
  const int first = (blockIdx.x / groups * (waves / p.heads_wg) + wave / p.heads_wg) * kTiles * kTileRows;
  const int len = uniform(min(p.seq_lens[b], p.max_seq_len));
  const int64_t slot = p.slot_ids[b];
  if (first >= len || v >= p.num_kv_heads || slot < 0 || slot >= p.num_slots) return;
  const int h0 = first_head_of(p, v), hv = heads_of(p, v), real = real_kv_head(p, v), kv_real = p.num_kv_heads / p.kv_split;
  const char *k_base = (const char *)(uintptr_t)p.k_ptrs[slot];
  const int last = min(len, first + kTiles * kTileRows);  // rows of this wave: [first, last)
  // 4-bit: the words that this lane's group multiplies
  const int word0 = kWords % 4 == 0 ? g * (kWords / 4) : g * (kWords / 4) + min(g, kWords % 4);
  const int words = kWords / 4 + (g < kWords % 4 ? 1 : 0);

  // ---- a tile on its way: into LDS, or (4-bit) into registers
  struct Codes {
    unsigned w[4][I4 ? kSteps : 1], pair;
  };
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)s_rows[I4 ? 0 : wave];
  auto ask = [&](int row0, Codes &next) {
    const int rows = min(kTileRows, last - row0);  // (rows past the end: the last one again, masked below)
    const char *k_rows = k_base + (int64_t)row0 * p.row_bytes;
    if constexpr (I4) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const char *from = k_rows + (uint32_t)min(16 * t + n, rows - 1) * (uint32_t)p.row_bytes + (uint32_t)real * kHeadBytes + 4 * word0;
        if constexpr (kSteps % 4 == 0 && kWords % 4 == 0) {
#pragma unroll
          for (int s = 0; s < kSteps; s += 4) {
            const u32x4 w = *(gvec4)(from + 4 * s);
#pragma unroll
            for (int i = 0; i < 4; ++i) next.w[t][s + i] = w[i];
          }
        } else {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) next.w[t][s] = s < words ? *(gvec1)(from + 4 * s) : 0u;
        }
      }
      next.pair = *(gvec1)(k_rows + (uint32_t)min(lane, rows - 1) * (uint32_t)p.row_bytes + (uint32_t)kv_real * kHeadBytes + 4 * real);
    } else {
      const uint64_t at = (uint64_t)(uintptr_t)k_rows + (uint64_t)real * kHeadBytes;
      const uint64_t base = (uint64_t)(uint32_t)uniform((int)(at >> 32)) << 32 | (uint32_t)uniform((int)at);
#pragma unroll
      for (int i = 0; i < kRowPieces; ++i) {
        const int u = 64 * i + lane, row = u / kRowPieces, slot16 = u % kRowPieces;
        const int piece = kSwizzle ? slot16 ^ (row & (kRowPieces - 1)) : slot16;
        load_to_lds(base, (uint32_t)min(row, rows - 1) * (uint32_t)p.row_bytes + piece * 16, lds + i * 1024);
      }
    }
  };
  Codes next;
  ask(first, next);

  // ---- the queries, as operands in the order of the codes
  u32x4 qop[kSteps];
  float q_back = p.scale_log2, q_sum = 0.f;
  {
    const uint16_t *q_row = p.q + (int64_t)b * p.q_stride + (int64_t)(h0 + min(h, hv - 1)) * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int at = I4 ? 8 * (word0 + s) : FP8 ? 16 * (4 * (s / 2) + g) + 8 * (s & 1) : 8 * (4 * s + g);
      const bool live = h < hv && (I4 ? s < words : at < D);
      qop[s] = (u32x4){0, 0, 0, 0};
      if (live) qop[s] = *reinterpret_cast<const u32x4 *>(q_row + at);
    }
  }
  if constexpr (I4) {
    LargestQuery<F16> largest;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) largest.take(qop[s]);
    const QueryScale q_scale = query_scale(largest.value());
    q_back = p.scale_log2 * 0x1p24f * q_scale.down;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qop[s] = query_operand<F16>(qop[s], q_scale.up);
    q_sum = query_sum(qop) * q_scale.down * p.scale_log2;
  }
  const float slope = p.alibi_slopes && h < hv ? p.alibi_slopes[h0 + h] * kLog2e : 0.f;
  const int row_at = 16 * (J == 2 ? j : 0) + 4 * g;  // this lane's rows of a tile: 16 J e + row_at + i

#pragma unroll 1
  for (int row0 = first; row0 < last; row0 += kTileRows) {
    const int rows = min(kTileRows, last - row0);
    const bool more = row0 + kTileRows < last;
    u32x4 kr[4][kPieces];
    Codes now = next;
    if constexpr (!I4) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
          const int piece = kRowPieces % 4 == 0 ? 4 * s + g : min(4 * s + g, kRowPieces - 1);  // (past the head: q is zero)
          const int at = kSwizzle ? piece ^ ((16 * t + n) & (kRowPieces - 1)) : piece;
          kr[t][s] = *reinterpret_cast<const u32x4 *>(s_rows[wave] + (16 * t + n) * kHeadBytes + at * 16);
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (more) ask(row0 + kTileRows, next);
    // ---- logits
    f32x4 x[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      f32x4 a[J];
#pragma unroll
      for (int q = 0; q < J; ++q) {
        const int t = J * e + q;
        a[q] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          if constexpr (I4) {
            const unsigned w = now.w[t][s], y = w >> 8;
            a[q] = mfma_16x16x32<true>((u32x4){w & 0x000f000fu, w & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u}, qop[s], a[q]);
          } else if constexpr (FP8) {
            a[q] = mfma_16x16x32<F16>(fp8x8_widen<F16>(kr[t][s / 2][2 * (s & 1)], kr[t][s / 2][2 * (s & 1) + 1]), qop[s], a[q]);
          } else {
            a[q] = mfma_16x16x32<F16>(kr[t][s], qop[s], a[q]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float dot = J == 2 ? (j == 0 ? a[0][i] : a[J - 1][i]) : a[0][i];
        if constexpr (I4) {
          const unsigned sz = (unsigned)__shfl((int)now.pair, 16 * J * e + row_at + i);
          x[e][i] = __builtin_fmaf(__builtin_bit_cast(float, sz << 16) * dot, q_back, __builtin_bit_cast(float, sz & 0xffff0000u) * q_sum);
        } else {
          x[e][i] = dot * q_back;
        }
      }
    }
    if (p.alibi_slopes) {
      const float ahead = (float)(row0 + row_at - len + 1);
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e][i] = __builtin_fmaf(slope, ahead + (float)(16 * J * e + i), x[e][i]);
    }
    if (rows < kTileRows) {
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * J * e + row_at + i >= rows) x[e][i] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kE; ++e) top = max3(max3(top, x[e][0], x[e][1]), x[e][2], x[e][3]);
    top = max_over_row_groups(top);
    if constexpr (J == 2) top = max3(top, other_part(top), top);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(x[e][i] - ref);
    sum = sum_over_row_groups(sum);
    if constexpr (J == 2) sum += other_part(sum);
    if (h < hv) {
      const int64_t head = (int64_t)b * p.num_heads + h0 + h;
      float *to = p.logits + head * p.pitch + row0 + row_at;
#pragma unroll
      for (int e = 0; e < kE; ++e) *reinterpret_cast<f32x4 *>(to + 16 * J * e) = x[e];
      if (g == 0 && j == 0) *reinterpret_cast<u32x2 *>(p.stats + (head * (p.pitch / kTileRows) + row0 / kTileRows) * 2) =
          (u32x2){__builtin_bit_cast(unsigned, top), __builtin_bit_cast(unsigned, sum)};
    }
  }
}

// weights += sum over the heads of 2^(logit - maximum) / sum, kSumRows rows of one kv head per workgroup, four in a row per
// thread: its waves reduce the heads' statistics, a head each, while the first heads' logits are on their way; then every
// thread adds up its rows over the heads.
constexpr int kSumHeads = 64;  // heads at a time
constexpr int kSumAhead = 4;   // heads whose logits are asked for ahead

__global__ void __launch_bounds__(kSumThreads) add_weights_kernel(WeightParams p) {
  __shared__ float s_max[kSumHeads], s_inv[kSumHeads];
  const int b = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int len = min(p.seq_lens[b], p.max_seq_len), row = blockIdx.x * kSumRows + 4 * tid;
  const int64_t slot = p.slot_ids[b];
  if ((int)blockIdx.x * kSumRows >= len || slot < 0 || slot >= p.num_slots) return;
  const int tiles = (len + kTileRows - 1) / kTileRows, G = p.group_real;
  const int64_t head0 = (int64_t)b * p.num_heads + (int64_t)kvh * G;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < G; g0 += kSumHeads) {
    const int heads = min(kSumHeads, G - g0);
    const float *logits = p.logits + (head0 + g0) * p.pitch + row;  // (the pitch is a multiple of 64, so rows < pitch are there)
    f32x4 x[kSumAhead];
#pragma unroll
    for (int a = 0; a < kSumAhead; ++a)
      if (row < len) x[a] = *reinterpret_cast<const f32x4 *>(logits + (int64_t)min(a, heads - 1) * p.pitch);
    if (g0 > 0) __syncthreads();
    for (int h = wave; h < heads; h += kSumThreads / 64) {
      const f32x2 *stats = reinterpret_cast<const f32x2 *>(p.stats) + (head0 + g0 + h) * (p.pitch / kTileRows);
      float m = -INFINITY, l = 0.f;
      for (int t = lane; t < tiles; t += 64) {
        const f32x2 tile = stats[t];
        const float mn = fmaxf(m, tile[0]), ref = mn == -INFINITY ? 0.f : mn;
        l = l * __builtin_amdgcn_exp2f(m - ref) + tile[1] * __builtin_amdgcn_exp2f(tile[0] - ref);
        m = mn;
      }
      float mw = m;
#pragma unroll
      for (int d = 32; d; d >>= 1) mw = fmaxf(mw, __shfl_xor(mw, d));
      if (mw == -INFINITY) mw = 0.f;
      l *= __builtin_amdgcn_exp2f(m - mw);
#pragma unroll
      for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
      if (lane == 0) {
        s_max[h] = mw;
        s_inv[h] = 1.f / l;
      }
    }
    __syncthreads();
    if (row < len)
      for (int h0 = 0; h0 < heads; h0 += kSumAhead) {
#pragma unroll
        for (int a = 0; a < kSumAhead; ++a) {
          if (h0 + a >= heads) break;
          const float m = s_max[h0 + a], inv = s_inv[h0 + a];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(x[a][i] - m), inv, acc[i]);
          if (h0 + kSumAhead + a < heads) x[a] = *reinterpret_cast<const f32x4 *>(logits + (int64_t)(h0 + kSumAhead + a) * p.pitch);
        }
      }
  }
  float *w = p.weights + slot * p.slot_stride + kvh * p.head_stride + row;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (row + i < len) w[i] += acc[i];
}

template <int D, int J>
void launch_logits(const WeightParams &p, int kv, bool f16, dim3 grid, int threads, hipStream_t st) {
  typedef void (*Kernel)(WeightParams);
  static const Kernel kernels[3][2] = {{attention_logits_kernel<D, 0, false, J>, attention_logits_kernel<D, 0, true, J>},
                                       {attention_logits_kernel<D, 1, false, J>, attention_logits_kernel<D, 1, true, J>},
                                       {attention_logits_kernel<D, 2, false, J>, attention_logits_kernel<D, 2, true, J>}};
  hipLaunchKernelGGL(kernels[kv][f16], grid, dim3((unsigned)threads), 0, st, p);
}
template <int D>
void launch_logits(const WeightParams &p, int kv, bool f16, dim3 grid, int threads, hipStream_t st) {
  if (p.group <= 8)
    launch_logits<D, 2>(p, kv, f16, grid, threads, st);
  else
    launch_logits<D, 1>(p, kv, f16, grid, threads, st);
}

// No two (slot, kv head) of the weights share one of their `rows` first elements (an expanded tensor's would: workgroups
// would add to them, or move them, at the same time).
bool weights_apart(int64_t slot_stride, int64_t head_stride, int64_t num_slots, int num_kv_heads, int rows) {
  typedef __int128 wide;
  if (num_kv_heads > 1 && head_stride < rows) return false;
  if (num_slots > 1 && slot_stride < rows) return false;
  return num_kv_heads == 1 || num_slots == 1 || slot_stride >= (wide)(num_kv_heads - 1) * head_stride + rows ||
         head_stride >= (wide)(num_slots - 1) * slot_stride + rows;
}

int64_t weight_pitch(int max_seq_len) { return ((int64_t)max_seq_len + kTileRows - 1) / kTileRows * kTileRows; }
int64_t weight_bytes_per_seq(int num_heads, int max_seq_len) {
  const int64_t pitch = weight_pitch(max_seq_len);
  return num_heads * (pitch + pitch / kTileRows * 2) * (int64_t)sizeof(float);
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
  bool held;       // an old row's key fits into LDS
  int num_kv_heads, row_bytes;
  int head_bytes, tail_off;  // bytes of one head in a row; 4-bit rows: where the (scale, zero) pairs start, else -1
};

// Larger weight <-> larger key; +0 and -0 are the same weight, every NaN is the largest.
__device__ __forceinline__ unsigned weight_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);
  if (w != w) return ~0u;
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

// One workgroup per (sequence, kv head).  The key of the last row that stays is found a byte at a time from the top, with a
// histogram of 256 bins, until all that share the bytes found stay; then the lists of places to fill and of rows that fill
// them, in order; then the moves, kFlight pieces of a thread asked for while as many before them are put down.  Up to
// kHeldKeys old rows have their keys, and later the lists, in LDS; more are read again each time, their lists in the
// workspace.  The first recent rows are asked for before the search starts.
//   Bound by the bytes moved, each read and written once, and by the search before them (15 to 19 us when nothing moves).
// 64 sequences of 8 kv heads of 128 bf16 elements that give up one row of 2049 and move 256 recent ones (139 MB read and
// written): 38 us, 3.7 TB/s; 32 sequences of 3001 to 4096 rows cut to 2048, 512 of them recent: 84 us.  Four
// pieces instead of two leave one workgroup per compute unit instead of two: 47 us and 85 us; without the second set of
// pieces in flight 39 us and 109 us; keys and lists in memory instead of LDS: 39 us and 88 us.
constexpr int kHeldKeys = 16384;
constexpr int kFlight = 2;

template <int UNIT>
__global__ void __launch_bounds__(kEvictThreads, 8) evict_kernel(EvictParams p) {
  typedef typename Unit<UNIT>::T vec;
  extern __shared__ unsigned s_key[];  // held: [old] keys, then the lists [pairs] of places and of movers
  __shared__ unsigned s_hist[2][256];
  __shared__ unsigned s_pick[3];
  __shared__ int s_wave[kEvictWaves][3];
  const int kvh = blockIdx.x % p.num_kv_heads, seq = blockIdx.x / p.num_kv_heads;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int n = min(p.seq_lens[seq], p.max_seq_len);
  const int64_t slot = p.slot_ids[seq];
  const bool skipped = slot < 0 || slot >= p.num_slots;  // (its rows stay where they are, and so does its length)
  if (kvh == 0 && tid == 0 && p.new_seq_lens != p.seq_lens) p.new_seq_lens[seq] = skipped ? p.seq_lens[seq] : max(0, min(n, p.keep));
  if (n <= p.keep || skipped) return;
  const int heavy = p.keep - p.recent, old = n - p.recent;  // old > heavy >= 0
  float *w = p.weights + slot * p.slot_stride + kvh * p.head_stride;
  const bool held = p.held;
  int32_t *holes = p.pairs + (int64_t)blockIdx.x * 2 * p.pair_cap, *movers = holes + p.pair_cap;  // (not held)

  // ---- rows move in pieces of UNIT bytes: thread -> (row of a step, side, piece)
  const int units = p.head_bytes / UNIT, per_row = 2 * units;  // (2: K and V)
  const int rows_step = kEvictThreads / per_row, step = kFlight * rows_step;
  const int sub = tid / per_row, u = tid % per_row, side = u >= units;
  const bool mine = sub < rows_step;
  char *const k_rows = reinterpret_cast<char *>(p.k_ptrs[slot]), *const v_rows = reinterpret_cast<char *>(p.v_ptrs[slot]);
  char *const pieces = (side ? v_rows : k_rows) + (int64_t)kvh * p.head_bytes + (u - side * units) * UNIT;
  struct Flight {
    vec v[kFlight];
  };
  // the recent rows from r0 on (past the end: the last one again, not put down)
  auto ask_recent = [&](Flight &f, int r0) {
#pragma unroll
    for (int i = 0; i < kFlight; ++i)
      f.v[i] = *reinterpret_cast<const vec *>(pieces + (int64_t)min(old + r0 + i * rows_step + sub, n - 1) * p.row_bytes);
  };
  auto put_recent = [&](const Flight &f, int r0) {
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int r = r0 + i * rows_step + sub;
      if (mine && r < p.recent) *reinterpret_cast<vec *>(pieces + (int64_t)(heavy + r) * p.row_bytes) = f.v[i];
    }
  };
  Flight ra, rb;
  ask_recent(ra, 0);
  ask_recent(rb, step);

  // ---- the key of the last row that stays: `rest` of the keys that share `prefix` in the bits of `mask` stay
  unsigned prefix = 0, mask = 0, rest = (unsigned)heavy, equals = 0;
  if (tid < 512) s_hist[tid >> 8][tid & 255] = 0;
  __syncthreads();
  if (heavy > 0)
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      unsigned *hist = s_hist[shift >> 3 & 1];
      for (int i0 = 0; i0 < old; i0 += kEvictThreads) {
        const int i = i0 + tid;
        unsigned k = 0;
        if (i < old) {
          k = shift == 24 || !held ? weight_key(w[i]) : s_key[i];
          if (held && shift == 24) s_key[i] = k;
        }
        // (neighbouring weights often share a byte: lanes that do so with the first one add up before they count)
        const bool in = i < old && (k & mask) == prefix;
        const unsigned digit = k >> shift & 255u;
        const unsigned long long all = __ballot(in);
        if (all) {
          const unsigned first = (unsigned)__builtin_amdgcn_readlane((int)digit, __builtin_ctzll(all));
          const unsigned long long same = __ballot(in && digit == first);
          if (in && digit != first) atomicAdd(&hist[digit], 1u);
          if (lane == __builtin_ctzll(all)) atomicAdd(&hist[first], (unsigned)__popcll(same));
        }
      }
      __syncthreads();
      if (wave == 0) {
        // lane l: bins 4 l .. 4 l + 3; how many keys lie above them
        unsigned c[4], own = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) own += c[q] = hist[4 * lane + q];
        unsigned from = own;  // sum over lanes >= this one
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const unsigned t = (unsigned)__shfl_down((int)from, d);
          if (lane + d < 64) from += t;
        }
        unsigned above = from - own;
#pragma unroll
        for (int q = 3; q >= 0; --q) {
          if (above < rest && rest <= above + c[q]) {
            s_pick[0] = (unsigned)(4 * lane + q);
            s_pick[1] = rest - above;
            s_pick[2] = c[q];
          }
          above += c[q];
        }
      } else if (wave == 1) {
#pragma unroll
        for (int q = 0; q < 4; ++q) s_hist[(shift >> 3 & 1) ^ 1][4 * lane + q] = 0;
      }
      __syncthreads();
      prefix |= s_pick[0] << shift;
      mask |= 255u << shift;
      rest = s_pick[1];
      equals = s_pick[2];
      if (rest == equals) break;  // all that share the prefix stay, whatever their other bits are
    }

  // ---- places and movers in order: each wave walks over its share of the old rows
  const int share = ((old + kEvictWaves - 1) / kEvictWaves + 63) / 64 * 64;
  const int begin = min(old, wave * share), end = min(old, begin + share);
  const unsigned long long below = (1ull << lane) - 1;
  int before_eq = 0, before_hole = 0, before_mover = 0, pairs = 0;
  unsigned bits = 0;  // held: bit c: this lane's row of chunk c of the wave's share stays
#pragma unroll 1
  // 0: equals per wave (where not all of them stay); 1: places and movers per wave; 2: the lists
  for (int pass = rest == equals ? 1 : 0; pass < 3; ++pass) {
    int eq = before_eq, hole = before_hole, mover = before_mover;
    for (int i0 = begin, c = 0; i0 < end; i0 += 64, ++c) {
      const int i = i0 + lane;
      bool stays;
      if (pass == 2 && held) {
        stays = bits >> c & 1u;
      } else {
        const unsigned k = i < end && heavy > 0 ? (held ? s_key[i] : weight_key(w[i])) & mask : 0u;
        const bool is_eq = i < end && heavy > 0 && k == prefix;
        const unsigned long long eqs = __ballot(is_eq);
        stays = i < end && heavy > 0 && (k > prefix || (is_eq && eq + __popcll(eqs & below) < (int)rest));
        eq += __popcll(eqs);
        if (pass == 1 && held) bits |= (unsigned)stays << c;
      }
      if (pass == 0) continue;
      const bool is_hole = i < end && !stays && i < heavy, is_mover = stays && i >= heavy;
      const unsigned long long hs = __ballot(is_hole), ms = __ballot(is_mover);
      if (pass == 2) {
        const int h = hole + __popcll(hs & below), m = mover + __popcll(ms & below);
        if (is_hole) held ? s_key[h] = (unsigned)i : (unsigned)(holes[h] = i);
        if (is_mover) held ? s_key[pairs + m] = (unsigned)i : (unsigned)(movers[m] = i);
      }
      hole += __popcll(hs);
      mover += __popcll(ms);
    }
    if (pass == 2) break;
    __syncthreads();
    if (lane == 0) {
      s_wave[wave][0] = eq;
      s_wave[wave][1] = hole;
      s_wave[wave][2] = mover;
    }
    __syncthreads();
    for (int v = 0; v < kEvictWaves; ++v) {
      if (pass == 0) {
        if (v < wave) before_eq += s_wave[v][0];
      } else {
        if (v < wave) before_hole += s_wave[v][1];
        if (v < wave) before_mover += s_wave[v][2];
        pairs += s_wave[v][2];  // (as many movers as places)
      }
    }
  }
  __syncthreads();

  // ---- the survivors into their places (no row is both read and written here); weights and, of 4-bit rows, the pairs of
  // scale and zero by themselves
  auto place = [&](int j) { return held ? (int)s_key[j] : holes[j]; };
  auto mover = [&](int j) { return held ? (int)s_key[pairs + j] : movers[j]; };
  auto pairs_of = [&](int j) { return reinterpret_cast<unsigned *>((j & 1 ? v_rows : k_rows) + p.tail_off + 4 * kvh); };
  auto at_row = [&](unsigned *base, int row) { return reinterpret_cast<unsigned *>((char *)base + (int64_t)row * p.row_bytes); };
  if (pairs > 0) {
    auto ask = [&](Flight &f, int j0) {
#pragma unroll
      for (int i = 0; i < kFlight; ++i)
        f.v[i] = *reinterpret_cast<const vec *>(pieces + (int64_t)mover(min(j0 + i * rows_step + sub, pairs - 1)) * p.row_bytes);
    };
    auto put = [&](const Flight &f, int j0) {
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const int j = j0 + i * rows_step + sub;
        if (mine && j < pairs) *reinterpret_cast<vec *>(pieces + (int64_t)place(j) * p.row_bytes) = f.v[i];
      }
    };
    Flight a, b;
    ask(a, 0);
    for (int j = tid; j < pairs; j += kEvictThreads) w[place(j)] = w[mover(j)];
    if (p.tail_off >= 0)
      for (int j = tid; j < 2 * pairs; j += kEvictThreads) *at_row(pairs_of(j), place(j >> 1)) = *at_row(pairs_of(j), mover(j >> 1));
    for (int j0 = 0; j0 < pairs; j0 += 2 * step) {
      ask(b, j0 + step);
      put(a, j0);
      ask(a, j0 + 2 * step);
      put(b, j0 + step);
    }
  }
  __syncthreads();

  // ---- the recent rows behind them, lowest first: a row moves down, so what is overwritten has been read before
  auto arrived = [&](const Flight &f) {
#pragma unroll
    for (int i = 0; i < kFlight; ++i) asm volatile("" ::"v"(f.v[i]));
    __syncthreads();
  };
  for (int r0 = 0; r0 < p.recent; r0 += 2 * step) {
    arrived(ra);
    put_recent(ra, r0);
    ask_recent(ra, r0 + 2 * step);
    arrived(rb);
    put_recent(rb, r0 + step);
    ask_recent(rb, r0 + 3 * step);
  }
  for (int r0 = 0; r0 < p.recent; r0 += kEvictThreads) {
    const int r = r0 + tid;
    const float x = r < p.recent ? w[old + r] : 0.f;
    __syncthreads();
    if (r < p.recent) w[heavy + r] = x;
  }
  if (p.tail_off >= 0)
    for (int r0 = 0; r0 < 2 * p.recent; r0 += kEvictThreads) {
      const int r = r0 + tid;
      unsigned x = 0;
      if (r < 2 * p.recent) x = *at_row(pairs_of(r), old + (r >> 1));
      __syncthreads();
      if (r < 2 * p.recent) *at_row(pairs_of(r), heavy + (r >> 1)) = x;
    }
  __syncthreads();
  for (int i = p.keep + tid; i < n; i += kEvictThreads) w[i] = 0.f;
}

// The new lengths where they replace the old ones (which every workgroup of the kernel above reads).
__global__ void __launch_bounds__(256) cut_lengths_kernel(int32_t *lens, const int64_t *slot_ids, int64_t num_slots, int num_seqs, int keep) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < num_seqs && slot_ids[i] >= 0 && slot_ids[i] < num_slots) lens[i] = max(0, min(lens[i], keep));
}

}  // namespace

extern "C" {

int64_t vtkv_accumulate_attention_weights_workspace_bytes(int num_seqs, int num_heads, int max_seq_len) {
  if (num_seqs <= 0 || num_heads <= 0 || max_seq_len <= 0) return 0;
  const int64_t per_seq = weight_bytes_per_seq(num_heads, max_seq_len);
  return std::min<int64_t>(num_seqs, std::max<int64_t>(1, kMostScratch / per_seq)) * per_seq;
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
  VTKV_REQUIRE(weights_apart(slot_stride, head_stride, num_slots, num_kv_heads, max_seq_len),
               "weights of different slots and kv heads overlap");
  VTKV_REQUIRE(max_seq_len <= 1 << 30, "max_seq_len %d is too large", max_seq_len);  // (rows are numbered with 32 bits)
  VTKV_REQUIRE(num_heads <= 65535, "too many query heads");
  VTKV_REQUIRE(vtkv_kv_row_bytes(num_kv_heads, head_size, kv_dtype) < (4 << 20), "rows of 4 MiB and more are not supported");
  if (num_seqs == 0) return VTKV_OK;
  const int64_t per_seq = weight_bytes_per_seq(num_heads, max_seq_len);
  const int64_t fit = workspace ? workspace_bytes / per_seq : 0;
  if (fit < 1 || (uintptr_t)workspace % 16 != 0)
    return vtkv::fail(VTKV_ENOMEM, "a 16-byte aligned workspace of at least %lld bytes is needed, got %lld", (long long)per_seq,
                      (long long)workspace_bytes);
  const int group_real = num_heads / num_kv_heads, split = vtkv_kv_split(group_real);
  WeightParams p;
  p.weights = weights;
  p.slot_stride = slot_stride;
  p.head_stride = head_stride;
  p.num_slots = num_slots;
  p.k_ptrs = k_ptrs;
  p.alibi_slopes = alibi_slopes;
  p.q_stride = q_stride;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads * split;
  p.kv_split = split;
  p.group = (group_real + split - 1) / split;
  p.group_real = group_real;
  p.row_bytes = (int)vtkv_kv_row_bytes(num_kv_heads, head_size, kv_dtype);
  p.max_seq_len = max_seq_len;
  p.pitch = (int)weight_pitch(max_seq_len);
  p.scale_log2 = scale * kLog2e * (kv_dtype == VTKV_FP8_E4M3 ? k_scale : 1.f);
  const int kv = kv_dtype == VTKV_INT4 ? 2 : kv_dtype == VTKV_FP8_E4M3 ? 1 : 0;
  const bool f16 = q_dtype == VTKV_F16;
  const int waves = kv == 2 ? 8 : 4;
  p.heads_wg = 1;
  while (p.heads_wg < waves && p.heads_wg < p.num_kv_heads) p.heads_wg *= 2;
  const int rows_wg = waves / p.heads_wg * kTileRows * kTiles;
  const int64_t gx = (p.num_kv_heads + p.heads_wg - 1) / p.heads_wg * (((int64_t)max_seq_len + rows_wg - 1) / rows_wg);
  VTKV_REQUIRE(gx * waves * 64 < (1ll << 31), "max_seq_len %d is too large", max_seq_len);
  const unsigned sx = (unsigned)(((int64_t)max_seq_len + kSumRows - 1) / kSumRows);
  hipStream_t st = (hipStream_t)stream;
  const int step = (int)std::min<int64_t>(fit, 65535);
  for (int at = 0; at < num_seqs; at += step) {
    const int n = std::min(step, num_seqs - at);
    p.q = (const uint16_t *)q + (int64_t)at * q_stride;
    p.slot_ids = slot_ids + at;
    p.seq_lens = seq_lens + at;
    p.logits = (float *)workspace;
    p.stats = p.logits + (int64_t)n * num_heads * p.pitch;
    const dim3 grid((unsigned)gx, 1, (unsigned)n);
    switch (head_size) {
      case 64: launch_logits<64>(p, kv, f16, grid, waves * 64, st); break;
      case 80: launch_logits<80>(p, kv, f16, grid, waves * 64, st); break;
      case 96: launch_logits<96>(p, kv, f16, grid, waves * 64, st); break;
      case 112: launch_logits<112>(p, kv, f16, grid, waves * 64, st); break;
      case 128: launch_logits<128>(p, kv, f16, grid, waves * 64, st); break;
      default: launch_logits<256>(p, kv, f16, grid, waves * 64, st); break;
    }
    hipLaunchKernelGGL(add_weights_kernel, dim3(sx, (unsigned)num_kv_heads, (unsigned)n), dim3(kSumThreads), 0, st, p);
  }
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
  VTKV_REQUIRE((int64_t)num_seqs * num_kv_heads < (1 << 20), "too many sequences");
  VTKV_REQUIRE(vtkv::int4_head_size(head_size), "head_size %d is not supported (64, 80, 96, 112, 128, 256)", head_size);
  VTKV_REQUIRE(kv_dtype == VTKV_F32 || kv_dtype == VTKV_BF16 || kv_dtype == VTKV_F16 || kv_dtype == VTKV_FP8_E4M3 ||
                   kv_dtype == VTKV_INT4, "bad kv_dtype %d", kv_dtype);
  VTKV_REQUIRE(keep_rows > 0 && recent_rows >= 0 && recent_rows <= keep_rows,
               "keep_rows %d must be positive and recent_rows %d between 0 and keep_rows", keep_rows, recent_rows);
  VTKV_REQUIRE(max_seq_len > 0, "max_seq_len must be > 0");
  VTKV_REQUIRE(weights_apart(slot_stride, head_stride, num_slots, num_kv_heads, max_seq_len),
               "weights of different slots and kv heads overlap");
  const intptr_t lens_apart = (intptr_t)new_seq_lens - (intptr_t)seq_lens, lens_bytes = (intptr_t)num_seqs * 4;
  VTKV_REQUIRE(lens_apart == 0 || lens_apart >= lens_bytes || -lens_apart >= lens_bytes,
               "new_seq_lens must be seq_lens itself or apart from it");
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
  const dim3 grid((unsigned)(num_seqs * num_kv_heads));
  hipStream_t st = (hipStream_t)stream;
  const int most_old = max_seq_len - recent_rows;
  p.held = most_old <= kHeldKeys;
  const size_t lds = p.held && most_old > 0 ? (size_t)most_old * sizeof(unsigned) : 0;
  if (p.head_bytes % 16 == 0)
    hipLaunchKernelGGL(evict_kernel<16>, grid, dim3(kEvictThreads), lds, st, p);
  else
    hipLaunchKernelGGL(evict_kernel<8>, grid, dim3(kEvictThreads), lds, st, p);
  if (new_seq_lens == seq_lens)
    hipLaunchKernelGGL(cut_lengths_kernel, dim3((unsigned)((num_seqs + 255) / 256)), dim3(256), 0, st, new_seq_lens, slot_ids,
                       num_slots, num_seqs, keep_rows);
  VTKV_HIP(hipGetLastError());
  return VTKV_OK;
}

}  // extern "C"
