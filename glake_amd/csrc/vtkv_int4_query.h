// Queries on their way to the dot products with bare 4-bit codes (vtkv_int4.h), shared by the kernels that form them.
//
// The codes of a word come as fp16 numbers c * 2^-24 (registers 0 and 2 of an operand) and c * 2^-20 (1 and 3), register r
// holding codes r and r + 4.  The other factor goes into q: a power of two per query head (and token) brings its largest value
// near 2^14 in fp16, the odd registers take a sixteenth of it.  That is exact for a bf16 value down to 2^-27 of its head's
// largest and for an fp16 value down to 2^-24; a smaller one is off by 2^-35 of the largest at most.  A head's dot products are
// brought back by its own power, so what another head or token of the same operand holds does not touch them.  The largest
// magnitude is found on pairs of 16-bit patterns and sum(q) comes from the matrix pipe: half the instructions of the plain
// form and eight registers less in the decode kernel (its times are the same).
#pragma once
#include "vtkv_attn_common.h"

namespace vtkv_attn {

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// The largest finite magnitude among pairs of 16-bit numbers.  Patterns without sign are in the order of the magnitudes;
// raised by one step of the exponent, infinity and NaN become negative and are passed over (they stay with their head).
template <bool F16>
struct LargestQuery {
  static constexpr unsigned short kStep = F16 ? 0x0400 : 0x0080;
  i16x2 most = {(short)kStep, (short)kStep};
  __device__ __forceinline__ void take(u32x4 raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned pair = raw[i] & 0x7fff7fffu;
      const u16x2 raised = __builtin_bit_cast(u16x2, pair) + (u16x2){kStep, kStep};
      most = __builtin_elementwise_max(most, __builtin_bit_cast(i16x2, raised));
    }
  }
  // of the lane's column, whose values its four row groups hold
  __device__ __forceinline__ float value() const {
    const unsigned bits = (unsigned)max((int)most[0], (int)most[1]) - kStep;
    return max_over_row_groups(unpack_16<F16>(bits, 0));
  }
};

// The power of two (and its inverse) that brings `largest` into [2^14, 2^15).
struct QueryScale {
  float up, down;
};
__device__ __forceinline__ QueryScale query_scale(float largest) {
  const int expo = max((int)(__builtin_bit_cast(unsigned, largest) >> 23), 15);
  return {__builtin_bit_cast(float, (unsigned)(268 - expo) << 23), __builtin_bit_cast(float, (unsigned)(expo - 14) << 23)};
}

// Eight query values as an operand.
template <bool F16>
__device__ __forceinline__ u32x4 query_operand(u32x4 raw, float up) {
  u32x4 op;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float f = r & 1 ? up * 0.0625f : up;
    const unsigned a = raw[r >> 1], b = raw[2 + (r >> 1)];
    op[r] = pack_16x2<true>(unpack_16<F16>(a, r & 1) * f, unpack_16<F16>(b, r & 1) * f);
  }
  return op;
}

// up * sum(q) of the lane's column in every element: a product with ones, sixteen where a register holds a sixteenth.
template <int STEPS>
__device__ __forceinline__ float query_sum(const u32x4 (&op)[STEPS]) {
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
    sum = mfma_16x16x32<true>((u32x4){0x3c003c00u, 0x4c004c00u, 0x3c003c00u, 0x4c004c00u}, op[s], sum);
  return sum[0];
}

}  // namespace vtkv_attn
