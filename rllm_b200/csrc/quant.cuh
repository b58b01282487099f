// What the kernels of quantised serving share: the rounding of a quotient, and the layout of the cache held in 4 bits.
//
// Rows in 8 bits: s = float(max |x| / 127), code = x / s to the nearest integer, ties to even. Groups of 32 numbers of a head in
// 4 bits: m the number of largest magnitude (the positive one of two), d = bf16(m / -8), code = x / d to the nearest integer, ties
// to even, clamped to -8..7; the number stands for code * d. The sign of d puts m itself on -8, so that all sixteen codes are
// used: the step is max / 8 where codes -7..7 with a positive scale would have max / 7, 23 % less noise power.
// A row (group) with an infinity or a NaN gets a scale of NaN and reads back as NaN throughout.
#pragma once
#include "common.cuh"

namespace rllm {

// x / s to the nearest integer by the exact quotient, ties to even, for quotients below 2^9. `inv` is 1 / s, rounded: x * inv is
// off by less than 2^-13, so only a product within 2^-12 of a half-integer leaves the question open. Then the quotient is
// rounded once by the division; where that gives a half-integer, the remainder x - q s (exact, as the quotient is to the
// nearest) says on which side of it the exact quotient lies.
__device__ __forceinline__ float round_quotient(float x, float s, float inv) {
  const float q0 = x * inv;
  float r = rintf(q0);
  if (fabsf(q0 - r) > 0.5f - 0.000244140625f) {
    const float q = __fdiv_rn(x, s);
    r = rintf(q);
    if (fabsf(q - r) == 0.5f) {
      const float rem = fmaf(-q, s, x);
      if (rem != 0.f) r = ((rem > 0.f) == (s > 0.f)) ? q + 0.5f : q - 0.5f;
    }
  }
  return r;
}

// One layer's keys (or values) in 4 bits: codes [page][kv head][offset in page][hd / 2 bytes], scales bf16 [..][hd / 32]. 64
// dimensions are 8 words (32 bytes); word w holds dimensions 4w..4w+3 in its lower half and 32 + 4w..32 + 4w + 3 in its upper half,
// the first dimension in the lowest nibble; a nibble is code + 8. A word so holds four numbers of each of two groups: the halves
// of two words, put side by side, are pairs of numbers of one group, which is what a fragment of a matrix instruction wants.
__device__ __forceinline__ int code4(uint32_t word, int i) { return (int)((word >> (4 * i)) & 15u) - 8; }   // i: 0..3 lower group, 4..7 upper
__device__ __forceinline__ float bf16_lo(uint32_t two) { return __uint_as_float(two << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t two) { return __uint_as_float(two & 0xffff0000u); }

}  // namespace rllm
