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

// x / s to the nearest integer by the exact quotient, ties to even, |x / s| below 2^9, s normal; inv is 1 / s, rounded. x * inv is off by
// less than 2^-13, so its nearest integer r is at most one off, next to a half-integer. What x has more than r s is a multiple of the
// last place of s and not above s, or a difference of numbers within a factor of two: the fused product gives it exactly, and half of s
// decides.
__device__ __forceinline__ int round_quotient(float x, float s, float inv) {
  const float y = fmaf(x, inv, 12582912.f);              // 1.5 2^23: the last bits are the integer
  const int r = __float_as_int(y) - 0x4b400000;
  const float e = fmaf(12582912.f - y, s, x), over = fabsf(e) - 0.5f * fabsf(s);
  const bool step = over > 0.f || (over == 0.f && (r & 1));
  return step ? r + ((e > 0.f) == (s > 0.f) ? 1 : -1) : r;
}

// A row's (group's) scale as the rounding wants it: where it is small enough for its inverse to leave the float range, numbers and scale
// are taken times 2^64.
struct Rounding {
  float up, s, inv;
  __device__ __forceinline__ explicit Rounding(float scale) {
    up = fabsf(scale) < 1e-30f ? 18446744073709551616.f : 1.f;
    s = scale * up;
    inv = 1.f / s;
  }
  __device__ __forceinline__ int code(float x, int lo, int hi) const { return min(max(round_quotient(x * up, s, inv), lo), hi); }
};

// Four 8-bit codes in a word, rounded by the exact quotients (out of line: most of the code, run for one group of four in 170, as half of a
// bfloat16 row's largest number is on a border).
static __device__ __noinline__ uint32_t codes8_exact(float a, float b, float c, float d, float s, float inv) {
  const int lo = -127, hi = 127;
  return ((uint32_t)min(max(round_quotient(a, s, inv), lo), hi) & 0xffu) | ((uint32_t)min(max(round_quotient(b, s, inv), lo), hi) & 0xffu) << 8 |
         ((uint32_t)min(max(round_quotient(c, s, inv), lo), hi) & 0xffu) << 16 | (uint32_t)min(max(round_quotient(d, s, inv), lo), hi) << 24;
}
// The 8-bit codes of N numbers of a row with scale s > 0, four a word, `rd` the row's Rounding. The exact quotient lies between x times numbers just below and just above 1 / s; where both have the same nearest integer, it is that. (A division
// for every number took as long again as a prompt's memory.)
template <int N>
__device__ __forceinline__ void codes8(const float (&v)[N], const Rounding& rd, uint32_t (&w)[N / 4]) {
  const float lo = rd.inv * (1.f - 2.384185791e-7f), hi = rd.inv * (1.f + 2.384185791e-7f);      // 2^-22, more than the two roundings of inv
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    uint32_t y[4], differ = rd.up != 1.f;                // (a tiny scale may have been rounded far enough down for codes beyond 127)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = __float_as_uint(fmaf(v[i + e], lo, 12582912.f));            // 1.5 2^23: the last byte is the code
      differ |= y[e] ^ __float_as_uint(fmaf(v[i + e], hi, 12582912.f));
    }
    w[i / 4] = __byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410);
    if (differ) w[i / 4] = codes8_exact(v[i] * rd.up, v[i + 1] * rd.up, v[i + 2] * rd.up, v[i + 3] * rd.up, rd.s, rd.inv);
  }
}

// silu(g) u; in full float precision, or for a result that is rounded to bfloat16
__device__ __forceinline__ float silu_gate(float g, float u, bool precise) {
  return precise ? g / (1.f + expf(-g)) * u : __fdividef(g, 1.f + __expf(-g)) * u;
}

// One layer's keys (or values) in 4 bits: codes [page][kv head][offset in page][hd / 2 bytes], scales bf16 [..][hd / 32]. 64
// dimensions are 8 words (32 bytes); word w holds dimensions 4w..4w+3 in its lower half and 32 + 4w..32 + 4w + 3 in its upper half,
// the first dimension in the lowest nibble; a nibble is code + 8. A word so holds four numbers of each of two groups: the halves
// of two words, put side by side, are pairs of numbers of one group, which is what a fragment of a matrix instruction wants.
__device__ __forceinline__ int code4(uint32_t word, int i) { return (int)((word >> (4 * i)) & 15u) - 8; }   // i: 0..3 lower group, 4..7 upper
__device__ __forceinline__ float bf16_lo(uint32_t two) { return __uint_as_float(two << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t two) { return __uint_as_float(two & 0xffff0000u); }

// How a page of values is held in the scratch of portions (kv4_read_kernel writes it, the portions' kernels read it): 16-bit numbers times
// 2^e, half numbers or, `wide`, bfloat16. One word a page and kv head. A group whose scale is NaN holds zeros there, so that the products of rows
// that do not see it stay as they are; the word says that there are such (`lost`), and a bit a place in [page][kv head][group][page
// size / 32] words which.
__host__ __device__ __forceinline__ int value_word(int e, bool wide, bool lost) { return 4 * e + (lost ? 2 : 0) + (wide ? 1 : 0); }
__host__ __device__ __forceinline__ int value_exponent(int word) { return word >> 2; }
__host__ __device__ __forceinline__ bool value_lost(int word) { return word & 2; }
__host__ __device__ __forceinline__ bool value_wide(int word) { return word & 1; }
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
constexpr int VALUE_EXPONENTS = 48;           // e lies between -48 and 48,
constexpr int ZEROS_EXPONENT = -70;           // that of a page of zeros below

}  // namespace rllm
