// Device helpers of the MXFP8 cache: the scale byte of a block from its largest magnitude, and E4M3 codes back to bf16.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace nc {

// Scale byte of a block from the bits of its largest |x| (bf16): biased exponent of the smallest power of two with
// 448 * 2^(b - 127) >= |x|. 448 = 1.75 * 2^8, so the answer is read off the exponent and mantissa fields:
// 1.m * 2^(E - 127) <= 1.75 * 2^(E - 127) needs b = E - 8, a larger mantissa one more. Zero: 127. Infinity: 253, the
// top of the range. NaN (its bits compare above infinity's): 255, the value that makes the whole block NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 7, m = amax_bits & 0x7f;
  const int b = static_cast<int>(e) - (m > 0x60 ? 7 : 8);
  if (amax_bits >= 0x7f80) return amax_bits > 0x7f80 ? 255u : 253u;
  return amax_bits == 0 ? 127u : static_cast<uint32_t>(b < 1 ? 1 : b);
}

// E4M3 -> bf16. A code's fields, put at bf16's mantissa top and exponent bottom, read as value * 2^-120 (biases 7 and
// 127), subnormals included; the multiplication that brings it back also applies the block's scale, and is exact:
// four significant bits, and every product of the ordinary range is a normal bf16 number. The multiplier
// 2^(b - 127 + 120) has a bf16 exponent field for b <= 134 (blocks up to 57344); above that a second factor takes the rest.
// The codes 0x7f / 0xff (NaN) only occur in blocks of scale 255, whose factor is NaN.
__device__ __forceinline__ uint32_t mx_factor_first(uint32_t b) { return (b < 134u ? b + 120u : 254u) << 7; }
__device__ __forceinline__ uint32_t mx_factor_second(uint32_t b) {
  return b <= 134u ? 0x3f80u : (b == 255u ? 0x7fc0u : (b - 134u + 127u) << 7);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Codes in bytes 0, 1 (lo) and 2, 3 (hi) of w -> bf16 pairs, not yet multiplied. With the codes in the low bytes of 16-bit
// fields, x * 16 puts the seven bits below the sign in place and the sign four places too low: 240 times the sign bit
// moves it up. (Multiplications, because logic runs at half their rate and is what these loops are short of.)
__device__ __forceinline__ void mx_spread(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t x = __byte_perm(w, 0, 0x4140), y = __byte_perm(w, 0, 0x4342);
  lo = (x & 0x00800080u) * 240u + x * 16u;
  hi = (y & 0x00800080u) * 240u + y * 16u;
}

}  // namespace nc
