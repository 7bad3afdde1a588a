// The 8-bit block format of the dense products: e4m3 codes, one e8m0 scale per 32 elements (norm.cu says how it is chosen).
#pragma once

#include <stdint.h>

namespace pnv {

constexpr uint32_t kMx8One = 127;                 // scale byte of 1.0
constexpr uint32_t kMx8NaN = 0xFF;
constexpr uint32_t kMx8SlopWord = 0x7F7F7F7Fu;

// Scale byte from the bits of the block's largest magnitude (as float bits: infinities and NaNs are above all numbers).
// With 448 = 1.75 * 2^8 the smallest power of two that brings it to 448 or below has the magnitude's exponent less 8, and one
// more where the mantissa is above 1.75: that carry is the addition's.
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return kMx8NaN;
  if (amax_bits == 0) return kMx8One;
  return (uint32_t)max((int)((amax_bits + 0x1FFFFFu) >> 23) - 8, 0);
}
// 2^(127 - byte), what the elements are multiplied with: exact, no scale byte of finite elements is above 247.
__device__ __forceinline__ float mx8_inverse(uint32_t byte) { return __uint_as_float((254u - (byte == kMx8NaN ? kMx8One : byte)) << 23); }

// Codes of v[at .. at + 3], first element in the lowest byte.
template <int N>
__device__ __forceinline__ uint32_t mx8_codes4(const float (&v)[N], int at, uint32_t byte, float inv) {
  if (byte == kMx8NaN) return 0x7F7F7F7Fu;        // e4m3 NaN
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r) : "f"(v[at] * inv), "f"(v[at + 1] * inv), "f"(v[at + 2] * inv), "f"(v[at + 3] * inv));
  return r;
}

}  // namespace pnv
