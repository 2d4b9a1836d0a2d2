// Block-scaled 8-bit values, shared by the quantisers and the 8-bit grouped GEMM.
//
// A block of 128 values (of one row) or of 128 x 128 values (of a weight)
// holds e4m3 numbers and one scale, a power of two 2^e kept as the biased
// exponent byte e + 127 (E8M0). e is the smallest integer with
// amax <= 448 * 2^e, 448 = 1.75 * 2^8 being the largest e4m3 number, so no
// value saturates. Dividing by a power of two is exact, so a value meets one
// rounding alone (to nearest even, at most half a step: 2^-4 of a normal
// e4m3 value), and the tensor core multiplies the scales itself
// (tcgen05 block scaling takes E8M0). A block of zeros has scale 1.
// Infinities and NaN do not enter amax and become NaN, so that a product
// they enter shows them.
#pragma once

#include "moe_common.cuh"

namespace moe {
namespace fp8 {

constexpr int kBlock = 128;
constexpr uint32_t kOne = 127;  // scale byte of 2^0

// |x| of a finite x, 0 of an infinity or NaN.
MOE_DEVICE float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// Scale byte of a block whose largest finite magnitude is amax. With
// amax = m * 2^p (1 <= m < 2): e = p - 8 if m <= 1.75, else p - 7. Adding
// 0x1FFFFF to the bits carries into the exponent exactly when the mantissa
// exceeds that of 1.75 (0x600000). Subnormal amax and anything below the
// scale type's range take its smallest scale, 2^-127.
MOE_DEVICE uint32_t scale_byte(float amax) {
  const uint32_t up = (__float_as_uint(amax) + 0x1FFFFFu) >> 23;  // biased exponent of 448 * 2^e, less 8
  return amax > 0.f ? (up > 8u ? up - 8u : 0u) : kOne;
}

// 2^-e of a scale byte that scale_byte gave (at most 247, so this is normal).
MOE_DEVICE float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// 2^e of any scale byte (255 is NaN, 0 the subnormal 2^-127).
MOE_DEVICE float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}

// x / 2^e for the conversion; an infinity becomes NaN instead of saturating.
MOE_DEVICE float scaled(float x, float inv) {
  return fabsf(x) == INFINITY ? __uint_as_float(0x7FC00000u) : x * inv;
}

// Two values to e4m3, round to nearest even, lo in the low byte.
MOE_DEVICE uint32_t pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
MOE_DEVICE uint32_t pack4(float a, float b, float c, float d) {
  return pack2(a, b) | (pack2(c, d) << 16);
}

// Two e4m3 values (low byte first) to fp32, exact.
MOE_DEVICE float2 unpack2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  float2 f;
  asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}"
      : "=f"(f.x), "=f"(f.y)
      : "r"(h));
  return f;
}

}  // namespace fp8
}  // namespace moe
