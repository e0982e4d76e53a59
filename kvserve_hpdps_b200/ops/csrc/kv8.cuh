// A paged KV cache held in 8 bits: layout and arithmetic shared by the kernels that write, read
// and attend over it.
//
// A (block, head) record of a cache with block size bs has 2 bs + 1 rows of 128 bytes:
//   K codes [bs][128]   V codes [bs][128]   scales [128]
// A code is an e4m3 number.  Each unit of 16 tokens has two bytes in the last row, for its keys and
// its values: a channel reads
//   value = code * 2^(byte - 127),
// and a byte of 0 (nothing written yet) reads as zeros.
//
// The exponent of a unit is the smallest e with amax <= 448 * 2^e, amax its largest finite
// magnitude, but at least kLowScale.  Why powers of two: e4m3's precision is relative, 2^-4 of each
// value wherever it lies between 2^-6 and 448, so a finer scale gains nothing; and codes that
// follow a scale which has grown, matrix operands, and weights times a value's scale then stay
// exact but for e4m3's subnormals.  Why e4m3 and not 8-bit integers: keys have channels that
// are ten times larger than the rest, and steps of the unit's largest magnitude / 127 would leave the
// others 8 % of error where e4m3 leaves 2.6 %.
#pragma once

#include "kv4.cuh"

namespace kvs {

constexpr int kUnit8 = 16;        // tokens that share a scale
constexpr int kLowScale = -110;   // smallest exponent: 448 times it is still a normal fp32 number
constexpr int kTopByte = 127 + 120;  // fp32's largest number needs 120

KVS_DEV float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// The exponent for a largest magnitude given by its bits (finite).
KVS_DEV int scale_exponent(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23) - 135 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return max(e, kLowScale);
}
// Two fp32 numbers as e4m3 codes, rounded to nearest even; what is not a number stays so.
KVS_DEV uint32_t codes8(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
KVS_DEV uint32_t codes8x4(const float* x) { return codes8(x[0], x[1]) | codes8(x[2], x[3]) << 16; }
// The codes in the low and in the high half of a word as fp16 pairs, exact.
KVS_DEV uint32_t half2_low8(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n"
      : "=r"(d)
      : "r"(w));
  return d;
}
KVS_DEV uint32_t half2_high8(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}\n"
      : "=r"(d)
      : "r"(w));
  return d;
}
// Four codes as fp32 numbers.
KVS_DEV void values8x4(uint32_t w, float* x) {
  const uint32_t a = half2_low8(w), b = half2_high8(w);
  x[0] = h2f<true>(a & 0xFFFFu), x[1] = h2f<true>(a >> 16);
  x[2] = h2f<true>(b & 0xFFFFu), x[3] = h2f<true>(b >> 16);
}
// The same in e5m2, which is fp16's upper byte.
KVS_DEV uint32_t codes52(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
KVS_DEV uint32_t codes52x4(const float* x) {
  return codes52(x[0], x[1]) | codes52(x[2], x[3]) << 16;
}
KVS_DEV void values52x4(uint32_t w, float* x) {
  x[0] = h2f<true>((w & 0xFFu) << 8), x[1] = h2f<true>(w & 0xFF00u);
  x[2] = h2f<true>(w >> 8 & 0xFF00u), x[3] = h2f<true>(w >> 16 & 0xFF00u);
}

}  // namespace kvs
