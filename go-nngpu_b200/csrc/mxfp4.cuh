// One block of the microscaled 4-bit format: scale, codes and back.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace gonn {
namespace mxfp4 {

constexpr uint32_t kScaleNan = 255;  // the block holds a NaN or an infinity

// Scale byte of a block whose largest magnitude has the bits `amax` (float, sign cleared):
// 127 + e with e = floor(log2 amax) - 2, so that the largest element lies in [4, 8) 2^e and the
// largest code, 6, in the same binade; at least e = -127.  The exponent field of a normal
// number is floor(log2) + 127; subnormal numbers and 0 give the smallest scale.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const uint32_t field = amax >> 23;
  if (field == 255u) return kScaleNan;
  return field > 2u ? field - 2u : 0u;
}
// 2^(127 - byte): what an element is multiplied by before it is rounded.  Never subnormal,
// since byte <= 252 (byte 255: 0, every code of such a block is 0).
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return byte == kScaleNan ? 0.f : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == kScaleNan ? __uint_as_float(0x7fffffffu)
                           : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
}
// e2m1 codes of `lo` (bits 0-3) and `hi` (bits 4-7): nearest, ties to even, magnitudes above 6
// become 6.
__device__ __forceinline__ uint32_t encode2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 b;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\t"
      "cvt.u32.u8 %0, b;\n\t"
      "}\n"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}
// The value of the code in the low four bits: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives.  Moved
// to the top of a float's exponent and mantissa the three bits read as that value times 2^-126
// (code 1, like the code itself, as a subnormal number).
__device__ __forceinline__ float decode(uint32_t code) {
  return __uint_as_float(((code & 7u) << 22) | ((code & 8u) << 28)) * 0x1p126f;
}

}  // namespace mxfp4
}  // namespace gonn
