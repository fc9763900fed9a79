// One MXFP4 block: its UE8M0 code and its E2M1 nibbles (see mx.cu).
#pragma once

#include "common.cuh"

namespace nvfp4b200 {
namespace mx {

// From the largest |v| of a block: its UE8M0 code and 2^(127 - code).  With the
// exponent held at 2 or above, code = exponent - 2 and the inverse's exponent
// is 256 - exponent; an infinite or NaN maximum gives code 255.
__device__ __forceinline__ void block_scale(float amax, uint32_t& code, float& inverse) {
  const uint32_t e = __float_as_uint(amax) & 0x7F800000u, t = max(e, 0x01000000u);
  inverse = __uint_as_float(0x80000000u - t);
  code = e == 0x7F800000u ? 255u : (t >> 23) - 2u;
}

// 2^(code - 127); code 0 is the subnormal 2^-127, code 255 is NaN.
__device__ __forceinline__ float code_scale(uint32_t code) {
  if (code == 255u) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(code ? code << 23 : 0x00400000u);
}

// 8 scaled values -> 8 E2M1 nibbles, element 0 in the low nibble of the low byte.
__device__ __forceinline__ uint32_t encode8(const float (&f)[8]) {
  uint32_t out;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(out)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return out;
}

}  // namespace mx
}  // namespace nvfp4b200
