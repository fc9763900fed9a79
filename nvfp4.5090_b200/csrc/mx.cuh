// One MXFP4 block: its UE8M0 code and its E2M1 nibbles (see mx.cu).
#pragma once

#include "common.cuh"

namespace nvfp4b200 {
namespace mx {

// UE8M0 code from the largest |v| of a block, given as fp32 bits.
__device__ __forceinline__ uint32_t block_code(uint32_t amax_bits) {
  const int field = (int)(amax_bits >> 23);
  return field == 255 ? 255u : (uint32_t)max(field - 2, 0);
}

// 2^(127 - code) for a finite code (at most 252, so the field stays normal).
__device__ __forceinline__ float code_inverse(uint32_t code) {
  return __uint_as_float((254u - min(code, 252u)) << 23);
}

// 2^(code - 127); code 0 is the subnormal 2^-127, code 255 is NaN.
__device__ __forceinline__ float code_scale(uint32_t code) {
  if (code == 255u) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(code ? code << 23 : 0x00400000u);
}

// 8 values -> 8 E2M1 nibbles, element 0 in the low nibble of the low byte.
__device__ __forceinline__ uint32_t encode8(const float (&f)[8], float inv) {
  uint32_t out;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(out)
      : "f"(f[0] * inv), "f"(f[1] * inv), "f"(f[2] * inv), "f"(f[3] * inv), "f"(f[4] * inv), "f"(f[5] * inv),
        "f"(f[6] * inv), "f"(f[7] * inv));
  return out;
}

}  // namespace mx
}  // namespace nvfp4b200
