// Numbers in 8 bits with a scale for each block of 128: x = code * 2^(scale - 127), code an e4m3 number.
//
// The scale is the smallest power of two that brings the block's largest magnitude to 448 or less, so dividing by it is
// exact and a value is rounded once, to nearest, ties to even; a block of zeros has scale 1 (127).  What is not finite
// does not count for the scale and is held as NaN.
#pragma once
#include "kad_vec.h"

namespace kad {

constexpr int BLOCK8 = 128;

typedef int intx8 __attribute__((ext_vector_type(8)));

// The bits of |v|, 0 where v is not finite: compared as whole numbers.
__device__ __forceinline__ uint32_t magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// A block's scale from the bits of its largest magnitude: 448 is 1.75 * 2^8.
__device__ __forceinline__ int scale_of(uint32_t bits) {
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
  return bits == 0 ? 127 : e > 0 ? e : 0;
}
// 2^(127 - scale), what a value is multiplied by; scale <= 247.
__device__ __forceinline__ float inverse(int scale) { return __uint_as_float((uint32_t)(254 - scale) << 23); }

// Four codes of four values times inv.
__device__ __forceinline__ int codes_of(float a, float b, float c, float d, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
}

}  // namespace kad
