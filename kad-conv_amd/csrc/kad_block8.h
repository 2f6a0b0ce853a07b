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

// Magnitudes as whole numbers, which order as the values do: of two 16-bit values or one of 32 bits in a word.
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
template <typename T> struct Bits {
  static constexpr uint32_t INF = sizeof(T) == 4 ? 0x7F800000u : 0x7C00u;  // half
  static constexpr uint32_t SIGNLESS = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
};
template <> struct Bits<bf16_t> {
  static constexpr uint32_t INF = 0x7F80u, SIGNLESS = 0x7FFF7FFFu;
};

template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) return a > b ? a : b;
  const ushort2_t m = __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b));
  return __builtin_bit_cast(uint32_t, m);
}
template <typename T>
__device__ __forceinline__ uint32_t magnitudes(uint32_t w) { return w & Bits<T>::SIGNLESS; }
// The larger of a word's two.
template <typename T>
__device__ __forceinline__ uint32_t largest_of(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  const uint32_t lo = m & 0xFFFFu, hi = m >> 16;
  return lo > hi ? lo : hi;
}
template <typename T>
__device__ __forceinline__ bool all_finite(uint32_t m) { return largest_of<T>(m) < Bits<T>::INF; }
// 0 in place of what is not finite.
template <typename T>
__device__ __forceinline__ uint32_t finite_of(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m < Bits<T>::INF ? m : 0u;
  const uint32_t lo = m & 0xFFFFu, hi = m >> 16;
  return (lo < Bits<T>::INF ? lo : 0u) | (hi < Bits<T>::INF ? hi : 0u) << 16;
}

// A block's scale from its largest finite magnitude: 448 is 1.75 * 2^8.
template <typename T>
__device__ __forceinline__ int scale_of(uint32_t m) {
  uint32_t bits = m;
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = (uint16_t)m;
    T v;
    __builtin_memcpy(&v, &h, 2);
    bits = __float_as_uint(to_f32(v));
  }
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
  return bits == 0 ? 127 : e > 0 ? e : 0;
}

// Four codes of four values: two words of two 16-bit ones, or four words.  The conversion divides by the power of two that
// it is given the exponent of, and rounds once; checked for every 16-bit value against a product and a rounding.
typedef short short2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ int codes_of(uint32_t a, uint32_t b, int scale) {
  const float s = __uint_as_float((uint32_t)scale << 23);
  short2_t r = {0, 0};
  if constexpr (__is_same(T, bf16_t)) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, a), s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, b), s, true);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(half2_t, a), s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(half2_t, b), s, true);
  }
  return __builtin_bit_cast(int, r);
}
__device__ __forceinline__ int codes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int scale) {
  const float s = __uint_as_float((uint32_t)scale << 23);
  short2_t r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(a), __uint_as_float(b), s, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(c), __uint_as_float(d), s, true);
  return __builtin_bit_cast(int, r);
}

// The largest finite magnitude among N words.
template <typename T, int N>
__device__ __forceinline__ uint32_t largest_finite(const uint32_t* w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = larger<T>(m, magnitudes<T>(w[i]));
  if (!all_finite<T>(m)) {
    m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = larger<T>(m, finite_of<T>(magnitudes<T>(w[i])));
  }
  return largest_of<T>(m);
}

template <typename T> constexpr int LANES = BLOCK8 / VEC<T>;  // that share a row's block

// Largest over the N (16 or 32) lanes of a row, by lane permutations of the vector unit.
template <int N>
__device__ __forceinline__ uint32_t lanes_largest(uint32_t v) {
  const auto with = [&](uint32_t o) { v = v > o ? v : o; };
  with(__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true));   // lane ^ 1
  with(__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true));   // lane ^ 2
  with(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));  // 7 - lane of eight
  with(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true));  // 15 - lane of sixteen
  if (N == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = r[0] > r[1] ? r[0] : r[1];
  }
  return v;
}

}  // namespace kad
