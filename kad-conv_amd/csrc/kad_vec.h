// 16-byte vectors of a map's or row's values at any alignment, and parameters of either type.
#pragma once
#include "kad_common.h"

namespace kad {

__device__ __forceinline__ float load_param(const void* p, int i, int dtype, float none) {
  if (!p) return none;
  if (dtype == KAD_F32) return ((const float*)p)[i];
  if (dtype == KAD_F16) return (float)((const half_t*)p)[i];
  return (float)((const bf16_t*)p)[i];
}
__device__ __forceinline__ void store_param(void* p, int i, int dtype, float v) {
  if (dtype == KAD_F32) ((float*)p)[i] = v;
  else if (dtype == KAD_F16) ((half_t*)p)[i] = (half_t)v;
  else ((bf16_t*)p)[i] = (bf16_t)v;
}

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);
// 16 bytes at a T's alignment.
typedef int intx4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef int intx4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct Loose { typedef intx4_at2 type; };
template <> struct Loose<float> { typedef intx4_at4 type; };
template <typename T> using loose = typename Loose<T>::type;

// 16 bytes at an address that need only be a T's (the memory unit takes wide accesses at any address).
template <typename T>
__device__ __forceinline__ intx4 load_vec(const T* p) {
  intx4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack(intx4 r, float v[VEC<T>]) {
  T t[VEC<T>];
  __builtin_memcpy(t, &r, 16);
#pragma unroll
  for (int i = 0; i < VEC<T>; ++i) v[i] = to_f32(t[i]);
}
// Forgets what was computed from a held vector: otherwise its unpacked values stay in registers too.
__device__ __forceinline__ void repack(intx4& r) { asm volatile("" : "+v"(r)); }
template <typename T>
__device__ __forceinline__ intx4 pack(const float v[VEC<T>]) {
  T t[VEC<T>];
#pragma unroll
  for (int i = 0; i < VEC<T>; ++i) t[i] = from_f32<T>(v[i]);
  intx4 r;
  __builtin_memcpy(&r, t, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float v[VEC<T>]) {
  const intx4 r = pack<T>(v);
  __builtin_memcpy(p, &r, 16);
}
// Past the caches.
template <typename T>
__device__ __forceinline__ void stream_vec(T* p, const float v[VEC<T>]) {
  __builtin_nontemporal_store(pack<T>(v), (loose<T>*)p);
}
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float v[VEC<T>]) {
#pragma unroll
  for (int i = 0; i < VEC<T>; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float v[VEC<T>]) {
#pragma unroll
  for (int i = 0; i < VEC<T>; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

// Orders a wave's accesses to LDS: the unit takes them in turn, so it is the compiler alone that has to.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace kad
