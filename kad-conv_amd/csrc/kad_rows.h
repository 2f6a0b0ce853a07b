// Rows of values in the registers of a few threads.
//
// A row belongs to G threads (a power of two), each with U 16-byte vectors of V values.  Where V does not divide its
// length, the last vector is moved back to end with the row: what it shares with the one before is computed and written
// twice, with the same bits, and counted once in sums.  So any row of V values and more is read in whole vectors, at any
// alignment; shorter ones go a value a thread.
#pragma once
#include "kad_vec.h"

namespace kad {

#define KAD_DPP(x, ctrl) __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), ctrl, 0xf, 0xf, true))
// Sum over the G (a power of two, at most 64) threads that share a row, by lane permutations of the vector unit.
__device__ __forceinline__ float lanes_sum(float v, int G) {
  if (G >= 2) v += KAD_DPP(v, 0xB1);    // lane ^ 1
  if (G >= 4) v += KAD_DPP(v, 0x4E);    // lane ^ 2
  if (G >= 8) v += KAD_DPP(v, 0x141);   // 7 - lane of eight: the other four, whose values are equal by now
  if (G >= 16) v += KAD_DPP(v, 0x140);  // 15 - lane of sixteen
  if (G >= 32) v = sum_xor16(v);
  if (G >= 64) v = sum_xor32(v);
  return v;
}

__device__ __forceinline__ float lanes_max(float v, int G) {
  if (G >= 2) v = fmaxf(v, KAD_DPP(v, 0xB1));
  if (G >= 4) v = fmaxf(v, KAD_DPP(v, 0x4E));
  if (G >= 8) v = fmaxf(v, KAD_DPP(v, 0x141));
  if (G >= 16) v = fmaxf(v, KAD_DPP(v, 0x140));
  if (G >= 32) v = fmaxf(v, __shfl_xor(v, 16));
  if (G >= 64) v = fmaxf(v, __shfl_xor(v, 32));
  return v;
}

#undef KAD_DPP

// Over all threads of a row; beyond a wave through red (one float a wave and call), with one barrier.
__device__ __forceinline__ float row_sum(float v, int G, float* red) {
  v = lanes_sum(v, G);
  if (G > 64) {
    const int wave = threadIdx.x >> 6, waves = G >> 6, first = wave & ~(waves - 1);
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = red[first];
    for (int i = 1; i < waves; ++i) v += red[first + i];
  }
  return v;
}

// Two at once (two floats a wave).
__device__ __forceinline__ void row_sums(float& v, float& w, int G, float* red) {
  v = lanes_sum(v, G);
  w = lanes_sum(w, G);
  if (G > 64) {
    const int wave = threadIdx.x >> 6, waves = G >> 6, first = wave & ~(waves - 1);
    if ((threadIdx.x & 63) == 0) {
      red[2 * wave] = v;
      red[2 * wave + 1] = w;
    }
    __syncthreads();
    v = red[2 * first];
    w = red[2 * first + 1];
    for (int i = 1; i < waves; ++i) {
      v += red[2 * (first + i)];
      w += red[2 * (first + i) + 1];
    }
  }
}

// VV values of a thread's vector: V, or 1 for rows shorter than a vector.
template <typename T, int VV>
struct Piece {
  intx4 raw;
  __device__ __forceinline__ void load(const T* p) {
    if (VV > 1) {
      raw = load_vec(p);
    } else {
      T v = p[0];
      raw = intx4{0, 0, 0, 0};
      __builtin_memcpy(&raw, &v, sizeof(T));
    }
  }
  __device__ __forceinline__ void get(float v[VV]) const {
    if constexpr (VV > 1) {
      unpack<T>(raw, v);
    } else {
      T t;
      __builtin_memcpy(&t, &raw, sizeof(T));
      v[0] = to_f32(t);
    }
  }
};
template <typename T, int VV>
__device__ __forceinline__ void put(T* p, const float v[VV]) {
  if constexpr (VV > 1) stream_vec<T>(p, v);
  else p[0] = from_f32<T>(v[0]);
}

// Where a thread's vectors lie in a row.  RAGGED: VV does not divide c.
template <int VV, int U, bool RAGGED>
struct Place {
  int at[U];     // first value
  int skip[U];   // how many of the vector's first values belong to the vector before
  bool on[U];    // there is a vector
  __device__ __forceinline__ Place(int l, int G, int c) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = (l + u * G) * VV;
      on[u] = j < c;
      at[u] = j < c - VV ? j : c - VV;
      skip[u] = RAGGED ? j - at[u] : 0;
    }
  }
  // Sum of the values that are its own.
  __device__ __forceinline__ float own(int u, const float v[VV]) const {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < VV; ++e) s += !RAGGED || e >= skip[u] ? v[e] : 0.f;
    return on[u] ? s : 0.f;
  }
};

}  // namespace kad
