// AdamW over many tensors in one launch, states in 32 or 8 bits.
//
//   m <- b1 m + (1 - b1) g     v <- b2 v + (1 - b2) g^2     p <- decay p - rate m / (sqrt(v) inv_root + eps)
//
// Every value is read and written once, so bytes bound it: 28 a value for fp32 with 32-bit states.  What a
// network of thousands of small tensors costs beside that is launches; a table of chunks in device memory
// makes it one.  A block takes a chunk (at most 4096 values of one tensor), a wave 256 values of it at a
// time, a lane 4 consecutive ones.
//
// 8-bit states: a wave's 256 values are a segment with one scale, so its largest magnitude is a wave
// reduction.  m and u = sqrt(v) are held as e4m3 (a root halves the range of exponents that v would need).
// Rounding is stochastic: in a step v changes by 1e-3 of itself, far under half of an e4m3 step, so rounding
// to nearest would leave it where it is; m likewise stops short of a steady gradient.  A u that is not 0 is
// held as the smallest positive code at least, so that a small m never meets a denominator of eps alone.
#include <math.h>

#include "kad_common.h"

namespace kad {
namespace {

constexpr int SEG = KAD_ADAMW_SEG, CHUNK = KAD_ADAMW_CHUNK;
constexpr float E4M3_MAX = 448.0f;
// Largest magnitude of a segment below which it is held as zeros: its scale would no longer be a normal float.
constexpr float SEG_TINY = 0x1p-110f;

// 32 bits in, 32 well mixed bits out; the odd factors are fractions of the square roots of 2 and 3.
__host__ __device__ inline uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}
__host__ __device__ inline uint32_t step_key(uint32_t seed, int64_t step) {
  return mix32(mix32(seed + 0x9E3779B1u) + (uint32_t)step);
}
__device__ __forceinline__ uint32_t value_bits(uint32_t key, int64_t i) {
  return mix32((uint32_t)i * 0x9E3779B1u + (uint32_t)(i >> 32) * 0x3C6EF373u + key);
}

// Four values at p, of which the first `left` (> 0) are there; pointers need the element's alignment only
// (the memory unit takes wide accesses at any address).
template <typename T>
__device__ __forceinline__ void load4(const T* p, int left, float v[4]) {
  if (left >= 4) {
    T t[4];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = to_f32(t[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = k < left ? to_f32(p[k]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, const float v[4]) {
  if (left >= 4) {
    T t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = from_f32<T>(v[k]);
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = from_f32<T>(v[k]);
  }
}

__device__ __forceinline__ void decode4(uint32_t codes, float scale, float v[4]) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * scale;
  v[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * scale;
  v[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * scale;
  v[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * scale;
}

// e4m3 code of y in [0, 448], rounded up with probability (distance to the number below) / step, for r in
// [0, 65536).  Codes of normal numbers (y >= 2^-6) are the float's bits without the last 20, less a bias;
// below, y 2^9 counts steps of 2^-9: both as fixed point with 20 bits of fraction, to which r 2^4 is added.
__device__ __forceinline__ uint32_t encode(float y, uint32_t r) {
  const uint32_t coarse = __float_as_uint(y) - (120u << 23);
  const uint32_t fine = (uint32_t)(__builtin_fminf(y, 0x1p-6f) * 0x1p29f);
  return ((y < 0x1p-6f ? fine : coarse) + (r << 4)) >> 20;
}

// Largest of the lanes' integers.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
    v = o > v ? o : v;
  }
  return v;
}

// The wave's 256 values as codes, and their scale.  Magnitudes are compared as integers, so that infinities
// and NaN count as largest: a segment that meets one is held as NaN.
template <bool POSITIVE>
__device__ __forceinline__ uint32_t encode4(const float v[4], const uint32_t r[4], float& scale) {
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t b = __float_as_uint(v[k]) & 0x7FFFFFFFu;
    most = b > most ? b : most;
  }
  most = wave_max(most);
  const float top = __uint_as_float(most);
  if (most >= 0x7F800000u) {
    scale = top;
    return 0x7F7F7F7Fu;
  }
  if (top < SEG_TINY) {
    scale = 0.f;
    return 0u;
  }
  scale = top * (1.0f / E4M3_MAX);
  const float inv = (1.0f / top) * E4M3_MAX;
  uint32_t out = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = __builtin_fabsf(v[k]);
    uint32_t c = encode(__builtin_fminf(a * inv, E4M3_MAX), r[k]);
    if (POSITIVE)
      c = (a > 0.f && c == 0) ? 1u : c;
    else
      c |= (__float_as_uint(v[k]) >> 24) & 0x80u;
    out |= c << (8 * k);
  }
  return out;
}

struct Step {
  const kad_adamw_chunk* chunks;
  void *exp_avg, *exp_avg_sq;
  float *exp_avg_scale, *exp_avg_sq_scale, *master;
  const float* grad_scale;
  const kad_adamw_scalars* scalars;
  kad_adamw_scalars values;
  float beta1, beta2, keep1, keep2, eps;  // keep = 1 - beta, rounded from 64 bits
};

template <typename T, int BITS, bool MASTER>
__global__ __launch_bounds__(256) void adamw_kernel(Step a) {
  const kad_adamw_chunk ch = a.chunks[blockIdx.x];
  const kad_adamw_scalars s = a.scalars ? *a.scalars : a.values;
  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  T* __restrict__ p = (T*)ch.param;
  const T* __restrict__ g = (const T*)ch.grad;
  const int lane = threadIdx.x & 63;
  for (int seg = threadIdx.x >> 6; seg * SEG < ch.count; seg += 4) {
    const int i = seg * SEG + lane * 4;
    const int left = ch.count - i;
    const int64_t at = ch.offset + i;
    float gv[4] = {0.f, 0.f, 0.f, 0.f}, pv[4] = {0.f, 0.f, 0.f, 0.f}, m[4], u[4], v[4];
    if (left > 0) {
      load4(g + i, left, gv);
      if (MASTER) load4(a.master + at, 4, pv);  // state buffers are whole segments
      else load4(p + i, left, pv);
    }
    float ms = 1.f, us = 1.f;
    const int64_t row = (ch.offset + (int64_t)seg * SEG) / SEG;
    if (BITS == 8) {
      ms = a.exp_avg_scale[row];
      us = a.exp_avg_sq_scale[row];
      decode4(*(const uint32_t*)((const uint8_t*)a.exp_avg + at), ms, m);
      decode4(*(const uint32_t*)((const uint8_t*)a.exp_avg_sq + at), us, u);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = u[k] * u[k];
    } else {
      load4((const float*)a.exp_avg + at, 4, m);
      load4((const float*)a.exp_avg_sq + at, 4, v);
    }
    {
      // Each product and sum is rounded by itself, as written: a held number depends on which side of a
      // border its value falls, so a program that computes this formula in 32 bits gets the same states, and
      // a parameter is its master rounded (joined with the conversion, the last product would not be).
#pragma clang fp contract(off)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gk = gv[k] * gs;
        m[k] = m[k] * a.beta1 + gk * a.keep1;
        v[k] = v[k] * a.beta2 + (gk * gk) * a.keep2;
        u[k] = sqrtf(v[k]);
        pv[k] = pv[k] * s.decay - (s.rate * m[k]) / (u[k] * s.inv_root + a.eps);
      }
    }
    if (BITS == 8) {
      uint32_t r[4], lo[4], hi[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        r[k] = value_bits(s.key, at + k);
        lo[k] = r[k] & 0xFFFFu;
        hi[k] = r[k] >> 16;
        if (left <= k) m[k] = u[k] = 0.f;  // past the tensor's end: zeros, whatever the buffer held
      }
      const uint32_t mc = encode4<false>(m, lo, ms);
      const uint32_t uc = encode4<true>(u, hi, us);
      *(uint32_t*)((uint8_t*)a.exp_avg + at) = mc;
      *(uint32_t*)((uint8_t*)a.exp_avg_sq + at) = uc;
      if (lane == 0) {
        a.exp_avg_scale[row] = ms;
        a.exp_avg_sq_scale[row] = us;
      }
    } else if (left > 0) {
      store4((float*)a.exp_avg + at, 4, m);
      store4((float*)a.exp_avg_sq + at, 4, v);
    }
    if (left > 0) {
      if (MASTER) store4(a.master + at, 4, pv);
      store4(p + i, left, pv);
    }
  }
}

__host__ __device__ inline kad_adamw_scalars scalars_of(double lr, double beta1, double beta2, double decay,
                                                        uint32_t seed, int64_t step) {
  kad_adamw_scalars s;
  s.decay = (float)(1.0 - lr * decay);
  s.rate = (float)(lr / (1.0 - pow(beta1, (double)step)));
  s.inv_root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  s.key = step_key(seed, step);
  return s;
}

__global__ void adamw_hyper_kernel(const int64_t* step, const float* lr_at, double lr, double beta1, double beta2,
                                   double decay, uint32_t seed, kad_adamw_scalars* out) {
  *out = scalars_of(lr_at ? (double)*lr_at : lr, beta1, beta2, decay, seed, *step);
}

int check_rates(const kad_adamw_args* a, const char* what) {
  KAD_CHECK_ARG(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0,
                "%s: betas must lie in [0, 1)", what);
  KAD_CHECK_ARG(a->eps >= 0.0 && a->weight_decay >= 0.0 && a->lr >= 0.0, "%s: lr, eps and weight_decay must be >= 0",
                what);
  return KAD_OK;
}

template <typename T>
void launch(const kad_adamw_args& a, const Step& s, hipStream_t st) {
  const dim3 grid((unsigned)a.nchunks), block(256);
  if (a.state_bits == 8) {
    if constexpr (sizeof(T) == 2)
      if (a.master) return adamw_kernel<T, 8, true><<<grid, block, 0, st>>>(s);
    adamw_kernel<T, 8, false><<<grid, block, 0, st>>>(s);
  } else {
    if constexpr (sizeof(T) == 2)
      if (a.master) return adamw_kernel<T, 32, true><<<grid, block, 0, st>>>(s);
    adamw_kernel<T, 32, false><<<grid, block, 0, st>>>(s);
  }
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_adamw_chunks(const int64_t* params, const int64_t* grads, const int64_t* numels, int n,
                                    int elem_bytes, kad_adamw_chunk* chunks, int64_t* state_elems) {
  KAD_CHECK_ARG(n >= 0 && (elem_bytes == 2 || elem_bytes == 4), "kad_adamw_chunks: bad count or element size");
  KAD_CHECK_ARG(n == 0 || (params && grads && numels), "kad_adamw_chunks: null pointer");
  int64_t count = 0, at = 0;
  for (int i = 0; i < n; ++i) {
    KAD_CHECK_ARG(numels[i] >= 0 && numels[i] <= ((int64_t)1 << 48), "kad_adamw_chunks: bad number of values");
    for (int64_t k = 0; k < numels[i]; k += CHUNK, ++count) {
      if (!grads[i]) break;
      if (!chunks) continue;
      kad_adamw_chunk& c = chunks[count];
      c.param = (void*)(params[i] + k * elem_bytes);
      c.grad = (const void*)(grads[i] + k * elem_bytes);
      c.offset = at + k;
      c.count = (int)(numels[i] - k < CHUNK ? numels[i] - k : CHUNK);
      c.reserved = 0;
    }
    at += (numels[i] + SEG - 1) / SEG * SEG;
  }
  if (state_elems) *state_elems = at;
  return count;
}

extern "C" int kad_adamw_step(const kad_adamw_args* a, void* stream) {
  KAD_CHECK_ARG(a, "kad_adamw_step: null pointer");
  KAD_CHECK_ARG(a->dtype == KAD_F32 || a->dtype == KAD_F16 || a->dtype == KAD_BF16, "kad_adamw_step: bad dtype");
  KAD_CHECK_ARG(a->state_bits == 32 || a->state_bits == 8, "kad_adamw_step: state_bits must be 32 or 8");
  KAD_CHECK_ARG(a->nchunks >= 0 && a->nchunks < ((int64_t)1 << 31), "kad_adamw_step: too many chunks");
  if (a->nchunks == 0) return KAD_OK;
  KAD_CHECK_ARG(a->chunks && a->exp_avg && a->exp_avg_sq, "kad_adamw_step: null pointer");
  KAD_CHECK_ARG(a->state_bits == 32 || (a->exp_avg_scale && a->exp_avg_sq_scale), "kad_adamw_step: 8-bit states need scales");
  KAD_CHECK_ARG(!a->master || a->dtype != KAD_F32, "kad_adamw_step: masters are for 16-bit parameters");
  KAD_CHECK_ARG(a->scalars || a->step >= 1, "kad_adamw_step: step must be at least 1");
  if (int rc = check_rates(a, "kad_adamw_step")) return rc;
  Step s;
  s.chunks = a->chunks;
  s.exp_avg = a->exp_avg;
  s.exp_avg_sq = a->exp_avg_sq;
  s.exp_avg_scale = a->exp_avg_scale;
  s.exp_avg_sq_scale = a->exp_avg_sq_scale;
  s.master = a->master;
  s.grad_scale = a->grad_scale;
  s.scalars = a->scalars;
  s.values = a->scalars ? kad_adamw_scalars{} : scalars_of(a->lr, a->beta1, a->beta2, a->weight_decay, a->seed, a->step);
  s.beta1 = (float)a->beta1;
  s.beta2 = (float)a->beta2;
  s.keep1 = (float)(1.0 - a->beta1);
  s.keep2 = (float)(1.0 - a->beta2);
  s.eps = (float)a->eps;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) launch<float>(*a, s, st);
  else if (a->dtype == KAD_F16) launch<half_t>(*a, s, st);
  else launch<bf16_t>(*a, s, st);
  return check_launch("kad_adamw_step");
}

extern "C" int kad_adamw_hyper(const kad_adamw_args* a, const int64_t* step, const float* lr,
                               kad_adamw_scalars* scalars, void* stream) {
  KAD_CHECK_ARG(a && step && scalars, "kad_adamw_hyper: null pointer");
  if (int rc = check_rates(a, "kad_adamw_hyper")) return rc;
  adamw_hyper_kernel<<<1, 1, 0, (hipStream_t)stream>>>(step, lr, a->lr, a->beta1, a->beta2, a->weight_decay, a->seed,
                                                      scalars);
  return check_launch("kad_adamw_hyper");
}
