// AdamW over many tensors in one launch, states in 32 or 8 bits.
//
//   m <- b1 m + (1 - b1) g     v <- b2 v + (1 - b2) g^2     p <- decay p - rate m / (sqrt(v) inv_root + eps)
//
// Every value is read and written once, so bytes bound it: 28 a value for fp32 with 32-bit states, 16 with 8-bit
// ones (bf16: 10, where 65 vector operations a value take as long).  What a network of thousands of small tensors costs beside that
// is launches; a table of chunks in device memory makes it one.  A block takes a chunk (at most 4096 values of one
// tensor), a wave 1024 values of it, all of whose loads are on their way at once (blocks that walk over chunks,
// with the next one's entry fetched ahead, take a tenth longer, and a wave a chunk a fifth).
//   64 M values, bf16 with masters, 32 bits: 314 us (5.7 TB/s), 8 bits 214 (4.8); 8 bits, no masters: 124 us (5.2 TB/s);
//   2944 tensors of 7 M values, fp32: 37 us and 27 us; 12 tensors of 150 000: 4.6 us.
// Where parameters may have been written since their last step they are read beside their masters: 335 and 235 us for
// the first two.
// A copy of 1 GiB runs at 5.1 TB/s here.
//
// 8-bit states: 256 values are a segment with one scale.  A lane has 16 of them, so 16 lanes (a row, that DPP
// reduces without LDS) share a segment and its scale's division, and a lane's codes are one load.
// m and u = sqrt(v) are held as e4m3 (a root halves the range of exponents that v would need).
// Rounding is stochastic: in a step v changes by 1e-3 of itself, far under half of an e4m3 step, so rounding
// to nearest would leave it where it is; m likewise stops short of a steady gradient.  A u that is not 0 is
// held as the smallest positive code at least, so that a small m never meets a denominator of eps alone.
#include <math.h>

#include "kad_common.h"

namespace kad {
namespace {

constexpr int SEG = KAD_ADAMW_SEG, CHUNK = KAD_ADAMW_CHUNK;
constexpr int64_t MOST_VALUES = (int64_t)1 << 48;  // of a tensor and of a table: any number of bytes fits 64 bits
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

// Device memory: an address out of a table could be anything's, for which the compiler has slower instructions.
#define KAD_GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ const KAD_GLOBAL T* global(const T* p) { return (const KAD_GLOBAL T*)p; }
template <typename T>
__device__ __forceinline__ KAD_GLOBAL T* global(T* p) { return (KAD_GLOBAL T*)p; }

// 8 and 16 bytes at an address that need only be an element's (the memory unit takes wide accesses at any address).
typedef uint32_t word2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(2)));
template <int BYTES> struct Piece { typedef word4 type; };
template <> struct Piece<8> { typedef word2 type; };

// N values at p, of which the first `left` are there; PAST: past the caches.
template <int N, bool PAST = false, typename T>
__device__ __forceinline__ void load(const T* p, int left, float v[N]) {
  if (left >= N) {
    typedef typename Piece<N * sizeof(T)>::type W;
    constexpr int PER = sizeof(W) / sizeof(T);
#pragma unroll
    for (int j = 0; j < N / PER; ++j) {
      const KAD_GLOBAL W* at = (const KAD_GLOBAL W*)global(p + j * PER);
      const W w = PAST ? __builtin_nontemporal_load(at) : *at;
      T t[PER];
      __builtin_memcpy(t, &w, sizeof(w));
#pragma unroll
      for (int k = 0; k < PER; ++k) v[j * PER + k] = to_f32(t[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k < left ? to_f32((T)global(p)[k]) : 0.f;
  }
}
template <int N, bool PAST = false, typename T>
__device__ __forceinline__ void store(T* p, int left, const float v[N]) {
  if (left >= N) {
    typedef typename Piece<N * sizeof(T)>::type W;
    constexpr int PER = sizeof(W) / sizeof(T);
#pragma unroll
    for (int j = 0; j < N / PER; ++j) {
      T t[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) t[k] = from_f32<T>(v[j * PER + k]);
      W w;
      __builtin_memcpy(&w, t, sizeof(w));
      KAD_GLOBAL W* at = (KAD_GLOBAL W*)global(p + j * PER);
      if (PAST) __builtin_nontemporal_store(w, at);
      else *at = w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < left) global(p)[k] = from_f32<T>(v[k]);
  }
}

__device__ __forceinline__ void decode4(uint32_t codes, float scale, float v[4]) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * scale;
  v[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * scale;
  v[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * scale;
  v[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * scale;
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

// What a step starts from in place of a master m whose parameter p someone else may have written: m while p is m
// rounded, else p.
template <typename T>
__device__ __forceinline__ float followed(float m, float p) { return to_f32(from_f32<T>(m)) == p ? m : p; }

// Where a step's 32-bit parameters come from.
enum Source { PARAM, MASTER, FOLLOW };  // FOLLOW: the master, unless the parameter is another value

constexpr int THREADS = 256;
constexpr int PIECE = 1024;  // values of a chunk that a wave takes at a time

// 32-bit states: a lane takes 4 consecutive values of each of a piece's 4 segments, all on their way at once.
template <typename T, Source FROM, bool PAST>
__global__ __launch_bounds__(THREADS) void adamw32_kernel(Step a) {
  const kad_adamw_chunk ch = a.chunks[blockIdx.x];
  const kad_adamw_scalars s = a.scalars ? *a.scalars : a.values;
  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  T* p = (T*)ch.param;
  const T* g = (const T*)ch.grad;
  float* exp_avg = (float*)a.exp_avg + ch.offset;
  float* exp_avg_sq = (float*)a.exp_avg_sq + ch.offset;
  float* master = a.master + ch.offset;
  constexpr int ROWS = PIECE / SEG;
  for (int first = threadIdx.x / 64 * PIECE; first < ch.count; first += 4 * PIECE) {
    float gv[ROWS][4], pv[ROWS][4], own[ROWS][4], m[ROWS][4], v[ROWS][4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int i = first + r * SEG + (threadIdx.x & 63) * 4, left = ch.count - i;
      if (left <= 0) continue;
      load<4, PAST>(g + i, left, gv[r]);
      if (FROM != PARAM) load<4, PAST>(master + i, 4, pv[r]);  // state buffers are whole segments
      else load<4, PAST>(p + i, left, pv[r]);
      if (FROM == FOLLOW) load<4, PAST>(p + i, left, own[r]);
      load<4, PAST>(exp_avg + i, 4, m[r]);
      load<4, PAST>(exp_avg_sq + i, 4, v[r]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int i = first + r * SEG + (threadIdx.x & 63) * 4, left = ch.count - i;
      if (left <= 0) continue;
      {
        // Each product and sum is rounded by itself, as written: a parameter is its master rounded (joined with
        // the conversion, the last product would not be).
#pragma clang fp contract(off)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (FROM == FOLLOW) pv[r][k] = followed<T>(pv[r][k], own[r][k]);
          const float gk = gv[r][k] * gs;
          m[r][k] = m[r][k] * a.beta1 + gk * a.keep1;
          v[r][k] = v[r][k] * a.beta2 + (gk * gk) * a.keep2;
          pv[r][k] = pv[r][k] * s.decay - (s.rate * m[r][k]) / (sqrtf(v[r][k]) * s.inv_root + a.eps);
        }
      }
      store<4, true>(exp_avg + i, 4, m[r]);
      store<4, true>(exp_avg_sq + i, 4, v[r]);
      if (FROM != PARAM) store<4, true>(master + i, 4, pv[r]);
      store<4, true>(p + i, left, pv[r]);
    }
  }
}

// Largest of a row of 16 lanes, for all of them (DPP: no LDS).
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  const auto step = [&](uint32_t o) { v = o > v ? o : v; };
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));   // lane ^ 2
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));  // half a row mirrored
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));  // the row mirrored
  return v;
}

// A lane's 16 values of a segment as codes, and the segment's scale.  Magnitudes are compared as integers, so that
// infinities and NaN count as largest: a segment that meets one is held as NaN.
// The conversion adds its 32 random bits' upper 20 to the bits that e4m3 has no place for and cuts: a magnitude
// |v| / scale becomes the code above with probability (distance to the code below) / step, whether the codes there
// are normal or not.  The largest may come to 448 (1 + 2^-22): its few low bits and 16 random ones above 4 zeros
// carry into no code.
template <bool POSITIVE>
__device__ __forceinline__ uint4 encode16(const float v[16], const uint32_t r[16], float& scale) {
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint32_t b = __float_as_uint(v[k]) & 0x7FFFFFFFu;
    most = b > most ? b : most;
  }
  most = row_max(most);
  const float top = __uint_as_float(most);
  const bool lost = most >= 0x7F800000u, tiny = top < SEG_TINY;
  scale = lost ? top : tiny ? 0.f : top * (1.0f / E4M3_MAX);
  const float inv = (1.0f / top) * E4M3_MAX;
  uint32_t out[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const auto number = [&](int k) {
      const float y = v[k] * inv;
      return POSITIVE ? __builtin_fmaxf(y, v[k] > 0.f ? 0x1p-9f : 0.f) : y;  // code 1 at least
    };
    int c = 0;
    c = __builtin_amdgcn_cvt_sr_fp8_f32(number(4 * w), r[4 * w], c, 0);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(number(4 * w + 1), r[4 * w + 1], c, 1);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(number(4 * w + 2), r[4 * w + 2], c, 2);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(number(4 * w + 3), r[4 * w + 3], c, 3);
    out[w] = lost ? 0x7F7F7F7Fu : tiny ? 0u : (uint32_t)c;
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// 8-bit states: a lane takes 16 consecutive values, a row of 16 lanes a segment.
template <typename T, Source FROM>
__global__ __launch_bounds__(THREADS) void adamw8_kernel(Step a) {
  const kad_adamw_chunk ch = a.chunks[blockIdx.x];
  const kad_adamw_scalars s = a.scalars ? *a.scalars : a.values;
  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  const int lane = threadIdx.x & 63;
  for (int first = threadIdx.x / 64 * PIECE; first < ch.count; first += 4 * PIECE) {
    const int seg = first + lane / 16 * SEG;
    if (seg >= ch.count) continue;  // whole rows
    const int i = seg + lane % 16 * 16, left = ch.count - i;
    const int64_t pos = ch.offset + i, row = (ch.offset + seg) / SEG;
    uint4* mc = (uint4*)((uint8_t*)a.exp_avg + pos);
    uint4* uc = (uint4*)((uint8_t*)a.exp_avg_sq + pos);
    T* p = (T*)ch.param + i;
    const uint4 mq = *mc, uq = *uc;
    float ms = a.exp_avg_scale[row], us = a.exp_avg_sq_scale[row];
    float gv[16], pv[16], own[16], m[16], u[16];
    load<16>((const T*)ch.grad + i, left, gv);
    if (FROM != PARAM) load<16>(a.master + pos, 16, pv);  // state buffers are whole segments
    else load<16>(p, left, pv);
    if (FROM == FOLLOW) load<16>(p, left, own);
    decode4(mq.x, ms, m);
    decode4(mq.y, ms, m + 4);
    decode4(mq.z, ms, m + 8);
    decode4(mq.w, ms, m + 12);
    decode4(uq.x, us, u);
    decode4(uq.y, us, u + 4);
    decode4(uq.z, us, u + 8);
    decode4(uq.w, us, u + 12);
    {
      // Each product and sum is rounded by itself, as written: a held number depends on which side of a border its
      // value falls, so a program that computes this formula in 32 bits gets the same states, and a parameter is
      // its master rounded.  So is the quotient, where 32 bits of it are kept; a 16-bit parameter alone takes the
      // hardware's reciprocal (off by one step of 32 bits at most, 2^-12 of its own), a third of a division (2944
      // tensors of 7 M fp32 values: 27.2 us by the quotient, 25.8 by the reciprocal).
#pragma clang fp contract(off)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        if (FROM == FOLLOW) pv[k] = followed<T>(pv[k], own[k]);
        const float gk = gv[k] * gs;
        m[k] = m[k] * a.beta1 + gk * a.keep1;
        u[k] = sqrtf((u[k] * u[k]) * a.beta2 + (gk * gk) * a.keep2);
        const float top = s.rate * m[k], below = u[k] * s.inv_root + a.eps;
        pv[k] = pv[k] * s.decay - (FROM == PARAM && sizeof(T) == 2 ? top * __builtin_amdgcn_rcpf(below) : top / below);
      }
    }
    if (left > 0) {
      if (FROM != PARAM) store<16>(a.master + pos, 16, pv);
      store<16>(p, left, pv);
    }
    if (left < 16) {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (left <= k) m[k] = u[k] = 0.f;  // past the tensor's end: zeros, whatever the buffer held
    }
    uint32_t lo[16], hi[16];
    const uint32_t base = (uint32_t)pos * 0x9E3779B1u + (uint32_t)(pos >> 32) * 0x3C6EF373u + s.key;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const uint32_t r = mix32(base + k * 0x9E3779B1u);  // pos is a multiple of 16: its upper half holds for all
      lo[k] = r << 16;
      hi[k] = r & 0xFFFF0000u;
    }
    *mc = encode16<false>(m, lo, ms);
    *uc = encode16<true>(u, hi, us);
    if (lane % 16 == 0) {
      a.exp_avg_scale[row] = ms;
      a.exp_avg_sq_scale[row] = us;
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

template <typename T, Source FROM>
void launch(const kad_adamw_args& a, const Step& s, hipStream_t st) {
  const dim3 grid((unsigned)a.nchunks), block(THREADS);
  if (a.state_bits == 8) adamw8_kernel<T, FROM><<<grid, block, 0, st>>>(s);
  // What one step moves is met by the next, as far as the 256 MB cache before memory holds it; beyond, loads go past it
  // too (fp32: 8 M values 40 us against 43 so, 12 M 68 against 62, 32 M 172 against 159).
  else if (a.values * 28 > (256 << 20)) adamw32_kernel<T, FROM, true><<<grid, block, 0, st>>>(s);
  else adamw32_kernel<T, FROM, false><<<grid, block, 0, st>>>(s);
}
template <typename T>
void launch(const kad_adamw_args& a, const Step& s, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (a.master) return a.follow ? launch<T, FOLLOW>(a, s, st) : launch<T, MASTER>(a, s, st);
  launch<T, PARAM>(a, s, st);
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
    KAD_CHECK_ARG(numels[i] >= 0 && numels[i] <= MOST_VALUES, "kad_adamw_chunks: bad number of values");
    KAD_CHECK_ARG(numels[i] == 0 || !grads[i] || (params[i] && (params[i] | grads[i]) % elem_bytes == 0),
                  "kad_adamw_chunks: addresses must be multiples of the element's size, and params' not 0");
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
    KAD_CHECK_ARG(at <= MOST_VALUES, "kad_adamw_chunks: too many values");
  }
  if (state_elems) *state_elems = at;
  return count;
}

extern "C" int kad_adamw_step(const kad_adamw_args* a, void* stream) {
  KAD_CHECK_ARG(a, "kad_adamw_step: null pointer");
  KAD_CHECK_ARG(a->dtype == KAD_F32 || a->dtype == KAD_F16 || a->dtype == KAD_BF16, "kad_adamw_step: bad dtype");
  KAD_CHECK_ARG(a->state_bits == 32 || a->state_bits == 8, "kad_adamw_step: state_bits must be 32 or 8");
  // a block a chunk, and a grid has fewer than 2^32 threads
  KAD_CHECK_ARG(a->nchunks >= 0 && a->nchunks <= UINT32_MAX / THREADS, "kad_adamw_step: too many chunks");
  if (a->nchunks == 0) return KAD_OK;
  KAD_CHECK_ARG(a->chunks && a->exp_avg && a->exp_avg_sq, "kad_adamw_step: null pointer");
  KAD_CHECK_ARG(a->state_bits == 32 || (a->exp_avg_scale && a->exp_avg_sq_scale), "kad_adamw_step: 8-bit states need scales");
  KAD_CHECK_ARG((((uintptr_t)a->exp_avg | (uintptr_t)a->exp_avg_sq | (uintptr_t)a->master) & 15) == 0,
                "kad_adamw_step: state buffers must begin at multiples of 16 bytes");
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
