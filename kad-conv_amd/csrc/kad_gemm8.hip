// Products of matrices in 8 bits with a scale for each block of 128 (kad_block8.h):
//
//   out[m][n] = act(sum over blocks of 2^(sa + sb - 254) sum over the block of a b + bias[n])
//
// The scales are powers of two, so the scaled matrix instruction takes them as they are: one of 16 x 16 x 128 meets one
// block of each of its rows, and the sums need no arithmetic beside it.  Every 8-bit matrix instruction cuts the products
// of eight consecutive k to 2^-13 of the largest of them (found by giving it single products: 2^3 next to 2^16 is kept,
// 2^2 is not) before it adds them up in 32 bits.  Of normally distributed numbers that is 1.3e-5 of a result, of channels of
// unlike sizes 4e-5, of codes with all bits random 5e-5: under the rounding of a 16-bit result (2.1e-4 in fp16, 1.7e-3 in
// bf16).  For 32-bit results (EXACT) codes become fp16 numbers, which hold them exactly, the fp16 instruction sums a block in
// 32 bits (1e-7), and the scales are applied to its sum.
//
// Three forms.  Many rows: tiles of BM x BN results, both operands' codes copied to LDS past the registers, ahead of their use, in
// two kernels: a stage ahead for tiles of 64 and 128, three for those of 256.
//
// Few rows (KAD_GEMM8_FEW): b's codes are read once, in whole lines that a wave turns into operands by way of its part of LDS;
// a block takes 16 rows of b, its waves take every eighth 128 columns and join in LDS.  a as values is brought to 8 bits in
// registers, by each block for itself: a launch less, and a is small (at 48 rows and [8192, 4096], b from memory, it was not: 48 us
// against 33).
//
// Many rows, short ones: a block brings its rows of values to 8 bits once and keeps them in LDS.
//
// The instruction computes b a^T: a lane then holds four results of one row of out that follow each other.
#include "kad_block8.h"

namespace kad {
namespace {

constexpr int LINE = BLOCK8;        // bytes of a row in a stage: one block of codes
constexpr int KB_GROUP = 4;         // scales are read by fours

// For 16-bit results the hardware's reciprocal alone, off by one step of 32 bits at most.
template <typename T>
__device__ __forceinline__ float activate(float z, int act) {
  if (act == KAD_ACT_SILU) return sizeof(T) == 2 ? z * __builtin_amdgcn_rcpf(1.0f + __expf(-z)) : z * sigmoidf_(z);
  return act == KAD_ACT_RELU ? (z > 0.f ? z : z != z ? z : 0.f) : z;
}

template <bool EXACT> struct Operand;
template <> struct Operand<false> {
  intx8 v;
  __device__ __forceinline__ void set(intx4 lo, intx4 hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
  }
};
template <> struct Operand<true> {
  half8_t v[4];
  __device__ __forceinline__ void set(intx4 lo, intx4 hi) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int w = q < 2 ? lo[2 * q + i] : hi[2 * (q - 2) + i];
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
        v[q][4 * i] = a[0];
        v[q][4 * i + 1] = a[1];
        v[q][4 * i + 2] = b[0];
        v[q][4 * i + 3] = b[1];
      }
    }
  }
};

// acc += a block of b's 16 rows times one of a's 16, of whose scales byte Q of sb and sa is this block's.  EXACT: eb are
// the scales of the four rows of b whose results the lane holds.
template <int Q>
__device__ __forceinline__ void multiply(floatx4& acc, const Operand<false>& b, const Operand<false>& a, int sb, int sa, const int*) {
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, acc, 0, 0, Q, sb, Q, sa);
}
template <int Q>
__device__ __forceinline__ void multiply(floatx4& acc, const Operand<true>& b, const Operand<true>& a, int, int sa, const int* eb) {
  floatx4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.v[q], a.v[q], t, 0, 0, 0);
  const int ea = ((sa >> (8 * Q)) & 255) - 254;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] += __builtin_amdgcn_ldexpf(t[i], ea + eb[i]);
}

template <typename T>
__device__ __forceinline__ void store_four(T* p, const float* v, int n) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(v[i]);
  if (n >= 4) {
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = t[i];
  }
}

template <typename T>
__device__ __forceinline__ float bias_at(const kad_gemm8_args& a, int n) {
  return a.bias && n < a.n ? load_param(a.bias, n, a.bias_dtype, 0.f) : 0.f;
}

// Four results of row m from column n on.
template <typename T>
__device__ __forceinline__ void finish(const kad_gemm8_args& a, int m, int n, const floatx4& acc) {
  if (m >= a.m || n >= a.n) return;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = activate<T>(acc[i] + bias_at<T>(a, n + i), a.act);
  store_four<T>((T*)a.out + (int64_t)m * a.n + n, v, a.n - n);
}

// ---------------------------------------------------------------------------- many rows
struct Tiles {
  int tm, tn;      // tiles of rows and columns
  int splits, per; // parts of k, and the 128s of k in each (a multiple of KB_GROUP)
};

// Blocks go to the eight XCDs in turn: each gets a run of tiles, which walks the rows of a few columns' worth of tiles, so
// that what shares an L2 shares operands.
__device__ __forceinline__ bool tile_of(const Tiles& o, int& m, int& n, int& split) {
  constexpr int XCDS = 8, GROUP = 8;
  const int total = o.tm * o.tn * o.splits, run = (total + XCDS - 1) / XCDS;
  int id = (int)(blockIdx.x % XCDS) * run + (int)(blockIdx.x / XCDS);
  if (id >= total || (int)(blockIdx.x / XCDS) >= run) return false;
  split = id / (o.tm * o.tn);
  id -= split * (o.tm * o.tn);
  const int first = id / (GROUP * o.tm) * GROUP, wide = o.tn - first < GROUP ? o.tn - first : GROUP;
  id -= first * o.tm;
  m = id / wide;
  n = first + id - m * wide;
  return true;
}

// A wave's 16-bit results: two rows of fragments at a time by way of its part of LDS, so that whole lines are written, and past
// the caches that hold the operands ([40000, 512] x [512, 512] fp16: 19.7 us, 22.4 through them; of tiles of 256, whose products
// take long, it makes no difference).
constexpr int store_bytes(int tn) { return 32 * (tn * 32 + 16); }
template <typename T, int TM, int TN, int ACT>
__device__ __forceinline__ void store_tile(const kad_gemm8_args& a, const floatx4 (&acc)[TM][TN], const float (&bias)[TN][4], char* lds,
                                           int lane, int m1, int n1) {
  constexpr int PITCH = TN * 32 + 16, PIECES = TN * 2, ROWS = 64 / PIECES;
  const int r16 = lane & 15, g = lane >> 4, piece = lane % PIECES, row = lane / PIECES;
  const int n = n1 + piece * 8, left = a.n - n;
#pragma unroll
  for (int i = 0; i < TM; i += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        T t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = from_f32<T>(activate<T>(acc[i + h][j][e] + bias[j][e], ACT));
        __builtin_memcpy(lds + (h * 16 + r16) * PITCH + (j * 16 + 4 * g) * 2, t, 8);
      }
    wave_order();
    intx4 v[32 / ROWS];
#pragma unroll
    for (int r = 0; r < 32 / ROWS; ++r) v[r] = *(const intx4*)(lds + (r * ROWS + row) * PITCH + piece * 16);
    wave_order();
#pragma unroll
    for (int r = 0; r < 32 / ROWS; ++r) {
      const int m = m1 + i * 16 + r * ROWS + row;
      if (m >= a.m || left <= 0) continue;
      T* to = (T*)a.out + (int64_t)m * a.n + n;
      if (left >= 8) {
        __builtin_nontemporal_store(v[r], (loose<T>*)to);
      } else {
        T t[8];
        __builtin_memcpy(t, &v[r], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) to[e] = t[e];
      }
    }
  }
}

template <typename T, int BM, int BN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void gemm8_tile_kernel(kad_gemm8_args a, Tiles o) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES;  // copies of a wave and stage: 8 rows each
  static_assert(WAVES % 2 == 0, "a wave's copies begin at rows 8 (wave & 1) of 16");
  __shared__ __attribute__((aligned(128))) char s0[(BM + BN) * LINE];
  __shared__ __attribute__((aligned(128))) char s1[(BM + BN) * LINE];
  int m0, n0, split;
  if (!tile_of(o, m0, n0, split)) return;
  m0 *= BM;
  n0 *= BN;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.k + BLOCK8 - 1) / BLOCK8, kp = blocks * BLOCK8, ks = (blocks + 3) / 4 * 4;
  const int begin = split * o.per, end = begin + o.per < blocks ? begin + o.per : blocks;
  // rows past the last read as zeros
  const int rows_a = a.m - m0 < BM ? a.m - m0 : BM, rows_b = a.n - n0 < BN ? a.n - n0 : BN;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc((const char*)a.a + (int64_t)m0 * kp, rows_a * kp);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc((const char*)a.b + (int64_t)n0 * kp, rows_b * kp);
  // 16-byte piece p of row r lies at piece p ^ (r / 2 & 7) of its line: lanes that read one piece of 16 rows meet all 64 banks
  const uint32_t off = (uint32_t)(lane >> 3) * kp + (((lane & 7) ^ ((wave & 1) << 2 | lane >> 4)) << 4);
  const auto stage = [&](char* s, int kb) {
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      const int r = (i * WAVES + wave) * 8;
      dma16(ra, s + r * LINE, off + (uint32_t)r * kp, kb * BLOCK8);
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) {
      const int r = (i * WAVES + wave) * 8;
      dma16(rb, s + (BM + r) * LINE, off + (uint32_t)r * kp, kb * BLOCK8);
    }
  };
  const int wm = wave / WN, wn = wave % WN, r16 = lane & 15, g = lane >> 4;
  const int line_a = (wm * TM * 16 + r16) * LINE, line_b = (BM + wn * TN * 16 + r16) * LINE;
  const int piece0 = ((2 * g) ^ (r16 >> 1)) << 4, piece1 = ((2 * g + 1) ^ (r16 >> 1)) << 4;
  const auto fetch = [&](const char* s, int line, int frag, Operand<EXACT>& v) {
    const char* p = s + line + frag * 16 * LINE;
    v.set(*(const intx4*)(p + piece0), *(const intx4*)(p + piece1));
  };
  // scales of the lane's rows, four blocks of k in each, a group ahead; past the last row 0, for codes of 0
  const __amdgpu_buffer_rsrc_t rsa = make_rsrc((const char*)a.a_scales + (int64_t)m0 * ks, rows_a * ks);
  const __amdgpu_buffer_rsrc_t rsb = make_rsrc((const char*)a.b_scales + (int64_t)n0 * ks, rows_b * ks);
  const uint32_t off_sa = (uint32_t)(wm * TM * 16 + r16) * ks, off_sb = (uint32_t)(wn * TN * 16 + r16) * ks;
  int scale_a[TM], scale_b[TN], next_a[TM], next_b[TN];
  const auto scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < TM; ++i) next_a[i] = __builtin_amdgcn_raw_buffer_load_b32(rsa, off_sa + (uint32_t)(i * 16 * ks), kb, 0);
#pragma unroll
    for (int i = 0; i < TN; ++i) next_b[i] = __builtin_amdgcn_raw_buffer_load_b32(rsb, off_sb + (uint32_t)(i * 16 * ks), kb, 0);
  };
  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  scales(begin);
  stage(s0, begin);
  // a's operands one ahead of the instructions that they feed
#define KAD_STEP(Q, NOW, NEXT)                                                           \
  if (kb + Q < end) {                                                                    \
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");             \
    if (Q == 0) {                                                                        \
      _Pragma("unroll") for (int i = 0; i < TM; ++i) scale_a[i] = next_a[i];             \
      _Pragma("unroll") for (int i = 0; i < TN; ++i) scale_b[i] = next_b[i];             \
    }                                                                                    \
    if (kb + Q + 1 < end) stage(NEXT, kb + Q + 1);                                       \
    if (Q == 0 && kb + KB_GROUP < end) scales(kb + KB_GROUP);                            \
    Operand<EXACT> fb[TN], fa[2];                                                        \
    int eb[TN][4];                                                                       \
    fetch(NOW, line_a, 0, fa[0]);                                                        \
    _Pragma("unroll") for (int j = 0; j < TN; ++j) {                                     \
      fetch(NOW, line_b, j, fb[j]);                                                      \
      if (EXACT) {                                                                       \
        const int e = (scale_b[j] >> (8 * Q)) & 255;                                     \
        _Pragma("unroll") for (int i = 0; i < 4; ++i) eb[j][i] = __shfl(e, 4 * g + i);   \
      }                                                                                  \
    }                                                                                    \
    _Pragma("unroll") for (int i = 0; i < TM; ++i) {                                     \
      if (i + 1 < TM) fetch(NOW, line_a, i + 1, fa[(i + 1) & 1]);                        \
      _Pragma("unroll") for (int j = 0; j < TN; ++j)                                     \
        multiply<Q>(acc[i][j], fb[j], fa[i & 1], scale_b[j], scale_a[i], eb[j]);         \
    }                                                                                    \
    if (!EXACT) {                                                                        \
      __builtin_amdgcn_sched_group_barrier(0x100, 2 + 2 * TN, 0);                        \
      _Pragma("unroll") for (int i = 0; i < TM; ++i) {                                   \
        if (i + 1 < TM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);               \
        __builtin_amdgcn_sched_group_barrier(0x008, TN, 0);                              \
      }                                                                                  \
    }                                                                                    \
  }
  for (int kb = begin; kb < end; kb += KB_GROUP) {
    KAD_STEP(0, s0, s1)
    KAD_STEP(1, s1, s0)
    KAD_STEP(2, s0, s1)
    KAD_STEP(3, s1, s0)
  }
#undef KAD_STEP
  const int m1 = m0 + wm * TM * 16, n1 = n0 + wn * TN * 16;
  if (o.splits > 1) {  // 32-bit sums that are joined later
    float* part = a.work + (int64_t)split * a.m * a.n;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int m = m1 + i * 16 + r16, n = n1 + j * 16 + 4 * g;
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        if (m < a.m && n < a.n) store_four<float>(part + (int64_t)m * a.n + n, v, a.n - n);
      }
    return;
  }
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) finish<T>(a, m1 + i * 16 + r16, n1 + j * 16 + 4 * g, acc[i][j]);
  } else {
    float bias[TN][4];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) bias[j][i] = bias_at<T>(a, n1 + j * 16 + 4 * g + i);
    __syncthreads();
    if (a.act == KAD_ACT_SILU) store_tile<T, TM, TN, KAD_ACT_SILU>(a, acc, bias, s0 + wave * store_bytes(TN), lane, m1, n1);
    else if (a.act == KAD_ACT_RELU) store_tile<T, TM, TN, KAD_ACT_RELU>(a, acc, bias, s0 + wave * store_bytes(TN), lane, m1, n1);
    else store_tile<T, TM, TN, KAD_ACT_NONE>(a, acc, bias, s0 + wave * store_bytes(TN), lane, m1, n1);
  }
}

// Tiles of 256 x 256 results for 16-bit results: 8 waves of 128 x 64, the 32 x 32 x 64 instruction, and a ring of four stages
// of 64 columns, so that three are on their way while one is used: with two stages of 128 the copies' latency was the step's
// time (4900 cycles, of which the instructions take 2048).
//
// The copies are written as assembly: of ones that it knows the compiler waits for more than a step needs before it reads
// LDS (it does not tell all stages apart), which ends the run ahead.  They write no register but m0, which they
// name, and every wait for them is one of KAD_STEP's.  Scales go the same way, two groups of four blocks in turn.
typedef float floatx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint32_t lds_address(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
__device__ __forceinline__ intx4 resource(const void* base, uint32_t bytes) {
  const uint64_t at = (uint64_t)base;
  return intx4{__builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)(at >> 32 & 0xFFFF)),
               __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// 16 or 4 bytes a lane from byte off + at of the resource to LDS, the lanes' one after the other; nothing is known to be
// there before a wait for vmcnt.
__device__ __forceinline__ void copy16(intx4 r, uint32_t lds, uint32_t off, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(r), "s"(at)
               : "m0", "memory");
}
__device__ __forceinline__ void copy4(intx4 r, uint32_t lds, uint32_t off, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(r), "s"(at)
               : "m0", "memory");
}

constexpr int WIDE = 256, HALF = 64;  // rows of a tile, bytes of a row in a stage

template <typename T, int ACT>
__device__ __forceinline__ void store_wide(const kad_gemm8_args& a, const floatx16 (&acc)[4][2], const float (&bias)[2][16], char* lds,
                                           int lane, int m1, int n1) {
  constexpr int PITCH = 64 * 2 + 16;
  const int r32 = lane & 31, h = lane >> 5, piece = lane & 7, row = lane >> 3;
  const int n = n1 + piece * 8, left = a.n - n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        T t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = from_f32<T>(activate<T>(acc[i][j][4 * q + e] + bias[j][4 * q + e], ACT));
        __builtin_memcpy(lds + r32 * PITCH + (j * 32 + 8 * q + 4 * h) * 2, t, 8);
      }
    wave_order();
    intx4 v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = *(const intx4*)(lds + (r * 8 + row) * PITCH + piece * 16);
    wave_order();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m1 + i * 32 + r * 8 + row;
      if (m >= a.m || left <= 0) continue;
      T* to = (T*)a.out + (int64_t)m * a.n + n;
      if (left >= 8) {
        __builtin_memcpy(to, &v[r], 16);
      } else {
        T t[8];
        __builtin_memcpy(t, &v[r], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) to[e] = t[e];
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(512) void gemm8_wide_kernel(kad_gemm8_args a, Tiles o) {
  __shared__ __attribute__((aligned(128))) char s0[2 * WIDE * HALF];
  __shared__ __attribute__((aligned(128))) char s1[2 * WIDE * HALF];
  __shared__ __attribute__((aligned(128))) char s2[2 * WIDE * HALF];
  __shared__ __attribute__((aligned(128))) char s3[2 * WIDE * HALF];
  __shared__ __attribute__((aligned(128))) char c0[2 * WIDE * 4], c1[2 * WIDE * 4];
  int m0, n0, split;
  if (!tile_of(o, m0, n0, split)) return;
  m0 *= WIDE;
  n0 *= WIDE;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.k + BLOCK8 - 1) / BLOCK8, kp = blocks * BLOCK8, ks = (blocks + 3) / 4 * 4;
  const int begin = split * o.per, end = begin + o.per < blocks ? begin + o.per : blocks, steps = 2 * (end - begin);
  // rows past the last read as zeros
  const int rows_a = a.m - m0 < WIDE ? a.m - m0 : WIDE, rows_b = a.n - n0 < WIDE ? a.n - n0 : WIDE;
  const intx4 ra = resource((const char*)a.a + (int64_t)m0 * kp, rows_a * kp), rb = resource((const char*)a.b + (int64_t)n0 * kp, rows_b * kp);
  // 16-byte piece p of row r lies at piece p ^ (r / 2 & 3) of its 64 bytes: lanes that read one piece of 8 rows meet 32 banks
  const uint32_t off = (uint32_t)(lane >> 2) * kp + (((lane & 3) ^ (lane >> 3 & 3)) << 4);
  const auto stage = [&](const char* s, int step) {
    const uint32_t at = begin * BLOCK8 + step * HALF, to = lds_address(s);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (i * 8 + wave) * 16;
      copy16(ra, to + r * HALF, off + (uint32_t)r * kp, at);
      copy16(rb, to + (WIDE + r) * HALF, off + (uint32_t)r * kp, at);
    }
  };
  const int wm = wave >> 2, wn = wave & 3, r32 = lane & 31, h = lane >> 5;
  const int line_a = (wm * 128 + r32) * HALF, line_b = (WIDE + wn * 64 + r32) * HALF;
  const int piece0 = ((2 * h) ^ (r32 >> 1 & 3)) << 4, piece1 = ((2 * h + 1) ^ (r32 >> 1 & 3)) << 4;
  const auto fetch = [&](const char* s, int line, int frag, intx8& v) {
    const char* p = s + line + frag * 32 * HALF;
    const intx4 lo = *(const intx4*)(p + piece0), hi = *(const intx4*)(p + piece1);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
  };
  // scales of 64 rows of a (the first four waves) or b, four blocks of k in each; past the last row 0, for codes of 0
  const intx4 rs = wave < 4 ? resource((const char*)a.a_scales + (int64_t)m0 * ks, rows_a * ks)
                            : resource((const char*)a.b_scales + (int64_t)n0 * ks, rows_b * ks);
  const auto scales = [&](const char* s, int kb) {
    copy4(rs, lds_address(s) + wave * 256, (uint32_t)((wave & 3) * 64 + lane) * ks, kb < ks - 4 ? kb : ks - 4);
  };
  int scale_a[4], scale_b[2];
  floatx16 acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  scales(c0, begin);
  stage(s0, 0);
  stage(s1, 1);
  if (2 < steps) stage(s2, 2);
  // Step s uses what was copied three steps ago: of the wave's own copies, those of the two stages after it (4 each) may be
  // under way, and in two steps the one of scales between them.
#define KAD_STEP(H, NOW, LATER)                                                                              \
  if (base + H < steps) {                                                                                    \
    if (base + H + 2 < steps) {                                                                              \
      if (H % 8 == 5 || H % 8 == 6) asm volatile("s_waitcnt vmcnt(9) lgkmcnt(0)\n\ts_barrier" ::: "memory"); \
      else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");                          \
    } else {                                                                                                 \
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");                               \
    }                                                                                                        \
    if (H % 8 == 4) scales(H < 8 ? c1 : c0, begin + (base + H + 4) / 2);                                     \
    if (base + H + 3 < steps) stage(LATER, base + H + 3);                                                    \
    if (H % 8 == 0) {                                                                                        \
      const int* c = (const int*)(H < 8 ? c0 : c1);                                                          \
      _Pragma("unroll") for (int i = 0; i < 4; ++i) scale_a[i] = c[wm * 128 + i * 32 + r32];                 \
      _Pragma("unroll") for (int i = 0; i < 2; ++i) scale_b[i] = c[WIDE + wn * 64 + i * 32 + r32];           \
    }                                                                                                        \
    intx8 fa[4], fb[2];                                                                                      \
    _Pragma("unroll") for (int j = 0; j < 2; ++j) fetch(NOW, line_b, j, fb[j]);                              \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) fetch(NOW, line_a, i, fa[i]);                              \
    _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                            \
      _Pragma("unroll") for (int j = 0; j < 2; ++j)                                                          \
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], acc[i][j], 0, 0, H % 8 / 2, scale_b[j], H % 8 / 2, scale_a[i]); \
    __builtin_amdgcn_sched_group_barrier(0x100, H % 8 == 0 ? 14 : 8, 0);                                     \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                          \
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);                                                     \
      if (i < 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);                                          \
    }                                                                                                        \
  }
  for (int base = 0; base < steps; base += 16) {
    KAD_STEP(0, s0, s3)
    KAD_STEP(1, s1, s0)
    KAD_STEP(2, s2, s1)
    KAD_STEP(3, s3, s2)
    KAD_STEP(4, s0, s3)
    KAD_STEP(5, s1, s0)
    KAD_STEP(6, s2, s1)
    KAD_STEP(7, s3, s2)
    KAD_STEP(8, s0, s3)
    KAD_STEP(9, s1, s0)
    KAD_STEP(10, s2, s1)
    KAD_STEP(11, s3, s2)
    KAD_STEP(12, s0, s3)
    KAD_STEP(13, s1, s0)
    KAD_STEP(14, s2, s1)
    KAD_STEP(15, s3, s2)
  }
#undef KAD_STEP
  const int m1 = m0 + wm * 128, n1 = n0 + wn * 64;
  if (o.splits > 1) {  // 32-bit sums that are joined later
    float* part = a.work + (int64_t)split * a.m * a.n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = m1 + i * 32 + r32, n = n1 + j * 32 + 8 * q + 4 * h;
          const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          if (m < a.m && n < a.n) store_four<float>(part + (int64_t)m * a.n + n, v, a.n - n);
        }
    return;
  }
  float bias[2][16];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[j][4 * q + e] = bias_at<T>(a, n1 + j * 32 + 8 * q + 4 * h + e);
  __syncthreads();
  char* lds = (wave < 4 ? s0 : s1) + (wave & 3) * (32 * 144);
  if (a.act == KAD_ACT_SILU) store_wide<T, KAD_ACT_SILU>(a, acc, bias, lds, lane, m1, n1);
  else if (a.act == KAD_ACT_RELU) store_wide<T, KAD_ACT_RELU>(a, acc, bias, lds, lane, m1, n1);
  else store_wide<T, KAD_ACT_NONE>(a, acc, bias, lds, lane, m1, n1);
}

// The parts of k, in order.
template <typename T>
__global__ __launch_bounds__(256) void gemm8_join_kernel(kad_gemm8_args a, int splits) {
  const int64_t all = (int64_t)a.m * a.n, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
    float s = a.work[i];
#pragma unroll 4
    for (int p = 1; p < splits; ++p) s += a.work[p * all + i];
    if (a.bias) s += load_param(a.bias, (int)(i % a.n), a.bias_dtype, 0.f);
    ((T*)a.out)[i] = from_f32<T>(activate<T>(s, a.act));
  }
}

// ---------------------------------------------------------------------------- few rows
constexpr int FEW_WAVES = 8;

// A lane's 32 numbers of a block: 8-bit ones, or values in registers until they are brought to 8 bits.  Rows past the last
// read the last one's: what comes of them is not stored.
template <typename X> struct Numbers {
  static constexpr int V = VEC<X>;
  intx4 raw[32 / V];
  static __device__ __forceinline__ int whole(const kad_gemm8_args& a) { return a.k / BLOCK8; }  // blocks without an end of k
  __device__ __forceinline__ void load(const kad_gemm8_args& a, int64_t, int64_t, int row, int kb, int g) {
    const X* p = (const X*)a.a + row * a.a_rs + kb * BLOCK8 + 32 * g;
#pragma unroll
    for (int i = 0; i < 32 / V; ++i) raw[i] = load_vec(p + i * V);
  }
  // Of the block where k ends: zeros behind.
  __device__ __forceinline__ void load_end(const kad_gemm8_args& a, int row, int kb, int g) {
    const X* p = (const X*)a.a + row * a.a_rs;
    X v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int at = kb * BLOCK8 + 32 * g + i;
      v[i] = p[at < a.k ? at : a.k - 1];
      if (at >= a.k) v[i] = (X)0.f;
    }
    __builtin_memcpy(raw, v, sizeof(v));
  }
  // Their codes, and their block's scale: the four lanes of a row hold a block.
  __device__ __forceinline__ int codes(intx4& lo, intx4& hi) const {
    constexpr int WORDS = 32 * sizeof(X) / 4;
    uint32_t w[WORDS];
    __builtin_memcpy(w, raw, sizeof(w));
    uint32_t m = largest_finite<X, WORDS>(w), other = __shfl_xor(m, 16);
    m = m > other ? m : other;
    other = __shfl_xor(m, 32);
    m = m > other ? m : other;
    const int s = scale_of<X>(m);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(X) == 2) {
        lo[i] = codes_of<X>(w[2 * i], w[2 * i + 1], s);
        hi[i] = codes_of<X>(w[8 + 2 * i], w[9 + 2 * i], s);
      } else {
        lo[i] = codes_of(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3], s);
        hi[i] = codes_of(w[16 + 4 * i], w[17 + 4 * i], w[18 + 4 * i], w[19 + 4 * i], s);
      }
    }
    return s;
  }
};
template <> struct Numbers<unsigned char> {
  intx4 lo, hi;
  int scale;
  static __device__ __forceinline__ int whole(const kad_gemm8_args& a) { return (a.k + BLOCK8 - 1) / BLOCK8; }
  __device__ __forceinline__ void load(const kad_gemm8_args& a, int64_t kp, int64_t ks, int row, int kb, int g) {
    const intx4* p = (const intx4*)((const char*)a.a + row * kp + kb * BLOCK8 + 32 * g);
    lo = p[0];
    hi = p[1];
    scale = ((const unsigned char*)a.a_scales)[row * ks + kb];
  }
  __device__ __forceinline__ void load_end(const kad_gemm8_args&, int, int, int) {}
  __device__ __forceinline__ int codes(intx4& l, intx4& h) const {
    l = lo;
    h = hi;
    return scale;
  }
};

// X: a's type as values, or unsigned char: a in 8 bits.  A wave has the loads of AT_ONCE blocks under way: they are made for
// the last block again where there are fewer, since the compiler waits for all loads where branches around some meet
// ([1, 4096] x [8192, 4096] bf16, weights from memory: 17.6 us with such branches, 12.7 without; 11.4 with b in whole lines, of
// which 3 are a's way into 8 bits: 8.2 where it is there already).
template <typename T, typename X, int MT, bool EXACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void gemm8_few_kernel(kad_gemm8_args a) {
  constexpr int AT_ONCE = 4 / MT;
  __shared__ floatx4 red[FEW_WAVES][MT][64];
  __shared__ __attribute__((aligned(128))) char lines[FEW_WAVES][16 * LINE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, row_b = n0 + r16 < a.n ? n0 + r16 : a.n - 1;
  const int blocks = (a.k + BLOCK8 - 1) / BLOCK8, whole = Numbers<X>::whole(a);
  const int64_t kp = (int64_t)blocks * BLOCK8, ks = (blocks + 3) / 4 * 4;
  // eight rows' lines at a time
  const int line = n0 + (lane >> 3);
  const char* codes_b[2] = {(const char*)a.b + (line < a.n ? line : a.n - 1) * kp + (lane & 7) * 16,
                            (const char*)a.b + (line + 8 < a.n ? line + 8 : a.n - 1) * kp + (lane & 7) * 16};
  char* mine = lines[wave];
  const int to = (lane >> 3) * LINE + (((lane & 7) ^ (lane >> 4)) << 4);
  const int to8 = (8 + (lane >> 3)) * LINE + (((lane & 7) ^ (4 + (lane >> 4))) << 4);
  const int piece0 = r16 * LINE + (((2 * g) ^ (r16 >> 1)) << 4), piece1 = r16 * LINE + (((2 * g + 1) ^ (r16 >> 1)) << 4);
  const unsigned char* scales_b = (const unsigned char*)a.b_scales + row_b * ks;
  int row[MT];
  floatx4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    row[i] = i * 16 + r16 < a.m ? i * 16 + r16 : a.m - 1;
    acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const auto add = [&](intx4 lo, intx4 hi, int sb, const Numbers<X> (&x)[MT]) {
    Operand<EXACT> fb, fa;
    wave_order();
    *(intx4*)(mine + to) = lo;
    *(intx4*)(mine + to8) = hi;
    wave_order();
    fb.set(*(const intx4*)(mine + piece0), *(const intx4*)(mine + piece1));
    int eb[4];
    if (EXACT)
#pragma unroll
      for (int i = 0; i < 4; ++i) eb[i] = __shfl(sb, 4 * g + i);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      intx4 l, h;
      const int s = x[i].codes(l, h);
      fa.set(l, h);
      multiply<0>(acc[i], fb, fa, sb, s, eb);
    }
  };
  for (int first = wave; first < whole; first += AT_ONCE * FEW_WAVES) {
    intx4 lo[AT_ONCE], hi[AT_ONCE];
    int sb[AT_ONCE];
    Numbers<X> x[AT_ONCE][MT];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int kb = first + u * FEW_WAVES < whole ? first + u * FEW_WAVES : whole - 1;
      lo[u] = *(const intx4*)(codes_b[0] + kb * BLOCK8);
      hi[u] = *(const intx4*)(codes_b[1] + kb * BLOCK8);
      sb[u] = scales_b[kb];
#pragma unroll
      for (int i = 0; i < MT; ++i) x[u][i].load(a, kp, ks, row[i], kb, g);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (first + u * FEW_WAVES < whole) add(lo[u], hi[u], sb[u], x[u]);
  }
  if (whole < blocks && wave == whole % FEW_WAVES) {
    Numbers<X> x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i].load_end(a, row[i], whole, g);
    add(*(const intx4*)(codes_b[0] + whole * BLOCK8), *(const intx4*)(codes_b[1] + whole * BLOCK8), scales_b[whole], x);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MT; i += FEW_WAVES) {
    floatx4 s = red[0][i][lane];
    const int waves = blocks < FEW_WAVES ? blocks : FEW_WAVES;
    for (int w = 1; w < waves; ++w) s += red[w][i][lane];
    finish<T>(a, i * 16 + r16, n0 + 4 * g, s);
  }
}

// ---------------------------------------------------------------------------- many short rows
// a as values of the result's type: a block brings 64 rows to 8 bits, keeps their codes in LDS, and meets them with all of
// b's rows, or a part.  So a is read once, and its codes take no way through memory.  A wave reads b's codes in whole lines, the
// next block's while it multiplies, and turns them into operands by way of its own part of LDS: read as operands, 16 bytes a
// lane and one row a lane, they came at a quarter of the rate.
constexpr int SHORT_ROWS = 64, SHORT_MOST = 512;  // rows of a block, their values
constexpr int short_bytes(int tn) { return tn * 16 * LINE; }
static_assert(short_bytes(2) >= store_bytes(2) && short_bytes(4) >= store_bytes(4), "results take the place of codes");

template <typename T, int WM, int TN>
__global__ __launch_bounds__(256) void gemm8_short_kernel(kad_gemm8_args a, int columns) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int WN = 4 / WM, TM = 4 / WM, V = VEC<T>, L = LANES<T>, PER = 64 / L, GROUPS = 16 / PER;
  extern __shared__ __attribute__((aligned(128))) char lds[];  // codes [blocks][64][128], scales [64][ks], the waves' results
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), m0 = blockIdx.x * SHORT_ROWS;
  const int whole = a.k / BLOCK8, blocks = (a.k + BLOCK8 - 1) / BLOCK8, ks = (blocks + 3) / 4 * 4;
  const int64_t kp = (int64_t)blocks * BLOCK8;
  unsigned char* scales = (unsigned char*)lds + blocks * SHORT_ROWS * LINE;
  char* mine = (char*)scales + SHORT_ROWS * ks + (t >> 6) * short_bytes(TN);  // of the wave: b's codes, then results
  {
    const int l = lane % L, sub = lane / L;
    const T* p[GROUPS];
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      const int m = m0 + wave * 16 + q * PER + sub;  // rows past the last read the last one: what comes of them is not stored
      p[q] = (const T*)a.a + (m < a.m ? m : a.m - 1) * a.a_rs;
    }
    const auto put_codes = [&](int q, int kb, const uint32_t* w) {
      const int r = wave * 16 + q * PER + sub, s = scale_of<T>(lanes_largest<L>(largest_finite<T, 4>(w)));
      char* to = lds + (kb * SHORT_ROWS + r) * LINE;
      if constexpr (sizeof(T) == 2) {
        int* two = (int*)(to + (((l >> 1) ^ (r >> 1 & 7)) << 4) + (l & 1) * 8);
        two[0] = codes_of<T>(w[0], w[1], s);
        two[1] = codes_of<T>(w[2], w[3], s);
      } else {
        *(int*)(to + (((l >> 2) ^ (r >> 1 & 7)) << 4) + (l & 3) * 4) = codes_of(w[0], w[1], w[2], w[3], s);
      }
      if (l == 0) scales[r * ks + kb] = (unsigned char)s;
    };
    if (whole) {
      intx4 next[GROUPS];
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) next[q] = load_vec(p[q] + l * V);
      for (int kb = 0; kb < whole; ++kb) {
        uint32_t w[GROUPS][4];
        const int then = kb + 1 < whole ? kb + 1 : kb;
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
          __builtin_memcpy(w[q], &next[q], 16);
          next[q] = load_vec(p[q] + then * BLOCK8 + l * V);
        }
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) put_codes(q, kb, w[q]);
      }
    }
    if (whole < blocks) {
      const int left = a.k - whole * BLOCK8 - l * V, n = left > 0 ? left : 0;
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        float v[V];
        uint32_t w[4];
        load_some(p[q] + (n ? whole * BLOCK8 + l * V : 0), n, v);
        const intx4 raw = pack<T>(v);
        __builtin_memcpy(w, &raw, 16);
        put_codes(q, whole, w);
      }
    }
  }
  __syncthreads();
  const int wm = wave / WN, wn = wave % WN, r16 = lane & 15, g = lane >> 4;
  const int line = (wm * TM * 16 + r16) * LINE, piece0 = ((2 * g) ^ (r16 >> 1)) << 4, piece1 = ((2 * g + 1) ^ (r16 >> 1)) << 4;
  constexpr int STRIP = TN * 16;
  const int first = blockIdx.y * columns, last = first + columns < a.n ? first + columns : a.n;
  intx4 raw[2 * TN];
  int sb[TN];
  const auto fetch = [&](int n1, int kb) {
#pragma unroll
    for (int i = 0; i < 2 * TN; ++i) {
      const int at = n1 + i * 8 + (lane >> 3), row = at < a.n ? at : a.n - 1;
      raw[i] = *(const intx4*)((const char*)a.b + row * kp + kb * BLOCK8 + (lane & 7) * 16);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int at = n1 + j * 16 + r16, row = at < a.n ? at : a.n - 1;
      sb[j] = ((const unsigned char*)a.b_scales)[(int64_t)row * ks + kb];
    }
  };
  int n1 = first + wn * STRIP;
  if (n1 >= last) return;
  fetch(n1, 0);
  for (; n1 < last; n1 += WN * STRIP) {
    float bias[TN][4];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) bias[j][i] = bias_at<T>(a, n1 + j * 16 + 4 * g + i);
    floatx4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int kb = 0; kb < blocks; ++kb) {
      Operand<EXACT> fb[TN];
      int s[TN], eb[TN][4];
      wave_order();
#pragma unroll
      for (int i = 0; i < 2 * TN; ++i) {
        const int r = i * 8 + (lane >> 3);
        *(intx4*)(mine + r * LINE + (((lane & 7) ^ (r >> 1 & 7)) << 4)) = raw[i];
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        s[j] = sb[j];
        if (EXACT)
#pragma unroll
          for (int i = 0; i < 4; ++i) eb[j][i] = __shfl(s[j], 4 * g + i);
      }
      const bool more = kb + 1 < blocks;
      fetch(more ? n1 : n1 + WN * STRIP, more ? kb + 1 : 0);  // past the last column its rows again
      wave_order();
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const char* p = mine + (j * 16 + r16) * LINE;
        fb[j].set(*(const intx4*)(p + piece0), *(const intx4*)(p + piece1));
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const char* p = lds + kb * SHORT_ROWS * LINE + line + i * 16 * LINE;
        Operand<EXACT> fa;
        fa.set(*(const intx4*)(p + piece0), *(const intx4*)(p + piece1));
        const int sa = scales[(wm * TM * 16 + i * 16 + r16) * ks + kb];
#pragma unroll
        for (int j = 0; j < TN; ++j) multiply<0>(acc[i][j], fb[j], fa, s[j], sa, eb[j]);
      }
    }
    const int m1 = m0 + wm * TM * 16;
    if constexpr (EXACT) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int m = m1 + i * 16 + r16, n = n1 + j * 16 + 4 * g;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = activate<T>(acc[i][j][e] + bias[j][e], a.act);
          if (m < a.m && n < a.n) store_four<T>((T*)a.out + (int64_t)m * a.n + n, v, a.n - n);
        }
    } else {
      wave_order();
      if (a.act == KAD_ACT_SILU) store_tile<T, TM, TN, KAD_ACT_SILU>(a, acc, bias, mine, lane, m1, n1);
      else if (a.act == KAD_ACT_RELU) store_tile<T, TM, TN, KAD_ACT_RELU>(a, acc, bias, mine, lane, m1, n1);
      else store_tile<T, TM, TN, KAD_ACT_NONE>(a, acc, bias, mine, lane, m1, n1);
    }
  }
}

// ---------------------------------------------------------------------------- host
constexpr int CUS = 256;

struct Plan {
  int bm, bn;
  Tiles o;
};

Plan plan_of(const kad_gemm8_args& a) {
  Plan p;
  const int blocks = ceil_div(a.k, BLOCK8);
  const bool exact = a.dtype == KAD_F32;
  const auto count = [&](int bm, int bn) { return (int64_t)ceil_div(a.m, bm) * ceil_div(a.n, bn); };
  // A round of 256 x 256 tiles, one a CU, is taken to be 22 us and 12.5 for each 1000 of k; one of 128 x 128 tiles, two a CU and
  // half the results, 7.9 and 9.2: a fit of 4096 x 4096 results at k of 4096 and 8192, where both are met to a tenth.  At smaller k
  // launches overlap what the fit counts as a round's ends, and only the order of the two is meant.  us with tiles of 256 and of
  // 128 (by the rule):
  //   [8192, 4096] x [4096, 4096] 146 (146) and 188 (182)     [8192, 2048] x [8192, 2048] 135 (190) and 151 (214)
  //   [4096, 8192] x [4096, 8192] 126 (124) and 168 (167)     [6000, 2000] x [6000, 2000]  92 (141) and  89 (132)
  //   [4096, 4096] x [4096, 4096]  65 (73)  and  86 (91)      [6000, 1000] x [6000, 1000]  56 (104) and  52 (86)
  //   [4096, 2048] x [4096, 2048]  36 (48)  and  41 (54)      [8192, 1024] x [8192, 1024]  82 (139) and  85 (139)
  //   [4096, 1024] x [4096, 1024]  23 (35)  and  23 (35)      [40000, 512] x [512, 512]    26 (57)  and  18 (38)
  // Not met: where 256 x 256 tiles are fewer than the CUs, k is cut and its parts joined, which the rule leaves out ([3000, 4096] x
  // [3000, 4096]: 111 and 70, and it takes 256).
  const auto rounds = [&](int tile, int at_once) { return (double)((count(tile, tile) + at_once - 1) / at_once); };
  const double k = a.k * 1e-3;
  p.bm = p.bn = !exact && rounds(WIDE, CUS) * (22 + 12.5 * k) < rounds(128, 2 * CUS) * (7.9 + 9.2 * k) ? WIDE
                : count(128, 128) >= CUS ? 128 : 64;
  p.o.tm = ceil_div(a.m, p.bm);
  p.o.tn = ceil_div(a.n, p.bn);
  const int64_t tiles = (int64_t)p.o.tm * p.o.tn;
  int64_t splits = tiles >= CUS ? 1 : CUS * 2 / tiles;
  const int most = ceil_div(blocks, 2 * KB_GROUP);
  if (splits > most) splits = most;
  p.o.per = round_up(ceil_div(blocks, (int)splits), KB_GROUP);
  p.o.splits = ceil_div(blocks, p.o.per);
  return p;
}

bool few(const kad_gemm8_args& a) { return a.m <= KAD_GEMM8_FEW; }

// Whether rows of a that are values are brought to 8 bits by the product's own blocks, against a launch before it, and by
// which blocks: of 64 columns at a time, which many find a place on a CU, or of 256, for which more of a block's loads are a's.
// us in one launch (64 and 256) and in two:
//   fp16 [40000, 64] x [64, 64]     7.7,  9.3 and 14.4     [40000, 512] x [64, 512]    13.5,  18.9 and 22.0
//        [40000, 256] x [128, 256] 11.6, 14.2 and 18.5     [20000, 256] x [256, 256]   11.8,   9.4 and 14.8
//        [300, 512] x [512, 512]    6.7,  9.1 and 9.9      [40000, 512] x [512, 512]   38.4,  32.4 and 34.4
//        [8000, 256] x [8000, 256] 59.4, 40.2 and 48.4     [40000, 512] x [2048, 512] 115,    86   and 82
//   fp32 [40000, 64] x [64, 64]    12.8, 32.3 and 23.2     [40000, 512] x [512, 512]   83.1, 100   and 75.0
//        [300, 512] x [512, 512]   10.8, 19.1 and 13.1     [40000, 512] x [256, 512]   51.8,  61.4 and 56.5
bool narrow(const kad_gemm8_args& a) {
  return a.n <= (a.dtype == KAD_F32 ? 256 : 128) || (int64_t)ceil_div(a.m, SHORT_ROWS) * ceil_div(a.n, 64) <= CUS;
}
bool takes_values(const kad_gemm8_args& a) {
  const bool known = a.a_dtype == KAD_F32 || a.a_dtype == KAD_F16 || a.a_dtype == KAD_BF16;
  return known && (few(a) || (a.a_dtype == a.dtype && a.k <= SHORT_MOST &&
                              (narrow(a) || (a.dtype != KAD_F32 && (a.n <= 1024 || a.k <= 256)))));
}

template <typename T, typename X, int MT>
void launch_few(const kad_gemm8_args& a, hipStream_t st) {
  gemm8_few_kernel<T, X, MT, sizeof(T) == 4><<<ceil_div(a.n, 16), 64 * FEW_WAVES, 0, st>>>(a);
}

template <typename T, typename X>
void launch_few(const kad_gemm8_args& a, hipStream_t st) {
  if (a.m <= 16) launch_few<T, X, 1>(a, st);
  else launch_few<T, X, 2>(a, st);
}

template <typename T, int WM, int TN>
void launch_short(const kad_gemm8_args& a, hipStream_t st) {
  constexpr int COLUMNS = 4 / WM * TN * 16;  // that a block's waves take at a time
  const int tm = ceil_div(a.m, SHORT_ROWS), most = ceil_div(a.n, COLUMNS), blocks = ceil_div(a.k, BLOCK8);
  int parts = tm >= 2 * CUS ? 1 : 2 * CUS / tm;
  if (parts > most) parts = most;
  const int columns = round_up(ceil_div(a.n, parts), COLUMNS);
  const size_t bytes = blocks * SHORT_ROWS * LINE + SHORT_ROWS * round_up(blocks, 4) + 4 * short_bytes(TN);
  allow_lds(gemm8_short_kernel<T, WM, TN>, bytes);
  gemm8_short_kernel<T, WM, TN><<<dim3(tm, ceil_div(a.n, columns)), 256, bytes, st>>>(a, columns);
}

template <typename T, int BM, int BN, int WM, int WN>
void launch_tiles(const kad_gemm8_args& a, const Tiles& o, hipStream_t st) {
  constexpr bool EXACT = sizeof(T) == 4;
  const int total = o.tm * o.tn * o.splits, blocks = ceil_div(total, 8) * 8;
  gemm8_tile_kernel<T, BM, BN, WM, WN, EXACT><<<blocks, 64 * WM * WN, 0, st>>>(a, o);
}

template <typename T>
void launch(const kad_gemm8_args& a, hipStream_t st) {
  if (few(a)) {
    if (a.a_scales) launch_few<T, unsigned char>(a, st);
    else if (a.a_dtype == KAD_F32) launch_few<T, float>(a, st);
    else if (a.a_dtype == KAD_F16) launch_few<T, half_t>(a, st);
    else launch_few<T, bf16_t>(a, st);
    return;
  }
  if (!a.a_scales) {
    if (narrow(a)) launch_short<T, 2, 2>(a, st);
    else if constexpr (sizeof(T) == 2) launch_short<T, 1, 4>(a, st);
    return;
  }
  const Plan p = plan_of(a);
  if constexpr (sizeof(T) == 2)
    if (p.bm == WIDE) gemm8_wide_kernel<T><<<ceil_div(p.o.tm * p.o.tn * p.o.splits, 8) * 8, 512, 0, st>>>(a, p.o);
  if (p.bm == 128) launch_tiles<T, 128, 128, 2, 2>(a, p.o, st);
  if (p.bm == 64) launch_tiles<T, 64, 64, 2, 2>(a, p.o, st);
  if (p.o.splits > 1) {
    const int64_t n = ((int64_t)a.m * a.n + 255) / 256;
    gemm8_join_kernel<T><<<n < 4096 ? n : 4096, 256, 0, st>>>(a, p.o.splits);
  }
}

int check_args(const kad_gemm8_args* a, const char* what) {
  const auto is_dtype = [](int t) { return t == KAD_F32 || t == KAD_F16 || t == KAD_BF16; };
  KAD_CHECK_ARG(a, "%s: null pointer", what);
  KAD_CHECK_ARG(is_dtype(a->dtype), "%s: bad dtype", what);
  KAD_CHECK_ARG(a->m > 0 && a->n > 0 && a->k > 0 && a->k <= KAD_GEMM8_MOST && a->m <= INT32_MAX - 255 && a->n <= INT32_MAX - 255,
                "%s: bad sizes", what);
  KAD_CHECK_ARG((int64_t)ceil_div(a->m, 64) * ceil_div(a->n, 64) < 1 << 24, "%s: fewer than 2^24 tiles of 64 x 64 results expected", what);
  KAD_CHECK_ARG(!few(*a) || a->n < 1 << 26, "%s: up to %d rows: fewer than 2^26 columns expected", what, KAD_GEMM8_FEW);
  KAD_CHECK_ARG(a->act == KAD_ACT_NONE || a->act == KAD_ACT_RELU || a->act == KAD_ACT_SILU, "%s: unknown activation", what);
  KAD_CHECK_ARG(a->a_scales || takes_values(*a), "%s: a as values is not taken at these sizes and types", what);
  KAD_CHECK_ARG(!a->bias || is_dtype(a->bias_dtype), "%s: bad bias_dtype", what);
  return KAD_OK;
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_gemm8_work_elems(const kad_gemm8_args* a) {
  if (int rc = check_args(a, "kad_gemm8_work_elems")) return rc;
  if (few(*a) || !a->a_scales) return 0;
  const Plan p = plan_of(*a);
  return p.o.splits > 1 ? (int64_t)p.o.splits * a->m * a->n : 0;
}

extern "C" int kad_gemm8_takes_values(const kad_gemm8_args* a) {
  return a && takes_values(*a);
}

extern "C" int kad_gemm8(const kad_gemm8_args* a, void* stream) {
  const char* what = "kad_gemm8";
  if (int rc = check_args(a, what)) return rc;
  KAD_CHECK_ARG(a->a && a->b && a->b_scales && a->out, "%s: null pointer", what);
  KAD_CHECK_ARG(((uintptr_t)a->b | (a->a_scales ? (uintptr_t)a->a : 0)) % 16 == 0, "%s: codes must be aligned to 16 bytes", what);
  KAD_CHECK_ARG(((uintptr_t)a->b_scales | (uintptr_t)a->a_scales) % 4 == 0, "%s: scales must be aligned to 4 bytes", what);
  KAD_CHECK_ARG(a->a_scales || (a->a_rs >= a->k && a->a_rs <= INT32_MAX), "%s: a_rs does not fit k", what);
  KAD_CHECK_ARG(a->work || kad_gemm8_work_elems(a) == 0, "%s: work is missing", what);
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) launch<float>(*a, st);
  else if (a->dtype == KAD_F16) launch<half_t>(*a, st);
  else launch<bf16_t>(*a, st);
  return check_launch(what);
}
