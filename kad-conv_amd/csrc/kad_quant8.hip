// Rows and columns of a matrix in 8 bits with a scale for each block of 128 (kad_block8.h).
//
// Memory bounds it: x [rows][c] is read once, and its codes along the rows, those along the columns (of the transposed
// matrix), or both are written.  A block of threads holds a tile of 128 rows and 128 columns in registers, which is one
// block of 8-bit numbers in either direction, so that neither scale needs more than the tile; what goes transposed takes
// its way through LDS, 8 or 16 rows of a column at a time.  The tile's column sums, of which a bias' gradient is made,
// are left in work and joined by a second launch, in an order that the sizes alone decide.
#include "kad_block8.h"

namespace kad {
namespace {

template <typename T> constexpr int LANES = BLOCK8 / VEC<T>;   // that share a row
template <typename T> constexpr int DEEP = LANES<T> / 2;       // rows of a thread
constexpr int PITCH = BLOCK8 + 16;                             // bytes from column to column in LDS

// Largest over the lanes of a row.
template <int N>
__device__ __forceinline__ uint32_t lanes_largest(uint32_t v) {
#pragma unroll
  for (int m = 1; m < N; m <<= 1) {
    const uint32_t o = __shfl_xor(v, m);
    v = v > o ? v : o;
  }
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void quant8_kernel(kad_quant8_args a) {
  constexpr int V = VEC<T>, L = LANES<T>, D = DEEP<T>, SUBS = 256 / L;  // SUBS threads share a column
  __shared__ uint32_t most[SUBS][BLOCK8];
  __shared__ __attribute__((aligned(16))) unsigned char flat[BLOCK8 * PITCH];
  const int t = threadIdx.x, l = t % L, sub = t / L;
  const int tiles = (a.c + BLOCK8 - 1) / BLOCK8;
  const int64_t band = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x - band * tiles), col = tile * BLOCK8 + l * V, left = a.c - col;
  const int64_t row0 = band * BLOCK8 + sub * D;
  float x[D][V];
  // whole vectors of whole rows first, all on their way at once
  if (left >= V && row0 + D <= a.rows) {
    intx4 raw[D];
    const T* p = (const T*)a.x + row0 * a.x_rs + col;
#pragma unroll
    for (int r = 0; r < D; ++r) raw[r] = load_vec(p + r * a.x_rs);
#pragma unroll
    for (int r = 0; r < D; ++r) unpack<T>(raw[r], x[r]);
  } else {
#pragma unroll
    for (int r = 0; r < D; ++r) {
      const int n = row0 + r < a.rows && left > 0 ? left : 0;
      load_some((const T*)a.x + (n ? (row0 + r) * a.x_rs + col : 0), n, x[r]);
    }
  }
  if (a.codes) {
    const int64_t kp = (int64_t)tiles * BLOCK8, kb = (tiles + 3) / 4 * 4;
#pragma unroll
    for (int r = 0; r < D; ++r) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t b = magnitude(x[r][e]);
        m = m > b ? m : b;
      }
      const int s = scale_of(lanes_largest<L>(m));
      if (row0 + r >= a.rows) continue;
      const float inv = inverse(s);
      int* to = (int*)((unsigned char*)a.codes + (row0 + r) * kp + col);
#pragma unroll
      for (int e = 0; e < V; e += 4) to[e / 4] = codes_of(x[r][e], x[r][e + 1], x[r][e + 2], x[r][e + 3], inv);
      unsigned char* sc = (unsigned char*)a.scales + (row0 + r) * kb;
      if (l == 0) sc[tile] = (unsigned char)s;
      if (tile == tiles - 1 && l < kb - tiles) sc[tiles + l] = 127;  // so that a row's scales can be read by fours
    }
  }
  if (!a.t_codes && !a.sums) return;
  float total[V];
  uint32_t m[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    total[e] = 0.f;
    m[e] = 0;
#pragma unroll
    for (int r = 0; r < D; ++r) {
      total[e] += x[r][e];
      const uint32_t b = magnitude(x[r][e]);
      m[e] = m[e] > b ? m[e] : b;
    }
  }
  if (a.sums) {
#pragma unroll
    for (int e = 0; e < V; ++e) most[sub][l * V + e] = __float_as_uint(total[e]);
    __syncthreads();
    if (t < BLOCK8 && tile * BLOCK8 + t < a.c) {
      float s = __uint_as_float(most[0][t]);
#pragma unroll
      for (int i = 1; i < SUBS; ++i) s += __uint_as_float(most[i][t]);
      a.work[band * a.c + tile * BLOCK8 + t] = s;
    }
    __syncthreads();
  }
  if (!a.t_codes) return;
#pragma unroll
  for (int e = 0; e < V; ++e) most[sub][l * V + e] = m[e];
  __syncthreads();
  const int bands = (int)((a.rows + BLOCK8 - 1) / BLOCK8);
  const int64_t mp = (int64_t)bands * BLOCK8, mb = (bands + 3) / 4 * 4;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < SUBS; ++i) b = b > most[i][l * V + e] ? b : most[i][l * V + e];
    const int s = scale_of(b);
    const float inv = inverse(s);
    int* to = (int*)(flat + (l * V + e) * PITCH + sub * D);
#pragma unroll
    for (int r = 0; r < D; r += 4) to[r / 4] = codes_of(x[r][e], x[r + 1][e], x[r + 2][e], x[r + 3][e], inv);
    if (sub == 0 && col + e < a.c) {
      unsigned char* sc = (unsigned char*)a.t_scales + (col + e) * mb;
      sc[band] = (unsigned char)s;
      if (band == bands - 1)
        for (int i = bands; i < mb; ++i) sc[i] = 127;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = t; i < BLOCK8 * 8; i += 256) {  // 16 bytes each
    const int c = i / 8, at = i % 8 * 16;
    if (tile * BLOCK8 + c < a.c)
      *(intx4*)((unsigned char*)a.t_codes + (tile * BLOCK8 + c) * mp + band * BLOCK8 + at) = *(const intx4*)(flat + c * PITCH + at);
  }
}

// 64 columns a block: 16 waves take every sixteenth band, in order.
__global__ __launch_bounds__(1024) void quant8_sums_kernel(kad_quant8_args a, int bands) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (col < a.c)
#pragma unroll 4
    for (int b = wave; b < bands; b += 16) s += a.work[(int64_t)b * a.c + col];
  red[wave][lane] = s;
  __syncthreads();
  if (wave || col >= a.c) return;
  for (int i = 1; i < 16; ++i) s += red[i][lane];
  store_param(a.sums, col, a.sums_dtype, s);
}

int check_args(const kad_quant8_args* a, const char* what) {
  KAD_CHECK_ARG(a, "%s: null pointer", what);
  KAD_CHECK_ARG(a->dtype == KAD_F32 || a->dtype == KAD_F16 || a->dtype == KAD_BF16, "%s: bad dtype", what);
  KAD_CHECK_ARG(a->rows > 0 && a->rows <= INT32_MAX - 127 && a->c > 0 && a->c <= KAD_QUANT8_MOST,
                "%s: 1 to 2^31 - 128 rows and 1 to %d columns expected", what, KAD_QUANT8_MOST);
  const int64_t tiles = (a->rows + 127) / 128 * ((a->c + 127) / 128);
  KAD_CHECK_ARG(tiles < 1 << 24, "%s: fewer than 2^24 tiles of 128 x 128 values", what);
  return KAD_OK;
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_quant8_work_elems(const kad_quant8_args* a) {
  if (int rc = check_args(a, "kad_quant8_work_elems")) return rc;
  return a->sums ? (a->rows + 127) / 128 * a->c : 0;
}

extern "C" int kad_quant8(const kad_quant8_args* a, void* stream) {
  const char* what = "kad_quant8";
  if (int rc = check_args(a, what)) return rc;
  KAD_CHECK_ARG(a->x && !a->codes == !a->scales && !a->t_codes == !a->t_scales, "%s: null pointer", what);
  KAD_CHECK_ARG(a->codes || a->t_codes || a->sums, "%s: nothing is wanted", what);
  KAD_CHECK_ARG(a->x_rs >= a->c && a->x_rs <= INT32_MAX, "%s: x_rs does not fit c", what);
  KAD_CHECK_ARG(((uintptr_t)a->codes | (uintptr_t)a->t_codes) % 16 == 0, "%s: codes must be aligned to 16 bytes", what);
  KAD_CHECK_ARG(!a->sums || a->work, "%s: work is missing", what);
  KAD_CHECK_ARG(!a->sums || a->sums_dtype == KAD_F32 || a->sums_dtype == KAD_F16 || a->sums_dtype == KAD_BF16, "%s: bad sums_dtype",
                what);
  const hipStream_t st = (hipStream_t)stream;
  const int bands = (int)((a->rows + 127) / 128);
  const int64_t tiles = (int64_t)bands * ceil_div(a->c, BLOCK8);
  if (a->dtype == KAD_F32) quant8_kernel<float><<<tiles, 256, 0, st>>>(*a);
  else if (a->dtype == KAD_F16) quant8_kernel<half_t><<<tiles, 256, 0, st>>>(*a);
  else quant8_kernel<bf16_t><<<tiles, 256, 0, st>>>(*a);
  if (a->sums) quant8_sums_kernel<<<ceil_div(a->c, 64), 1024, 0, st>>>(*a, bands);
  return check_launch(what);
}
