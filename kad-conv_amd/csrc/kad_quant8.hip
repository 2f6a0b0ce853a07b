// Rows and columns of a matrix in 8 bits with a scale for each block of 128 (kad_block8.h).
//
// Memory bounds it: x [rows][c] is read once, and its codes along the rows, those along the columns (of the transposed
// matrix), or both are written.  A block of threads holds a tile of 128 rows and 128 columns in registers, which is one
// block of 8-bit numbers in either direction, so that neither scale needs more than the tile; what goes transposed takes
// its way through LDS, 8 or 16 rows of a column at a time.  The tile's column sums, of which a bias' gradient is made,
// are left in work and joined by a second launch, in an order that the sizes alone decide.
//
// [8192, 4096] bf16 along its rows 20.1 us (5.0 TB/s; 17.4 where the matrix is still in the memory-side cache), both ways 32.7 (4.2:
// every tile's way through LDS, and its two barriers; 35 with 30 KB of LDS and columns that met in a few banks).
#include "kad_block8.h"

namespace kad {
namespace {

template <typename T> constexpr int DEEP = LANES<T> / 2;       // rows of a thread

// Where 16-byte piece p of a column of codes lies in LDS: so that neither the threads that write some rows of many columns nor
// those that read whole columns meet in a few banks.
__device__ __forceinline__ int piece_of(int c, int p) { return (c ^ (c >> 3 & 1)) * BLOCK8 + ((p ^ (c >> 4 & 3) << 1) << 4); }

template <typename T>
__global__ __launch_bounds__(256) void quant8_kernel(kad_quant8_args a) {
  constexpr int V = VEC<T>, L = LANES<T>, D = DEEP<T>, SUBS = 256 / L;  // SUBS threads share a column
  // 20 KB in all, of which a CU holds eight
  __shared__ uint32_t most[SUBS][L * 4];  // of a thread's columns, as its words hold them
  __shared__ __attribute__((aligned(16))) unsigned char flat[BLOCK8 * BLOCK8];
  float(*column_sums)[BLOCK8] = (float(*)[BLOCK8])flat;  // before the codes
  const int t = threadIdx.x, l = t % L, sub = t / L;
  const int tiles = (a.c + BLOCK8 - 1) / BLOCK8;
  const int64_t band = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x - band * tiles), col = tile * BLOCK8 + l * V, left = a.c - col;
  const int64_t row0 = band * BLOCK8 + sub * D;
  uint32_t x[D][4];
  // whole vectors of whole rows, all on their way at once
  if (left >= V && row0 + D <= a.rows) {
    const T* p = (const T*)a.x + row0 * a.x_rs + col;
#pragma unroll
    for (int r = 0; r < D; ++r) {
      const intx4 v = load_vec(p + r * a.x_rs);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[r][i] = v[i];
    }
  } else {
#pragma unroll
    for (int r = 0; r < D; ++r) {
      const int n = row0 + r < a.rows && left > 0 ? left : 0;
      float v[V];
      load_some((const T*)a.x + (n ? (row0 + r) * a.x_rs + col : 0), n, v);
      const intx4 w = pack<T>(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[r][i] = w[i];
    }
  }
  if (a.codes) {
    const int64_t kp = (int64_t)tiles * BLOCK8, kb = (tiles + 3) / 4 * 4;
#pragma unroll
    for (int r = 0; r < D; ++r) {
      const int s = scale_of<T>(lanes_largest<L>(largest_finite<T, 4>(x[r])));
      if (row0 + r >= a.rows) continue;
      int* to = (int*)((unsigned char*)a.codes + (row0 + r) * kp + col);
      if constexpr (sizeof(T) == 2) {
        to[0] = codes_of<T>(x[r][0], x[r][1], s);
        to[1] = codes_of<T>(x[r][2], x[r][3], s);
      } else {
        to[0] = codes_of(x[r][0], x[r][1], x[r][2], x[r][3], s);
      }
      unsigned char* sc = (unsigned char*)a.scales + (row0 + r) * kb;
      if (l == 0) sc[tile] = (unsigned char)s;
      if (tile == tiles - 1 && l < kb - tiles) sc[tiles + l] = 127;  // so that a row's scales can be read by fours
    }
  }
  if (a.sums) {
    float total[V];
#pragma unroll
    for (int e = 0; e < V; ++e) total[e] = 0.f;
#pragma unroll
    for (int r = 0; r < D; ++r) {
      float v[V];
      unpack<T>(intx4{(int)x[r][0], (int)x[r][1], (int)x[r][2], (int)x[r][3]}, v);
#pragma unroll
      for (int e = 0; e < V; ++e) total[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) column_sums[sub][l * V + e] = total[e];
    __syncthreads();
    if (t < BLOCK8 && tile * BLOCK8 + t < a.c) {
      float s = column_sums[0][t];
#pragma unroll
      for (int i = 1; i < SUBS; ++i) s += column_sums[i][t];
      a.work[band * a.c + tile * BLOCK8 + t] = s;
    }
  }
  if (!a.t_codes) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < D; ++r) m = larger<T>(m, magnitudes<T>(x[r][i]));
    if (!all_finite<T>(m)) {
      m = 0;
#pragma unroll
      for (int r = 0; r < D; ++r) m = larger<T>(m, finite_of<T>(magnitudes<T>(x[r][i])));
    }
    most[sub][l * 4 + i] = m;
  }
  __syncthreads();
  const int bands = (int)((a.rows + BLOCK8 - 1) / BLOCK8);
  const int64_t mp = (int64_t)bands * BLOCK8, mb = (bands + 3) / 4 * 4;
  constexpr int PER = V / 4;  // columns of a word
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < SUBS; ++k) m = larger<T>(m, most[k][l * 4 + i]);
#pragma unroll
    for (int h = 0; h < PER; ++h) {
      const int s = scale_of<T>(PER == 1 ? m : h ? m >> 16 : m & 0xFFFFu), c = l * V + i * PER + h;
      int* to = (int*)(flat + piece_of(c, sub * D / 16) + sub * D % 16);
#pragma unroll
      for (int r = 0; r < D; r += 4) {
        if constexpr (PER == 1) {
          to[r / 4] = codes_of(x[r][i], x[r + 1][i], x[r + 2][i], x[r + 3][i], s);
        } else {  // the column's halves of two rows at a time
          const uint32_t pick = h ? 0x07060302u : 0x05040100u;
          to[r / 4] = codes_of<T>(__builtin_amdgcn_perm(x[r + 1][i], x[r][i], pick), __builtin_amdgcn_perm(x[r + 3][i], x[r + 2][i], pick), s);
        }
      }
      if (sub == 0 && tile * BLOCK8 + c < a.c) {
        unsigned char* sc = (unsigned char*)a.t_scales + (tile * BLOCK8 + c) * mb;
        sc[band] = (unsigned char)s;
        if (band == bands - 1)
          for (int k = bands; k < mb; ++k) sc[k] = 127;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = t; i < BLOCK8 * 8; i += 256) {  // 16 bytes each
    const int c = i / 8, at = i % 8 * 16;
    if (tile * BLOCK8 + c < a.c)
      *(intx4*)((unsigned char*)a.t_codes + (tile * BLOCK8 + c) * mp + band * BLOCK8 + at) = *(const intx4*)(flat + piece_of(c, at / 16));
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
