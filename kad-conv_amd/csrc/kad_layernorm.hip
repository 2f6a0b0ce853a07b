// Layer norm of rows, forward and backward.
//
//   forward   y = w xhat + b, xhat = (x - mean) rstd
//   backward  dx = rstd (w dy - s1 - xhat s2), s1 = mean of w dy, s2 = mean of w dy xhat over the row
//             dw = sum dy xhat, db = sum dy over rows
//
// Memory bounds it: a row stays in registers (at most 16 values a thread), so x is read once and y written once, x and dy
// read once and dx written.
//
// Layout.  A row belongs to G threads (1 .. 1024), each with U vectors (kad_rows.h).  A block walks rows with its
// parameters (and, backward, its share of dw and db) in registers, the next row's values on their way while it computes.
// [16384, 4096] bf16: forward 54 us (5.0 TB/s), backward 67 (6.3, part of x still in the memory-side cache) and 5 for the join;
// the map [8, 256, 100, 100] 15 us (5.5); a copy reaches 5.1.  [3, 86, 67, 41] fp32: 4.6 + 5.9 + 4.8, latencies.
//
// Sums.  The variance is that of the differences to the mean, in 32 bits, whose own mean corrects both: a row of one value
// repeated is 0 everywhere.  All sums are joined in an order that the sizes alone decide: dw and db first over a block's
// rows, then over blocks in a second launch.
#include "kad_rows.h"

namespace kad {
namespace {

template <typename Q, int VV, int U, bool RAGGED>
__device__ __forceinline__ void params(const void* p, float none, const Place<VV, U, RAGGED>& o, float f[U][VV]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    Q q[VV];
    if (p) __builtin_memcpy(q, (const Q*)p + o.at[u], sizeof(q));
#pragma unroll
    for (int e = 0; e < VV; ++e) f[u][e] = p ? to_f32(q[e]) : none;
  }
}

template <typename T, int VV, int U, bool RAGGED, int MOST>
__global__ __launch_bounds__(MOST) void layer_norm_fwd_kernel(kad_layer_norm_args a, int G) {
  __shared__ float red[2][32];
  const int sub = threadIdx.x / G, l = threadIdx.x & (G - 1), per = blockDim.x / G;
  const Place<VV, U, RAGGED> o(l, G, a.c);
  float w[U][VV], b[U][VV];
  if (a.param_dtype == KAD_F32) {
    params<float>(a.weight, 1.f, o, w);
    params<float>(a.bias, 0.f, o, b);
  } else {
    params<T>(a.weight, 1.f, o, w);
    params<T>(a.bias, 0.f, o, b);
  }
  const float n = (float)a.c;
  const int64_t step = (int64_t)gridDim.x * per, last = a.rows - 1;
  int64_t base = (int64_t)blockIdx.x * per;
  Piece<T, VV> next[U];
  const auto fetch = [&](int64_t row) {
    const T* x = (const T*)a.x + (row < last ? row : last) * a.x_rs;
#pragma unroll
    for (int u = 0; u < U; ++u) next[u].load(x + o.at[u]);
  };
  fetch(base + sub);
  for (; base < a.rows; base += step) {
    const int64_t row = base + sub;
    float x[U][VV], s = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      next[u].get(x[u]);
      s += o.own(u, x[u]);
    }
    fetch(row + step);
    const float about = row_sum(s, G, red[0]) / n;
    // the differences' own mean is what the first one lost
    float s2 = 0.f;
    s = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float q[VV];
#pragma unroll
      for (int e = 0; e < VV; ++e) {
        x[u][e] -= about;
        q[e] = x[u][e] * x[u][e];
      }
      s += o.own(u, x[u]);
      s2 += o.own(u, q);
    }
    row_sums(s, s2, G, red[1]);
    const float rest = s / n, mean = about + rest, rstd = 1.0f / sqrtf(fmaxf(s2 / n - rest * rest, 0.f) + a.eps);
    if (row > last) continue;  // a whole row's threads, and only after the block's last barrier
    if (l == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    T* y = (T*)a.out + row * a.c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!o.on[u]) continue;
#pragma unroll
      for (int e = 0; e < VV; ++e) x[u][e] = (x[u][e] - rest) * rstd * w[u][e] + b[u][e];
      put<T, VV>(y + o.at[u], x[u]);
    }
  }
}

template <typename T, int VV, int U, bool RAGGED, int MOST>
__global__ __launch_bounds__(MOST) void layer_norm_bwd_kernel(kad_layer_norm_args a, int G) {
  __shared__ float red[2][32];
  extern __shared__ float sums[];  // VV floats a thread
  const int sub = threadIdx.x / G, l = threadIdx.x & (G - 1), per = blockDim.x / G;
  const Place<VV, U, RAGGED> o(l, G, a.c);
  float w[U][VV], dw[U][VV], db[U][VV];
  if (a.param_dtype == KAD_F32) params<float>(a.weight, 1.f, o, w);
  else params<T>(a.weight, 1.f, o, w);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < VV; ++e) dw[u][e] = db[u][e] = 0.f;
  const float n = (float)a.c;
  const int64_t step = (int64_t)gridDim.x * per, last = a.rows - 1;
  int64_t base = (int64_t)blockIdx.x * per;
  Piece<T, VV> nx[U], nd[U];
  float nmean, nrstd;
  const auto fetch = [&](int64_t row) {
    row = row < last ? row : last;
    const T *x = (const T*)a.x + row * a.x_rs, *d = (const T*)a.dy + row * a.dy_rs;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      nx[u].load(x + o.at[u]);
      nd[u].load(d + o.at[u]);
    }
    nmean = a.mean[row];
    nrstd = a.rstd[row];
  };
  fetch(base + sub);
  for (int turn = 0; base < a.rows; base += step, turn ^= 1) {
    const int64_t row = base + sub;
    const bool live = row <= last;
    float x[U][VV], d[U][VV], s1 = 0.f, s2 = 0.f;
    const float mean = live ? nmean : 0.f, rstd = live ? nrstd : 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!live) nx[u].raw = nd[u].raw = intx4{0, 0, 0, 0};  // adds 0 to dw and db
      nx[u].get(x[u]);
      nd[u].get(d[u]);
    }
    fetch(row + step);
    // what two vectors share is in the dw and db of both, of which one writes it
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float g[VV], gx[VV];
#pragma unroll
      for (int e = 0; e < VV; ++e) {
        x[u][e] = (x[u][e] - mean) * rstd;
        g[e] = d[u][e] * w[u][e];
        gx[e] = g[e] * x[u][e];
        dw[u][e] += d[u][e] * x[u][e];
        db[u][e] += d[u][e];
      }
      s1 += o.own(u, g);
      s2 += o.own(u, gx);
    }
    if (!a.out) continue;
    row_sums(s1, s2, G, red[turn]);  // two buffers in turn: one barrier a row does
    s1 /= n;
    s2 /= n;
    if (!live) continue;
    T* dx = (T*)a.out + row * a.c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!o.on[u]) continue;
#pragma unroll
      for (int e = 0; e < VV; ++e) d[u][e] = rstd * (d[u][e] * w[u][e] - s1 - x[u][e] * s2);
      put<T, VV>(dx + o.at[u], d[u]);
    }
  }
  if (!a.dweight && !a.dbias) return;
  // [block][dw, db][c]
  float* part = a.work + (int64_t)blockIdx.x * 2 * a.c;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (per > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VV; ++e) sums[threadIdx.x * VV + e] = k ? db[u][e] : dw[u][e];
        __syncthreads();
        for (int i = threadIdx.x; i < G * VV; i += blockDim.x) {
          const int j = (i / VV + u * G) * VV, at = j < a.c - VV ? j : a.c - VV, e = i % VV;
          float s = sums[i];
          for (int r = 1; r < per; ++r) s += sums[r * G * VV + i];
          if (j < a.c && e >= j - at) part[k * a.c + at + e] = s;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VV; ++e)
          if (o.on[u] && e >= o.skip[u]) part[k * a.c + o.at[u] + e] = k ? db[u][e] : dw[u][e];
      }
    }
}

// 64 columns of dw or db a block: 16 waves take every sixteenth part, in order.
__global__ __launch_bounds__(1024) void layer_norm_param_kernel(kad_layer_norm_args a, int parts) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (col < a.c)
#pragma unroll 4
    for (int p = wave; p < parts; p += 16) s += a.work[((int64_t)p * 2 + blockIdx.y) * a.c + col];
  red[wave][lane] = s;
  __syncthreads();
  void* to = blockIdx.y ? a.dbias : a.dweight;
  if (wave || col >= a.c || !to) return;
  for (int i = 1; i < 16; ++i) s += red[i][lane];
  store_param(to, col, a.param_dtype, s);
}

struct Shape {
  int vv, u, G, threads;
  int64_t blocks;
};

Shape shape_of(const kad_layer_norm_args& a, bool backward) {
  Shape s;
  const int v = 16 / dtype_size(a.dtype);
  s.vv = a.c >= v ? v : 1;
  const int vecs = ceil_div(a.c, s.vv), most = s.vv == 1 ? 1 : 16 / v;
  s.u = 1;
  while (s.u < most && vecs > 64 * s.u) s.u *= 2;  // a wave a row where it does
  while (s.u < most && vecs >= 16 * s.u && a.rows * vecs >= 256 * 1024) s.u *= 2;
  s.G = 1;
  while (s.G * s.u < vecs) s.G *= 2;
  s.threads = s.G > 256 ? s.G : 256;
  const int64_t turns = (a.rows + s.threads / s.G - 1) / (s.threads / s.G);
  const int64_t most_blocks = (backward ? 512 : 2048) * 256 / s.threads;
  s.blocks = turns < most_blocks ? turns : most_blocks;
  return s;
}

int check_args(const kad_layer_norm_args* a, const char* what) {
  KAD_CHECK_ARG(a, "%s: null pointer", what);
  KAD_CHECK_ARG(a->dtype == KAD_F32 || a->dtype == KAD_F16 || a->dtype == KAD_BF16, "%s: bad dtype", what);
  KAD_CHECK_ARG(a->param_dtype == KAD_F32 || a->param_dtype == a->dtype, "%s: param_dtype must be float or dtype", what);
  KAD_CHECK_ARG(a->rows > 0 && a->rows <= (int64_t)1 << 40, "%s: 1 to 2^40 rows expected", what);
  KAD_CHECK_ARG(a->c > 0 && a->c <= KAD_LAYER_NORM_MOST, "%s: rows of 1 to %d values expected", what, KAD_LAYER_NORM_MOST);
  KAD_CHECK_ARG(a->eps >= 0.f, "%s: eps must be >= 0", what);
  return KAD_OK;
}

int check_call(const kad_layer_norm_args* a, bool backward, const char* what) {
  if (int rc = check_args(a, what)) return rc;
  KAD_CHECK_ARG(a->x && !a->mean == !a->rstd && (backward ? a->dy && a->mean : a->out != nullptr), "%s: null pointer", what);
  KAD_CHECK_ARG(a->x_rs >= a->c && a->x_rs <= INT32_MAX, "%s: x_rs does not fit c", what);
  KAD_CHECK_ARG(!backward || (a->dy_rs >= a->c && a->dy_rs <= INT32_MAX), "%s: dy_rs does not fit c", what);
  KAD_CHECK_ARG(!backward || a->work || (!a->dweight && !a->dbias), "%s: work is missing", what);
  return KAD_OK;
}

template <typename T, int VV, int U, bool RAGGED, int MOST>
void launch(const kad_layer_norm_args& a, const Shape& s, bool backward, hipStream_t st) {
  if (backward)
    layer_norm_bwd_kernel<T, VV, U, RAGGED, MOST><<<s.blocks, s.threads, s.threads * VV * sizeof(float), st>>>(a, s.G);
  else
    layer_norm_fwd_kernel<T, VV, U, RAGGED, MOST><<<s.blocks, s.threads, 0, st>>>(a, s.G);
}

template <typename T, int VV, int U>
void launch(const kad_layer_norm_args& a, const Shape& s, bool backward, hipStream_t st) {
  if (VV > 1 && a.c % VV) s.threads > 256 ? launch<T, VV, U, true, 1024>(a, s, backward, st) : launch<T, VV, U, true, 256>(a, s, backward, st);
  else s.threads > 256 ? launch<T, VV, U, false, 1024>(a, s, backward, st) : launch<T, VV, U, false, 256>(a, s, backward, st);
}

template <typename T>
void launch(const kad_layer_norm_args& a, bool backward, hipStream_t st) {
  const Shape s = shape_of(a, backward);
  if (s.vv == 1) launch<T, 1, 1, false, 256>(a, s, backward, st);  // fewer values than a vector: one block's at most
  else if (s.u == 1) launch<T, VEC<T>, 1>(a, s, backward, st);
  else if (s.u == 2) launch<T, VEC<T>, 2>(a, s, backward, st);
  else if constexpr (sizeof(T) == 4) launch<T, VEC<T>, 4>(a, s, backward, st);
  if (backward && (a.dweight || a.dbias))
    layer_norm_param_kernel<<<dim3(ceil_div(a.c, 64), 2), 1024, 0, st>>>(a, (int)s.blocks);
}

int run(const kad_layer_norm_args* a, bool backward, void* stream, const char* what) {
  if (int rc = check_call(a, backward, what)) return rc;
  if (backward && !a->out && !a->dweight && !a->dbias) return KAD_OK;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) launch<float>(*a, backward, st);
  else if (a->dtype == KAD_F16) launch<half_t>(*a, backward, st);
  else launch<bf16_t>(*a, backward, st);
  return check_launch(what);
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_layer_norm_work_elems(const kad_layer_norm_args* a) {
  if (int rc = check_args(a, "kad_layer_norm_work_elems")) return rc;
  return shape_of(*a, true).blocks * 2 * a->c;
}

extern "C" int kad_layer_norm_fwd(const kad_layer_norm_args* a, void* stream) {
  return run(a, false, stream, "kad_layer_norm_fwd");
}

extern "C" int kad_layer_norm_bwd(const kad_layer_norm_args* a, void* stream) {
  return run(a, true, stream, "kad_layer_norm_bwd");
}
