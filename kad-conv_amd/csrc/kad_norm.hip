// Group norm with an activation on NHWC maps, forward and backward.
//
//   forward   z = w (x - mean) rstd + b, y = act(z)
//   backward  dz = dy act'(z), xhat = (x - mean) rstd
//             db = sum dz, dw = sum dz xhat        over images and pixels
//             dx = rstd (w dz - (s1 + xhat s2) / M), s1 = sum w dz, s2 = sum w dz xhat over the group's M values
//
// Memory bounds it: a map is read (x; x and dy) and written (y; dx), with 20 to 25 vector operations a
// value, a third of them the SiLU's exponential and reciprocal.
//
// Layout.  Threads own 16-byte vectors of V channels.  Where V does not divide C, k = V / gcd(C, V) pixels
// are taken as one row of k C channels, which V divides: a thread's vector meets the same V channels in
// every row, so its sums, weights and biases stay in registers, and any C is read in whole vectors.  A
// block of R x S threads takes R rows of S vectors at a time.
//
// Statistics.  A variance from sums of squares loses all digits where the mean is large, and a shift by the
// first value does where that one is an outlier: a thread takes means and squares about them over a few
// rows in registers and merges these (Chan's formula), so 32 bits suffice for any order of the values.
#include "kad_common.h"

namespace kad {
namespace {

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

// 1 / (1 + e^-z) with the hardware's reciprocal (off by one step of 32 bits at most): 0 where e^-z overflows.
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// act(z), and act'(z) times dy.
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  return ACT == KAD_ACT_SILU ? z * logistic(z) : ACT == KAD_ACT_RELU ? (z > 0.f ? z : z != z ? z : 0.f) : z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z, float dy) {
  if (ACT == KAD_ACT_SILU) {
    const float s = logistic(z);
    return dy * s * (1.f + z * (1.f - s));
  }
  return ACT == KAD_ACT_RELU ? (z > 0.f ? dy : 0.f) : dy;
}

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);

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
__device__ __forceinline__ void store_vec(T* p, const float v[VEC<T>]) {
  T t[VEC<T>];
#pragma unroll
  for (int i = 0; i < VEC<T>; ++i) t[i] = from_f32<T>(v[i]);
  __builtin_memcpy(p, t, 16);
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

// How a block's columns (q groups of D channels, W in all) are cut into rows and vectors.
struct Geo {
  int k, S, R;    // pixels in a row, vectors in a row, rows at a time
  int full;       // whole rows of an image
  int tail;       // values of the pixels after them (fewer than k; 0 where k = 1)
  int W, q, D;
  int rows, tiles;  // split kernels: rows of a tile, tiles of an image
  int tpg;          // threads that sum one group: a power of two, at most 64
  int tpc;          // and one channel
  int share;        // resident kernel: consecutive sets of groups that one 128-byte line may hold
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// Sums over runs of D of the block's values.  Thread t < active holds val[0 .. VV), which are the places
// t VV + v of a matrix of rows of W values; out[g] becomes the sum of columns [g D, (g + 1) D), in an order
// that the sizes alone decide.  red: VV values a thread; out may be read by all threads afterwards.
template <int VV>
__device__ __forceinline__ void run_sums(const float* val, int active, int W, int q, int D, int per, float* red, float* out) {
  const int t = threadIdx.x, T = blockDim.x;
  if (q == 1) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < VV; ++v) s += val[v];
    s = wave_sum(t < active ? s : 0.f);
    __syncthreads();
    if ((t & 63) == 0) red[t >> 6] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < T >> 6; ++w) s += red[w];
    if (t == 0) out[0] = s;
    __syncthreads();
    return;
  }
  __syncthreads();
  if (t < active)
#pragma unroll
    for (int v = 0; v < VV; ++v) red[t * VV + v] = val[v];
  __syncthreads();
  const int rows = active * VV / W, l = t & (per - 1);
  const int dp = per / D, dd = per - dp * D;
  for (int g = t / per; g < q; g += T / per) {
    int p = l / D, d = l - p * D;
    float s = 0.f;
    while (p < rows) {
      s += red[p * W + g * D + d];
      p += dp;
      d += dd;
      if (d >= D) {
        d -= D;
        ++p;
      }
    }
    for (int m = 1; m < per; m <<= 1) s += __shfl_xor(s, m);
    if (l == 0) out[g] = s;
  }
  __syncthreads();
}

// A thread's place and its V channels' weights and biases.  ONE: its vector lies in one group.
template <typename T, bool ONE>
struct Columns {
  static constexpr int V = VEC<T>, NG = ONE ? 1 : V;
  int r, j, c0;
  bool on;
  int ntail;  // values of the last, short row that are this thread's
  __device__ __forceinline__ Columns(const Geo& o, int first) {
    const int t = threadIdx.x;
    r = t / o.S;
    j = t - r * o.S;
    on = r < o.R;
    c0 = first;
    ntail = o.tail - j * V;
    ntail = !on || r != 0 || ntail < 0 ? 0 : ntail > V ? V : ntail;
  }
  // Channel (among the block's) of value v, and its group.
  __device__ __forceinline__ int channel(const Geo& o, int v) const { return o.k == 1 ? j * V + v : (j * V + v) % o.W; }
  __device__ __forceinline__ int group(const Geo& o, int v) const { return channel(o, v) / o.D; }
  __device__ __forceinline__ void params(const Geo& o, const kad_group_norm_args& a, float w[V], float b[V]) const {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = c0 + channel(o, v);
      w[v] = on ? load_param(a.weight, c, a.param_dtype, 1.f) : 0.f;
      b[v] = on ? load_param(a.bias, c, a.param_dtype, 0.f) : 0.f;
    }
  }
  __device__ __forceinline__ void of_groups(const Geo& o, const float* lds, float m[NG]) const {
#pragma unroll
    for (int v = 0; v < NG; ++v) m[v] = on ? lds[group(o, v)] : 0.f;
  }
};

template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void norm_vec(float x[VEC<T>], const float* mean, const float* w, const float* b) {
#pragma unroll
  for (int v = 0; v < VEC<T>; ++v) x[v] = act_of<ACT>((x[v] - mean[ONE ? 0 : v]) * w[v] + b[v]);
}

// ---------------------------------------------------------------------------- resident forward
// One block an image and set of groups, whose values stay in registers (U vectors a thread): x is read once,
// and the variance is that of the differences to the mean.
template <typename T, bool ONE, int U, int ACT>
__device__ __forceinline__ void resident_write(const kad_group_norm_args& a, const Geo& o, const Columns<T, ONE>& col,
                                               const intx4 raw[U], float xt[VEC<T>], T* y, const float* mean,
                                               const float* w, const float* b) {
  constexpr int V = VEC<T>;
  const int64_t ys = (int64_t)(o.k == 1 ? a.c : o.k * a.c);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = col.r + u * o.R;
    if (row < o.full) {
      float x[V];
      unpack<T>(raw[u], x);
      norm_vec<T, ONE, ACT>(x, mean, w, b);
      store_vec(y + row * ys, x);
    }
  }
  if (col.ntail) {
    norm_vec<T, ONE, ACT>(xt, mean, w, b);
    store_some(y + o.full * ys, col.ntail, xt);
  }
}

template <typename T, bool ONE, int U>
__global__ __launch_bounds__(1024) void group_norm_resident_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V;
  extern __shared__ float lds[];
  // Sets whose channels share lines run on one XCD (blocks go round the 8 of them), so its L2 fetches a line once.
  const int sets = a.groups / o.q;
  const int id = (blockIdx.x / (8 * o.share) * 8 + (blockIdx.x & 7)) * o.share + (blockIdx.x >> 3) % o.share;
  if (id >= a.n * sets) return;
  const int n = id / sets, set = id - n * sets;
  const Columns<T, ONE> col(o, set * o.W);
  float* mean = lds + blockDim.x * NG;
  float* rstd = mean + o.q;
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs + col.c0 + col.j * V;
  T* y = (T*)a.out + n * P * a.c + col.c0 + col.j * V;
  intx4 raw[U];
  float xt[V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = col.r + u * o.R;
    raw[u] = intx4{0, 0, 0, 0};
    if (col.on && row < o.full) raw[u] = load_vec(x + row * xs);
  }
  load_some(x + o.full * xs, col.ntail, xt);
  float s[NG], m[NG];
#pragma unroll
  for (int v = 0; v < NG; ++v) s[v] = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) s[ONE ? 0 : v] += xt[v];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[V];
    unpack<T>(raw[u], f);
#pragma unroll
    for (int v = 0; v < V; ++v) s[ONE ? 0 : v] += f[v];
  }
  const int active = o.R * o.S, rw = ONE ? o.S : o.W, rd = ONE ? o.D / V : o.D;
  const float M = (float)(P * o.D);
  run_sums<NG>(s, active, rw, o.q, rd, o.tpg, lds, mean);
  for (int g = threadIdx.x; g < o.q; g += blockDim.x) mean[g] /= M;
  if (sizeof(T) == 2) {
#pragma unroll
    for (int u = 0; u < U; ++u) repack(raw[u]);
  }
  __syncthreads();
  col.of_groups(o, mean, m);
#pragma unroll
  for (int v = 0; v < NG; ++v) s[v] = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float d = xt[v] - m[ONE ? 0 : v];
    s[ONE ? 0 : v] += v < col.ntail ? d * d : 0.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (col.r + u * o.R < o.full) {
      float f[V];
      unpack<T>(raw[u], f);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = f[v] - m[ONE ? 0 : v];
        s[ONE ? 0 : v] += d * d;
      }
    }
  run_sums<NG>(s, active, rw, o.q, rd, o.tpg, lds, rstd);
  if (sizeof(T) == 2) {
#pragma unroll
    for (int u = 0; u < U; ++u) repack(raw[u]);
  }
  for (int g = threadIdx.x; g < o.q; g += blockDim.x) {
    rstd[g] = 1.0f / sqrtf(rstd[g] / M + a.eps);
    a.mean[n * a.groups + set * o.q + g] = mean[g];
    a.rstd[n * a.groups + set * o.q + g] = rstd[g];
  }
  __syncthreads();
  if (!col.on) return;
  float w[V], b[V], rs[NG];
  col.params(o, a, w, b);
  col.of_groups(o, rstd, rs);
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] *= rs[ONE ? 0 : v];
  if (a.act == KAD_ACT_SILU) resident_write<T, ONE, U, KAD_ACT_SILU>(a, o, col, raw, xt, y, m, w, b);
  else if (a.act == KAD_ACT_RELU) resident_write<T, ONE, U, KAD_ACT_RELU>(a, o, col, raw, xt, y, m, w, b);
  else resident_write<T, ONE, U, KAD_ACT_NONE>(a, o, col, raw, xt, y, m, w, b);
}

// ---------------------------------------------------------------------------- split forward
// Rows of tile t of an image, and how many pixels it holds.
struct Tile {
  int first, last;
  bool tail;
  __device__ __forceinline__ Tile(const Geo& o, int t) {
    first = t * o.rows;
    last = first + o.rows < o.full ? first + o.rows : o.full;
    tail = t == o.tiles - 1;
  }
};
__device__ __forceinline__ int tile_pixels(const Geo& o, int64_t P, int t) {
  const int64_t first = (int64_t)t * o.rows * o.k, next = first + (int64_t)o.rows * o.k;
  return (int)((t == o.tiles - 1 ? P : next) - first);
}

// Count, mean and squares about the mean of values seen so far.
template <int NG>
struct Moments {
  float n, mean[NG], m2[NG];
  __device__ __forceinline__ Moments() : n(0.f) {
#pragma unroll
    for (int v = 0; v < NG; ++v) mean[v] = m2[v] = 0.f;
  }
  __device__ __forceinline__ void merge(float nc, const float mc[NG], const float qc[NG]) {
    const float t = n + nc, f = nc * __builtin_amdgcn_rcpf(t), nf = n * f;
#pragma unroll
    for (int v = 0; v < NG; ++v) {
      const float d = mc[v] - mean[v];
      mean[v] += d * f;
      m2[v] += qc[v] + d * d * nf;
    }
    n = t;
  }
};

// The moments of B rows of V values, over the rows (for each channel) or over all of them.
template <typename T, bool ONE, int B>
__device__ __forceinline__ void add_rows(Moments<ONE ? 1 : VEC<T>>& acc, const intx4 raw[B]) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V;
  float f[B][V], m[NG], q[NG];
#pragma unroll
  for (int i = 0; i < B; ++i) unpack<T>(raw[i], f[i]);
#pragma unroll
  for (int v = 0; v < NG; ++v) m[v] = q[v] = 0.f;
#pragma unroll
  for (int i = 0; i < B; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) m[ONE ? 0 : v] += f[i][v];
  constexpr float count = ONE ? B * V : B;
#pragma unroll
  for (int v = 0; v < NG; ++v) m[v] *= 1.0f / count;
#pragma unroll
  for (int i = 0; i < B; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float d = f[i][v] - m[ONE ? 0 : v];
      q[ONE ? 0 : v] += d * d;
    }
  acc.merge(count, m, q);
}

template <typename T, bool ONE>
__global__ __launch_bounds__(1024) void group_norm_stats_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V, B = 4;
  extern __shared__ float lds[];
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const Tile rows(o, tile);
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs + col.j * V;
  Moments<NG> acc;
  if (col.on) {
    int row = rows.first + col.r;
    for (; row + (B - 1) * o.R < rows.last; row += B * o.R) {
      intx4 raw[B];
#pragma unroll
      for (int i = 0; i < B; ++i) raw[i] = load_vec(x + (row + i * o.R) * xs);
      add_rows<T, ONE, B>(acc, raw);
    }
    for (; row < rows.last; row += o.R) {
      const intx4 raw[1] = {load_vec(x + row * xs)};
      add_rows<T, ONE, 1>(acc, raw);
    }
  }
  // The short row's values: of a channel each, so counts differ from channel to channel.
  float xt[V], s[NG];
  const int nt = rows.tail ? col.ntail : 0;
  load_some(x + o.full * xs, nt, xt);
#pragma unroll
  for (int v = 0; v < NG; ++v) s[v] = acc.n * acc.mean[v];
#pragma unroll
  for (int v = 0; v < V; ++v) s[ONE ? 0 : v] += xt[v];
  const int active = o.R * o.S, rw = ONE ? o.S : o.W, rd = ONE && o.q > 1 ? o.D / V : o.D;
  float *mean = lds + blockDim.x * NG, *m2 = mean + o.q;
  const float count = (float)tile_pixels(o, P, tile) * (float)o.D;
  run_sums<NG>(s, active, rw, o.q, rd, o.tpg, lds, mean);
  for (int g = threadIdx.x; g < o.q; g += blockDim.x) mean[g] /= count;
  __syncthreads();
  float m[NG];
  col.of_groups(o, mean, m);
#pragma unroll
  for (int v = 0; v < NG; ++v) {
    const float d = acc.mean[v] - m[v];
    s[v] = acc.n > 0.f ? acc.m2[v] + acc.n * d * d : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float d = xt[v] - m[ONE ? 0 : v];
    s[ONE ? 0 : v] += v < nt ? d * d : 0.f;
  }
  run_sums<NG>(s, active, rw, o.q, rd, o.tpg, lds, m2);
  float2* part = (float2*)a.work + ((int64_t)n * o.tiles + tile) * o.q;
  for (int g = threadIdx.x; g < o.q; g += blockDim.x) part[g] = make_float2(mean[g], m2[g]);
}

template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void apply_rows(const Geo& o, const Columns<T, ONE>& col, const Tile& rows, const T* x, int64_t xs,
                                           T* y, int64_t ys, const float* mean, const float* w, const float* b) {
  constexpr int V = VEC<T>, B = 4;
  int row = rows.first + col.r;
  for (; row + (B - 1) * o.R < rows.last; row += B * o.R) {
    intx4 raw[B];
#pragma unroll
    for (int i = 0; i < B; ++i) raw[i] = load_vec(x + (row + i * o.R) * xs);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float f[V];
      unpack<T>(raw[i], f);
      norm_vec<T, ONE, ACT>(f, mean, w, b);
      store_vec(y + (row + i * o.R) * ys, f);
    }
  }
  for (; row < rows.last; row += o.R) {
    float f[V];
    unpack<T>(load_vec(x + row * xs), f);
    norm_vec<T, ONE, ACT>(f, mean, w, b);
    store_vec(y + row * ys, f);
  }
  if (rows.tail && col.ntail) {
    float f[V];
    load_some(x + o.full * xs, col.ntail, f);
    norm_vec<T, ONE, ACT>(f, mean, w, b);
    store_some(y + o.full * ys, col.ntail, f);
  }
}

template <typename T, bool ONE>
__global__ __launch_bounds__(1024) void group_norm_apply_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V;
  extern __shared__ float lds[];
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const int64_t P = (int64_t)a.h * a.w;
  float *mean = lds, *rstd = lds + o.q;
  {  // the tiles' means and squares, joined
    const float2* part = (const float2*)a.work + (int64_t)n * o.tiles * o.q;
    const float M = (float)P * (float)o.D;
    const int per = o.tpg, l = threadIdx.x & (per - 1);
    for (int g = threadIdx.x / per; g < o.q; g += blockDim.x / per) {
      float s = 0.f;
      for (int t = l; t < o.tiles; t += per) s += part[t * o.q + g].x * (float)tile_pixels(o, P, t);
      for (int m = 1; m < per; m <<= 1) s += __shfl_xor(s, m);
      const float mu = s / (float)P;
      s = 0.f;
      for (int t = l; t < o.tiles; t += per) {
        const float2 p = part[t * o.q + g];
        const float d = p.x - mu;
        s += p.y + d * d * ((float)tile_pixels(o, P, t) * (float)o.D);
      }
      for (int m = 1; m < per; m <<= 1) s += __shfl_xor(s, m);
      if (l == 0) {
        const float rs = 1.0f / sqrtf(s / M + a.eps);
        mean[g] = mu;
        rstd[g] = rs;
        if (tile == 0) {
          a.mean[n * a.groups + g] = mu;
          a.rstd[n * a.groups + g] = rs;
        }
      }
    }
    __syncthreads();
  }
  if (!col.on) return;
  float w[V], b[V], m[NG], rs[NG];
  col.params(o, a, w, b);
  col.of_groups(o, mean, m);
  col.of_groups(o, rstd, rs);
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] *= rs[ONE ? 0 : v];
  const Tile rows(o, tile);
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c, ys = (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs + col.j * V;
  T* y = (T*)a.out + n * P * a.c + col.j * V;
  if (a.act == KAD_ACT_SILU) apply_rows<T, ONE, KAD_ACT_SILU>(o, col, rows, x, xs, y, ys, m, w, b);
  else if (a.act == KAD_ACT_RELU) apply_rows<T, ONE, KAD_ACT_RELU>(o, col, rows, x, xs, y, ys, m, w, b);
  else apply_rows<T, ONE, KAD_ACT_NONE>(o, col, rows, x, xs, y, ys, m, w, b);
}

// ---------------------------------------------------------------------------- backward
// Two launches: the sums of dz and dz xhat of each channel in each tile, and of w times them in each group;
// then dx.  The last blocks of the second one sum the channels' parts to dw and db.
template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void sum_vec(const float x[VEC<T>], const float dy[VEC<T>], const float* mean, const float* rstd,
                                        const float* w, const float* b, float* db, float* dw) {
#pragma unroll
  for (int v = 0; v < VEC<T>; ++v) {
    const float xhat = (x[v] - mean[ONE ? 0 : v]) * rstd[ONE ? 0 : v];
    const float dz = act_grad<ACT>(xhat * w[v] + b[v], dy[v]);
    db[v] += dz;
    dw[v] += dz * xhat;
  }
}

template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void sum_rows(const Geo& o, const Columns<T, ONE>& col, const Tile& rows, const T* x, int64_t xs,
                                         const T* dy, int64_t ds, const float* mean, const float* rstd, const float* w,
                                         const float* b, float* db, float* dw) {
  constexpr int V = VEC<T>, B = 2;
  int row = rows.first + col.r;
  for (; row + (B - 1) * o.R < rows.last; row += B * o.R) {
    intx4 rx[B], rd[B];
#pragma unroll
    for (int i = 0; i < B; ++i) rx[i] = load_vec(x + (row + i * o.R) * xs);
#pragma unroll
    for (int i = 0; i < B; ++i) rd[i] = load_vec(dy + (row + i * o.R) * ds);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float f[V], g[V];
      unpack<T>(rx[i], f);
      unpack<T>(rd[i], g);
      sum_vec<T, ONE, ACT>(f, g, mean, rstd, w, b, db, dw);
    }
  }
  for (; row < rows.last; row += o.R) {
    float f[V], g[V];
    unpack<T>(load_vec(x + row * xs), f);
    unpack<T>(load_vec(dy + row * ds), g);
    sum_vec<T, ONE, ACT>(f, g, mean, rstd, w, b, db, dw);
  }
  if (rows.tail && col.ntail) {
    float f[V], g[V], d1[V], d2[V];
    load_some(x + o.full * xs, col.ntail, f);
    load_some(dy + o.full * ds, col.ntail, g);
#pragma unroll
    for (int v = 0; v < V; ++v) d1[v] = d2[v] = 0.f;
    sum_vec<T, ONE, ACT>(f, g, mean, rstd, w, b, d1, d2);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      db[v] += v < col.ntail ? d1[v] : 0.f;
      dw[v] += v < col.ntail ? d2[v] : 0.f;
    }
  }
}

template <typename T, bool ONE>
__global__ __launch_bounds__(1024) void group_norm_bwd_sums_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V;
  extern __shared__ float lds[];
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const Tile rows(o, tile);
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c, ds = o.k == 1 ? a.dy_cs : (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs + col.j * V;
  const T* dy = (const T*)a.dy + n * P * a.dy_cs + col.j * V;
  float db[V], dw[V];
#pragma unroll
  for (int v = 0; v < V; ++v) db[v] = dw[v] = 0.f;
  if (col.on) {
    float w[V], b[V], m[NG], rs[NG];
    col.params(o, a, w, b);
    col.of_groups(o, a.mean + n * o.q, m);
    col.of_groups(o, a.rstd + n * o.q, rs);
    if (a.act == KAD_ACT_SILU) sum_rows<T, ONE, KAD_ACT_SILU>(o, col, rows, x, xs, dy, ds, m, rs, w, b, db, dw);
    else if (a.act == KAD_ACT_RELU) sum_rows<T, ONE, KAD_ACT_RELU>(o, col, rows, x, xs, dy, ds, m, rs, w, b, db, dw);
    else sum_rows<T, ONE, KAD_ACT_NONE>(o, col, rows, x, xs, dy, ds, m, rs, w, b, db, dw);
  }
  const int active = o.R * o.S, T_ = blockDim.x;
  float *cb = lds + T_ * V, *cw = cb + o.W;
  run_sums<V>(db, active, o.W, o.W, 1, o.tpc, lds, cb);
  run_sums<V>(dw, active, o.W, o.W, 1, o.tpc, lds, cw);
  const int64_t part = (int64_t)n * o.tiles + tile;
  float2* groups = (float2*)a.work + part * o.q;
  const int l = threadIdx.x & (o.tpg - 1);
  for (int g = threadIdx.x / o.tpg; g < o.q; g += T_ / o.tpg) {
    float s1 = 0.f, s2 = 0.f;
    for (int c = g * o.D + l; c < (g + 1) * o.D; c += o.tpg) {
      const float w = load_param(a.weight, c, a.param_dtype, 1.f);
      s1 += w * cb[c];
      s2 += w * cw[c];
    }
    for (int m = 1; m < o.tpg; m <<= 1) {
      s1 += __shfl_xor(s1, m);
      s2 += __shfl_xor(s2, m);
    }
    if (l == 0) groups[g] = make_float2(s1, s2);
  }
  if (a.dweight || a.dbias) {
    float2* chans = (float2*)a.work + (int64_t)a.n * o.tiles * o.q + part * o.W;
    for (int c = threadIdx.x; c < o.W; c += T_) chans[c] = make_float2(cb[c], cw[c]);
  }
}

template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void dx_vec(float x[VEC<T>], const float dy[VEC<T>], const float* mean, const float* rstd,
                                       const float* w, const float* b, const float* s1, const float* s2) {
#pragma unroll
  for (int v = 0; v < VEC<T>; ++v) {
    const int g = ONE ? 0 : v;
    const float xhat = (x[v] - mean[g]) * rstd[g];
    const float dz = act_grad<ACT>(xhat * w[v] + b[v], dy[v]);
    x[v] = rstd[g] * (w[v] * dz - s1[g] - xhat * s2[g]);
  }
}

template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void dx_rows(const Geo& o, const Columns<T, ONE>& col, const Tile& rows, const T* x, int64_t xs,
                                        const T* dy, int64_t ds, T* dx, int64_t os, const float* mean, const float* rstd,
                                        const float* w, const float* b, const float* s1, const float* s2) {
  constexpr int V = VEC<T>, B = 2;
  int row = rows.first + col.r;
  for (; row + (B - 1) * o.R < rows.last; row += B * o.R) {
    intx4 rx[B], rd[B];
#pragma unroll
    for (int i = 0; i < B; ++i) rx[i] = load_vec(x + (row + i * o.R) * xs);
#pragma unroll
    for (int i = 0; i < B; ++i) rd[i] = load_vec(dy + (row + i * o.R) * ds);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float f[V], g[V];
      unpack<T>(rx[i], f);
      unpack<T>(rd[i], g);
      dx_vec<T, ONE, ACT>(f, g, mean, rstd, w, b, s1, s2);
      store_vec(dx + (row + i * o.R) * os, f);
    }
  }
  for (; row < rows.last; row += o.R) {
    float f[V], g[V];
    unpack<T>(load_vec(x + row * xs), f);
    unpack<T>(load_vec(dy + row * ds), g);
    dx_vec<T, ONE, ACT>(f, g, mean, rstd, w, b, s1, s2);
    store_vec(dx + row * os, f);
  }
  if (rows.tail && col.ntail) {
    float f[V], g[V];
    load_some(x + o.full * xs, col.ntail, f);
    load_some(dy + o.full * ds, col.ntail, g);
    dx_vec<T, ONE, ACT>(f, g, mean, rstd, w, b, s1, s2);
    store_some(dx + o.full * os, col.ntail, f);
  }
}

// dw and db of 16 channels from the tiles' parts: a thread in each 16 takes a channel, over rows of parts.
constexpr int PARAM_CHANNELS = 16;
__device__ __forceinline__ void param_sums(const kad_group_norm_args& a, const Geo& o, int block, float* lds) {
  const int c = block * PARAM_CHANNELS + (threadIdx.x & (PARAM_CHANNELS - 1));
  const int parts = a.n * o.tiles, step = blockDim.x / PARAM_CHANNELS;
  const float2* chans = (const float2*)a.work + (int64_t)parts * o.q;
  float db = 0.f, dw = 0.f;
  if (c < o.W)
    for (int i = threadIdx.x / PARAM_CHANNELS; i < parts; i += step) {
      const float2 p = chans[(int64_t)i * o.W + c];
      db += p.x;
      dw += p.y;
    }
#pragma unroll
  for (int d = PARAM_CHANNELS; d < 64; d <<= 1) {
    db += __shfl_xor(db, d);
    dw += __shfl_xor(dw, d);
  }
  float2* waves = (float2*)lds;
  if ((threadIdx.x & 63) < PARAM_CHANNELS) waves[(threadIdx.x >> 6) * PARAM_CHANNELS + (threadIdx.x & 63)] = make_float2(db, dw);
  __syncthreads();
  if (threadIdx.x < PARAM_CHANNELS && c < o.W) {
    db = dw = 0.f;
    for (int w = 0; w < blockDim.x >> 6; ++w) {
      db += waves[w * PARAM_CHANNELS + threadIdx.x].x;
      dw += waves[w * PARAM_CHANNELS + threadIdx.x].y;
    }
    if (a.dweight) store_param(a.dweight, c, a.param_dtype, dw);
    if (a.dbias) store_param(a.dbias, c, a.param_dtype, db);
  }
}

template <typename T, bool ONE>
__global__ __launch_bounds__(1024) void group_norm_dx_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V;
  extern __shared__ float lds[];
  const int maps = a.out ? a.n * o.tiles : 0;
  if ((int)blockIdx.x >= maps) return param_sums(a, o, blockIdx.x - maps, lds);
  const int n = blockIdx.x / o.tiles, tile = blockIdx.x - n * o.tiles;
  const Columns<T, ONE> col(o, 0);
  const int64_t P = (int64_t)a.h * a.w;
  float *l1 = lds, *l2 = lds + o.q;
  {
    const float2* part = (const float2*)a.work + (int64_t)n * o.tiles * o.q;
    const float inv = 1.0f / ((float)P * (float)o.D);
    const int per = o.tpg, l = threadIdx.x & (per - 1);
    for (int g = threadIdx.x / per; g < o.q; g += blockDim.x / per) {
      float s1 = 0.f, s2 = 0.f;
      for (int t = l; t < o.tiles; t += per) {
        const float2 p = part[t * o.q + g];
        s1 += p.x;
        s2 += p.y;
      }
      for (int m = 1; m < per; m <<= 1) {
        s1 += __shfl_xor(s1, m);
        s2 += __shfl_xor(s2, m);
      }
      if (l == 0) {
        l1[g] = s1 * inv;
        l2[g] = s2 * inv;
      }
    }
    __syncthreads();
  }
  if (!col.on) return;
  float w[V], b[V], m[NG], rs[NG], s1[NG], s2[NG];
  col.params(o, a, w, b);
  col.of_groups(o, a.mean + n * o.q, m);
  col.of_groups(o, a.rstd + n * o.q, rs);
  col.of_groups(o, l1, s1);
  col.of_groups(o, l2, s2);
  const Tile rows(o, tile);
  const int64_t os = (int64_t)o.k * a.c, xs = o.k == 1 ? a.x_cs : os, ds = o.k == 1 ? a.dy_cs : os;
  const T* x = (const T*)a.x + n * P * a.x_cs + col.j * V;
  const T* dy = (const T*)a.dy + n * P * a.dy_cs + col.j * V;
  T* dx = (T*)a.out + n * P * a.c + col.j * V;
  if (a.act == KAD_ACT_SILU) dx_rows<T, ONE, KAD_ACT_SILU>(o, col, rows, x, xs, dy, ds, dx, os, m, rs, w, b, s1, s2);
  else if (a.act == KAD_ACT_RELU) dx_rows<T, ONE, KAD_ACT_RELU>(o, col, rows, x, xs, dy, ds, dx, os, m, rs, w, b, s1, s2);
  else dx_rows<T, ONE, KAD_ACT_NONE>(o, col, rows, x, xs, dy, ds, dx, os, m, rs, w, b, s1, s2);
}

// ---------------------------------------------------------------------------- any width
// Rows of more than 1024 vectors (C over 8192, or over 1024 and odd, for 16-bit types): one block an (image,
// group), a value at a time, the group read again for each sum.
__device__ __forceinline__ float wide_act(float z, int act) {
  return act == KAD_ACT_SILU ? act_of<KAD_ACT_SILU>(z) : act == KAD_ACT_RELU ? act_of<KAD_ACT_RELU>(z) : z;
}
__device__ __forceinline__ float wide_grad(float z, float dy, int act) {
  return act == KAD_ACT_SILU ? act_grad<KAD_ACT_SILU>(z, dy) : act == KAD_ACT_RELU ? act_grad<KAD_ACT_RELU>(z, dy) : dy;
}

// Sum over the block's 256 threads, for all of them.
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_kernel(kad_group_norm_args a) {
  __shared__ float lds[4];
  const int g = blockIdx.x, n = blockIdx.y, D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w, M = P * D;
  const T* x = (const T*)a.x + (int64_t)n * P * a.x_cs + g * D;
  T* y = (T*)a.out + (int64_t)n * P * a.c + g * D;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < M; i += 256) s += to_f32(x[i / D * a.x_cs + i % D]);
  const float mean = block_sum(s, lds) / (float)M;
  s = 0.f;
  for (int64_t i = threadIdx.x; i < M; i += 256) {
    const float d = to_f32(x[i / D * a.x_cs + i % D]) - mean;
    s += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, lds) / (float)M + a.eps);
  if (threadIdx.x == 0) {
    a.mean[n * a.groups + g] = mean;
    a.rstd[n * a.groups + g] = rstd;
  }
  for (int64_t i = threadIdx.x; i < M; i += 256) {
    const int c = (int)(i % D);
    const float w = load_param(a.weight, g * D + c, a.param_dtype, 1.f);
    const float b = load_param(a.bias, g * D + c, a.param_dtype, 0.f);
    y[i / D * a.c + c] = from_f32<T>(wide_act((to_f32(x[i / D * a.x_cs + c]) - mean) * rstd * w + b, a.act));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_dx_kernel(kad_group_norm_args a) {
  __shared__ float lds[4];
  const int g = blockIdx.x, n = blockIdx.y, D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w, M = P * D;
  const T* x = (const T*)a.x + (int64_t)n * P * a.x_cs + g * D;
  const T* dy = (const T*)a.dy + (int64_t)n * P * a.dy_cs + g * D;
  T* dx = (T*)a.out + (int64_t)n * P * a.c + g * D;
  const float mean = a.mean[n * a.groups + g], rstd = a.rstd[n * a.groups + g];
  float s1 = 0.f, s2 = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t i = threadIdx.x; i < M; i += 256) {
      const int c = (int)(i % D);
      const int64_t p = i / D;
      const float w = load_param(a.weight, g * D + c, a.param_dtype, 1.f);
      const float b = load_param(a.bias, g * D + c, a.param_dtype, 0.f);
      const float xhat = (to_f32(x[p * a.x_cs + c]) - mean) * rstd;
      const float wdz = w * wide_grad(xhat * w + b, to_f32(dy[p * a.dy_cs + c]), a.act);
      if (pass == 0) {
        s1 += wdz;
        s2 += wdz * xhat;
      } else {
        dx[p * a.c + c] = from_f32<T>(rstd * (wdz - s1 - xhat * s2));
      }
    }
    if (pass == 0) {
      s1 = block_sum(s1, lds) / (float)M;
      s2 = block_sum(s2, lds) / (float)M;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_param_kernel(kad_group_norm_args a) {
  __shared__ float lds[4];
  const int c = blockIdx.x, g = c / (a.c / a.groups);
  const int64_t P = (int64_t)a.h * a.w, rows = P * a.n;
  const float w = load_param(a.weight, c, a.param_dtype, 1.f), b = load_param(a.bias, c, a.param_dtype, 0.f);
  float dw = 0.f, db = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 256) {
    const int k = (int)(r / P) * a.groups + g;
    const float xhat = (to_f32(((const T*)a.x)[r * a.x_cs + c]) - a.mean[k]) * a.rstd[k];
    const float dz = wide_grad(xhat * w + b, to_f32(((const T*)a.dy)[r * a.dy_cs + c]), a.act);
    dw += dz * xhat;
    db += dz;
  }
  dw = block_sum(dw, lds);
  db = block_sum(db, lds);
  if (threadIdx.x == 0) {
    if (a.dweight) store_param(a.dweight, c, a.param_dtype, dw);
    if (a.dbias) store_param(a.dbias, c, a.param_dtype, db);
  }
}

// ---------------------------------------------------------------------------- host
constexpr int MOST_THREADS = 1024, MOST_GROUPS = 2048, MOST_RESIDENT = 16;

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }
int pow2_at_most(int v, int most) {
  int p = 1;
  while (2 * p <= v && 2 * p <= most) p *= 2;
  return p;
}

// Rows and vectors of columns of q groups; false where a row has too many vectors for a block.
bool lay_out(const kad_group_norm_args& a, int q, Geo& o) {
  const int V = 16 / dtype_size(a.dtype);
  const int64_t P = (int64_t)a.h * a.w;
  o = Geo{};
  o.q = q;
  o.D = a.c / a.groups;
  o.W = q * o.D;
  o.k = V / gcd(o.W, V);
  if (P / o.k > INT32_MAX - 8 * MOST_THREADS) return false;  // row numbers and the steps past them are 32-bit
  if (o.W > MOST_THREADS * V || o.k * o.W / V > MOST_THREADS || q > MOST_GROUPS) return false;
  o.S = o.k * o.W / V;
  o.full = (int)(P / o.k);
  o.tail = (int)(P % o.k) * o.W;
  return true;
}
void count_threads(Geo& o, int rows, int& threads) {
  o.R = rows < 1 ? 1 : rows;
  threads = round_up(o.R * o.S, 64);
  o.tpg = pow2_at_most(threads / o.q, 64);
  o.tpc = pow2_at_most(threads / o.W, 64);
}

// The resident kernel's layout, and the vectors a thread holds; 0: the split kernels' case.
int resident(const kad_group_norm_args& a, Geo& o, int& threads) {
  const int V = 16 / dtype_size(a.dtype), D = a.c / a.groups;
  int q = a.c % V ? a.groups : V / gcd(D, V);  // groups whose channels are whole vectors together
  if (a.groups % q) q = a.groups;
  if (!lay_out(a, q, o)) return 0;
  const int64_t vectors = (int64_t)o.full * o.S;
  if (vectors > MOST_RESIDENT * MOST_THREADS) return 0;
  const int want = (int)(vectors / 4 < 64 ? 64 : vectors / 4 < MOST_THREADS ? vectors / 4 : MOST_THREADS);
  int rows = want / o.S;
  if (rows > o.full) rows = o.full;
  count_threads(o, rows, threads);
  const int held = ceil_div(o.full, o.R);
  if (held > MOST_RESIDENT) return 0;
  const int64_t blocks = (int64_t)a.n * (a.groups / q), bytes = vectors * 16;
  if (bytes > 32 * 1024 && blocks < 128) return 0;
  const int line = 128 / (o.W * dtype_size(a.dtype));
  o.share = line > 1 && (a.groups / q) % line == 0 ? line : 1;
  return held < 1 ? 1 : held;
}

// The split kernels' layout; false: the any-width kernels' case.
bool split(const kad_group_norm_args& a, Geo& o, int& threads) {
  if (!lay_out(a, a.groups, o)) return false;
  count_threads(o, 512 / o.S < o.full ? 512 / o.S : o.full, threads);
  // About 2048 threads a CU over all images, and 4 rows a thread at least.
  int tiles = ceil_div(256 * 2048 / threads, a.n);
  const int most = ceil_div(o.full, 4 * o.R);
  if (tiles > most) tiles = most;
  if (tiles < 1) tiles = 1;
  o.rows = round_up(ceil_div(o.full, tiles), o.R);
  if (o.rows < 1) o.rows = o.R;
  o.tiles = o.full ? ceil_div(o.full, o.rows) : 1;
  return true;
}

int check_args(const kad_group_norm_args* a, const char* what) {
  KAD_CHECK_ARG(a, "%s: null pointer", what);
  KAD_CHECK_ARG(a->dtype == KAD_F32 || a->dtype == KAD_F16 || a->dtype == KAD_BF16, "%s: bad dtype", what);
  KAD_CHECK_ARG(a->param_dtype == KAD_F32 || a->param_dtype == a->dtype, "%s: param_dtype must be float or dtype", what);
  KAD_CHECK_ARG(a->n > 0 && a->h > 0 && a->w > 0 && a->c > 0 && a->groups > 0 && a->c % a->groups == 0,
                "%s: sizes must be positive and groups divide c", what);
  KAD_CHECK_ARG(a->n <= 65535 && a->c <= (1 << 20) && (int64_t)a->h * a->w <= INT32_MAX,
                "%s: at most 65535 images, 2^20 channels and 2^31 - 1 pixels", what);
  KAD_CHECK_ARG(a->act == KAD_ACT_NONE || a->act == KAD_ACT_RELU || a->act == KAD_ACT_SILU, "%s: unknown activation", what);
  KAD_CHECK_ARG(a->eps >= 0.f, "%s: eps must be >= 0", what);
  return KAD_OK;
}

int check_call(const kad_group_norm_args* a, bool backward, const char* what) {
  if (int rc = check_args(a, what)) return rc;
  KAD_CHECK_ARG(a->x && a->mean && a->rstd && (backward ? a->dy : a->out), "%s: null pointer", what);
  const int v = 16 / dtype_size(a->dtype);
  KAD_CHECK_ARG(a->x_cs == a->c || (a->x_cs > a->c && a->c % v == 0), "%s: x_cs does not fit c", what);
  KAD_CHECK_ARG(!backward || a->dy_cs == a->c || (a->dy_cs > a->c && a->c % v == 0), "%s: dy_cs does not fit c", what);
  KAD_CHECK_ARG(a->work || kad_group_norm_work_elems(a, backward) == 0, "%s: work is missing", what);
  return KAD_OK;
}

template <typename T, bool ONE>
void launch_resident(const kad_group_norm_args& a, const Geo& o, int held, int threads, hipStream_t st) {
  const int64_t blocks = (int64_t)a.n * (a.groups / o.q), unit = 8 * o.share;
  const dim3 grid((unsigned)((blocks + unit - 1) / unit * unit));
  const size_t lds = (size_t)(threads * (ONE ? 1 : VEC<T>) + 2 * o.q) * sizeof(float);
  if (held <= 4) group_norm_resident_kernel<T, ONE, 4><<<grid, threads, lds, st>>>(a, o);
  else if (held <= 10) group_norm_resident_kernel<T, ONE, 10><<<grid, threads, lds, st>>>(a, o);
  else group_norm_resident_kernel<T, ONE, MOST_RESIDENT><<<grid, threads, lds, st>>>(a, o);
}

template <typename T>
void forward(const kad_group_norm_args& a, hipStream_t st) {
  Geo o;
  int threads;
  if (const int held = resident(a, o, threads)) {
    if (o.q == 1) launch_resident<T, true>(a, o, held, threads, st);
    else launch_resident<T, false>(a, o, held, threads, st);
  } else if (split(a, o, threads)) {
    const dim3 grid(o.tiles, a.n);
    const bool one = o.q == 1 || o.D % VEC<T> == 0;
    const size_t own = 2 * o.q * sizeof(float), lds = threads * (one ? 1 : VEC<T>) * sizeof(float) + own;
    if (one) {
      group_norm_stats_kernel<T, true><<<grid, threads, lds, st>>>(a, o);
      group_norm_apply_kernel<T, true><<<grid, threads, own, st>>>(a, o);
    } else {
      group_norm_stats_kernel<T, false><<<grid, threads, lds, st>>>(a, o);
      group_norm_apply_kernel<T, false><<<grid, threads, own, st>>>(a, o);
    }
  } else {
    group_norm_wide_kernel<T><<<dim3(a.groups, a.n), 256, 0, st>>>(a);
  }
}

template <typename T, bool ONE>
void launch_backward(const kad_group_norm_args& a, const Geo& o, int threads, hipStream_t st) {
  const size_t sums = (size_t)(threads * VEC<T> + 2 * o.W) * sizeof(float);
  allow_lds(group_norm_bwd_sums_kernel<T, ONE>, sums);
  group_norm_bwd_sums_kernel<T, ONE><<<dim3(o.tiles, a.n), threads, sums, st>>>(a, o);
  const int blocks = (a.out ? a.n * o.tiles : 0) + (a.dweight || a.dbias ? ceil_div(o.W, PARAM_CHANNELS) : 0);
  const int own = 2 * o.q, waves = threads / 64 * PARAM_CHANNELS * 2;
  group_norm_dx_kernel<T, ONE><<<dim3(blocks), threads, (own > waves ? own : waves) * sizeof(float), st>>>(a, o);
}

template <typename T>
void backward(const kad_group_norm_args& a, hipStream_t st) {
  Geo o;
  int threads;
  if (!a.out && !a.dweight && !a.dbias) return;
  if (split(a, o, threads)) {
    if (o.q == 1 || o.D % VEC<T> == 0) launch_backward<T, true>(a, o, threads, st);
    else launch_backward<T, false>(a, o, threads, st);
    return;
  }
  if (a.out) group_norm_wide_dx_kernel<T><<<dim3(a.groups, a.n), 256, 0, st>>>(a);
  if (a.dweight || a.dbias) group_norm_wide_param_kernel<T><<<dim3(a.c), 256, 0, st>>>(a);
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_group_norm_work_elems(const kad_group_norm_args* a, int backward) {
  if (int rc = check_args(a, "kad_group_norm_work_elems")) return rc;
  Geo o;
  int threads;
  if (!backward && resident(*a, o, threads)) return 0;
  if (!split(*a, o, threads)) return 0;
  return (int64_t)a->n * o.tiles * 2 * (o.q + (backward ? o.W : 0));
}

extern "C" int kad_group_norm_fwd(const kad_group_norm_args* a, void* stream) {
  if (int rc = check_call(a, false, "kad_group_norm_fwd")) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) forward<float>(*a, st);
  else if (a->dtype == KAD_F16) forward<half_t>(*a, st);
  else forward<bf16_t>(*a, st);
  return check_launch("kad_group_norm_fwd");
}

extern "C" int kad_group_norm_bwd(const kad_group_norm_args* a, void* stream) {
  if (int rc = check_call(a, true, "kad_group_norm_bwd")) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) backward<float>(*a, st);
  else if (a->dtype == KAD_F16) backward<half_t>(*a, st);
  else backward<bf16_t>(*a, st);
  return check_launch("kad_group_norm_bwd");
}
