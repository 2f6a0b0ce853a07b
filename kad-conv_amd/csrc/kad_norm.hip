// Group norm with an activation on NHWC maps, forward and backward.
//
//   forward   z = w (x - mean) rstd + b, y = act(z)
//   backward  dz = dy act'(z), xhat = (x - mean) rstd
//             db = sum dz, dw = sum dz xhat        over images and pixels
//             dx = rstd (w dz - (s1 + xhat s2) / M), s1 = sum w dz, s2 = sum w dz xhat over the group's M values
//
// Memory bounds it: a map is read (x; x and dy) and written (y; dx), with 15 to 20 vector operations a
// value, half of them the SiLU's exponential and reciprocal (quarter rate).
//
// Two forms.  A group of up to 32 KB stays in the registers of one block: one launch, one read.  Beyond, an
// image is cut into tiles of whole rows: one launch leaves each tile's sums, the next joins them (every block
// for itself, while its first rows are on their way) and writes the result, walking its rows backwards to meet
// what the first left in the cache before memory (an XCD's L2 is emptied between launches; forwards: 5 % more at
// 41 MB, [16, 256, 200, 200] bf16 205 and 331 us against 174 and 303).  Its stores pass the caches by, which leaves
// x in them: a bare read and a bare copy of 41 MB take 23.3 us in two launches, 19.1 us with such stores (one copy
// alone: 17.4, 12.5).
// [8, 256, 100, 100] fp16 (41 MB): 25.2 us forward (statistics 9, result 16), backward 43 us (sums 21,
// dx 22), where a bare read of x and dy takes 13.6 us, and their vector operations 11 and 12: what a block does
// beside its rows (1 us of launch, 2 of places, weights and tiles joined, 1 of sums joined) is the rest.
//
// Layout.  Threads own 16-byte vectors of V channels.  Where V does not divide C, k = V / gcd(C, V) pixels
// are taken as one row of k C channels, which V divides: a thread's vector meets the same V channels in
// every row, so its sums, weights and biases stay in registers, and any C is read in whole vectors.  A
// block of R x S threads takes R rows of S vectors at a time.
//
// Statistics.  A variance from sums of squares loses all digits where the mean is large, and a shift by the
// first value does where that one is an outlier: a thread takes means and squares about them over a few
// rows in registers and merges these (Chan's formula), so 32 bits suffice for any order of the values.
#include "kad_vec.h"

namespace kad {
namespace {

// 1 / (1 + e^-z): 0 where e^-z overflows.  For fp32 maps the quotient rounded.  For 16-bit ones the hardware's reciprocal
// alone, off by one step of 32 bits at most: 2^-12 of a step of y and dx, and in a term of dw and db no more than its
// other roundings.  Rounded, [16, 128, 200, 200] bf16 takes 90.2 and 144 us, with the reciprocal 88.0 and 137 (backward:
// both launches); [8, 256, 100, 100] fp16 26.9 and 45.0, and 25.5 and 42.9.
template <typename T>
__device__ __forceinline__ float logistic(float z) {
  return sizeof(T) == 2 ? __builtin_amdgcn_rcpf(1.0f + __expf(-z)) : sigmoidf_(z);
}

// act(z), and act'(z) times dy.
template <typename T, int ACT>
__device__ __forceinline__ float act_of(float z) {
  return ACT == KAD_ACT_SILU ? z * logistic<T>(z) : ACT == KAD_ACT_RELU ? (z > 0.f ? z : z != z ? z : 0.f) : z;
}
template <typename T, int ACT>
__device__ __forceinline__ float act_grad(float z, float dy) {
  if (ACT == KAD_ACT_SILU) {
    // z (1 - s) is taken before it meets 1: of s + y - y s, 2^-24 |z| of the slope is lost, and all of it from 2^24 on.
    const float s = logistic<T>(z), y = z * s;
    return dy * (s + y * (1.0f - s));
  }
  return ACT == KAD_ACT_RELU ? (z > 0.f ? dy : 0.f) : dy;
}

// How a block's columns (q groups of D channels, W in all) are cut into rows and vectors.
struct Geo {
  int k, S, R;    // pixels in a row, vectors in a row, rows at a time
  int full;       // whole rows of an image
  int tail;       // values of the pixels after them (fewer than k; 0 where k = 1)
  int W, q, D;
  float inv_s, inv_w, inv_d, inv_q;  // 1 / S ...
  int sets;       // resident kernel: sets of q groups
  int tpg, tpc;   // threads that join what a group, and a channel, has in a block: powers of two
  // split kernels
  int rows, tiles;  // rows of a tile (whole R), tiles of an image
  int whole, last, rest;  // the last tile's rows: last R + rest
  int parts, part_rows;   // tiles and their rows in the launch whose sums are joined
  int per;          // threads that join a group's parts
};
// x / d for x in [0, 2^16), from 1 / d: an integer division is some forty instructions.
__device__ __forceinline__ int over(int x, float inv) { return (int)(((float)x + 0.5f) * inv); }

// Count, mean and squares about the mean of some values.
struct Moments {
  float n, mean, m2;
  __device__ __forceinline__ Moments join(const Moments& o) const {
    const float all = n + o.n, f = all > 0.f ? o.n * __builtin_amdgcn_rcpf(all) : 0.f, d = o.mean - mean;
    return {all, mean + d * f, m2 + o.m2 + d * d * (n * f)};
  }
  __device__ __forceinline__ Moments from(int lane_mask) const {
    return {__shfl_xor(n, lane_mask), __shfl_xor(mean, lane_mask), __shfl_xor(m2, lane_mask)};
  }
};
struct Sums {
  float a, b;
  __device__ __forceinline__ Sums join(const Sums& o) const { return {a + o.a, b + o.b}; }
  __device__ __forceinline__ Sums from(int lane_mask) const { return {__shfl_xor(a, lane_mask), __shfl_xor(b, lane_mask)}; }
};

// Joins over runs of D of the block's values.  Thread t < active holds val[0 .. VV), which are the places
// t VV + v of a matrix of `lines` rows of W values; done(g, e) is called by one thread with what columns
// [g D, (g + 1) D) come to, joined in an order that the sizes alone decide.  `per` threads (a power of two)
// share a run.  red: VV values a thread.  Ends with a barrier.
template <int VV, typename E, typename Done>
__device__ __forceinline__ void join_runs(const E* val, int active, int lines, int W, int q, int D, int per, E* red, Done done) {
  const int t = threadIdx.x, T = blockDim.x;
  if (t < active)
#pragma unroll
    for (int v = 0; v < VV; ++v) red[t * VV + v] = val[v];
  __syncthreads();
  const int count = lines * D, l = t & (per - 1), wide = per < 64 ? per : 64;
  const float inv = __builtin_amdgcn_rcpf((float)D);
  const int shift = __builtin_ctz(per), at_once = T >> shift;
  for (int base = 0; base < q; base += at_once) {
    const int g = base + (t >> shift);
    E acc{};
    if (g < q)
      for (int i = l; i < count; i += 4 * per) {
        E f[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int e = i + u * per, p = over(e, inv);
          f[u] = E{};
          if (e < count) f[u] = red[p * (W - D) + e + g * D];
        }
        acc = acc.join(f[0].join(f[1]).join(f[2].join(f[3])));
      }
    for (int m = 1; m < wide; m <<= 1) acc = acc.join(acc.from(m));
    if (per > 64) {  // waves share a run: per is at most T / q, so one pass meets all runs
      __syncthreads();
      if ((l & 63) == 0) red[t >> 6] = acc;
      __syncthreads();
      if (l == 0 && g < q)
        for (int w = 1; w < per >> 6; ++w) acc = acc.join(red[(t >> 6) + w]);
    }
    if (l == 0 && g < q) done(g, acc);
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
    r = over(t, o.inv_s);
    j = t - r * o.S;
    on = r < o.R;
    if (!on) r = j = 0;  // reads as the first thread does, and is told apart where it counts
    c0 = first;
    ntail = o.tail - j * V;
    ntail = !on || r != 0 || ntail < 0 ? 0 : ntail > V ? V : ntail;
  }
  // Channel, among the block's, of its first value.
  __device__ __forceinline__ int channel(const Geo& o) const { return o.k == 1 ? j * V : j * V - over(j * V, o.inv_w) * o.W; }
  template <typename Q>
  __device__ __forceinline__ void param(const Geo& o, const void* p, float none, float f[V]) const {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = none;
    if (!p) return;
    Q q[V];
    if (o.k == 1) {
      __builtin_memcpy(q, (const Q*)p + c0 + j * V, sizeof(q));
    } else {
      int c = channel(o);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        q[v] = ((const Q*)p)[c];
        c = c + 1 == o.W ? 0 : c + 1;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = to_f32(q[v]);
  }
  __device__ __forceinline__ void params(const Geo& o, const kad_group_norm_args& a, float w[V], float b[V]) const {
    if (a.param_dtype == KAD_F32) {
      param<float>(o, a.weight, 1.f, w);
      param<float>(o, a.bias, 0.f, b);
    } else {
      param<T>(o, a.weight, 1.f, w);
      param<T>(o, a.bias, 0.f, b);
    }
  }
  // What p holds for the groups of its values.
  __device__ __forceinline__ void of_groups(const Geo& o, const float* p, float m[NG]) const {
    const int c = channel(o);
    int g = over(c, o.inv_d), d = c - g * o.D;
#pragma unroll
    for (int v = 0; v < NG; ++v) {
      m[v] = p[g];
      if (++d == o.D) {
        d = 0;
        g = g + 1 == o.q ? 0 : g + 1;
      }
    }
  }
};

template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void norm_vec(float x[VEC<T>], const float* mean, const float* w, const float* b) {
#pragma unroll
  for (int v = 0; v < VEC<T>; ++v) x[v] = act_of<T, ACT>((x[v] - mean[ONE ? 0 : v]) * w[v] + b[v]);
}

// ---------------------------------------------------------------------------- resident forward
constexpr int MOST_RESIDENT = 4;  // vectors a thread

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

template <typename T, bool ONE>
__global__ __launch_bounds__(1024) void group_norm_resident_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V, U = MOST_RESIDENT;
  extern __shared__ float lds[];
  const int sets = o.sets, id = (blockIdx.z * 8 + blockIdx.x) * gridDim.y + blockIdx.y;
  if (id >= a.n * sets) return;
  const int n = id / sets, set = id - n * sets;
  const Columns<T, ONE> col(o, set * o.W);
  float* mean = lds + blockDim.x * NG * 3;
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
  float w[V], b[V];
  col.params(o, a, w, b);
  // The thread's own values first, for each channel or for all; then the block's.
  int mine = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) mine += col.on && col.r + u * o.R < o.full ? 1 : 0;
  Moments mo[NG];
  float m[NG], s[NG];
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
#pragma unroll
  for (int v = 0; v < NG; ++v) {
    mo[v].n = (float)(ONE ? mine * V + col.ntail : mine + (v < col.ntail ? 1 : 0));
    m[v] = mo[v].mean = mo[v].n > 0.f ? s[v] / mo[v].n : 0.f;
    s[v] = 0.f;
  }
  if (sizeof(T) == 2) {
#pragma unroll
    for (int u = 0; u < U; ++u) repack(raw[u]);
  }
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
#pragma unroll
  for (int v = 0; v < NG; ++v) mo[v].m2 = s[v];
  if (sizeof(T) == 2) {
#pragma unroll
    for (int u = 0; u < U; ++u) repack(raw[u]);
  }
  // ONE: every thread's values are of the block's one group
  join_runs<NG>(mo, o.R * o.S, ONE ? 1 : o.R * o.k, ONE ? o.R * o.S : o.W, o.q, ONE ? o.R * o.S : o.D, o.tpg, (Moments*)lds,
                [&](int g, const Moments& e) {
                  const float r = 1.0f / sqrtf(e.m2 / e.n + a.eps);
                  mean[g] = e.mean;
                  rstd[g] = r;
                  a.mean[n * a.groups + set * o.q + g] = e.mean;
                  a.rstd[n * a.groups + set * o.q + g] = r;
                });
  col.of_groups(o, mean, m);
  if (!col.on) return;
  float rs[NG];
  col.of_groups(o, rstd, rs);
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] *= rs[ONE ? 0 : v];
  if (a.act == KAD_ACT_SILU) resident_write<T, ONE, U, KAD_ACT_SILU>(a, o, col, raw, xt, y, m, w, b);
  else if (a.act == KAD_ACT_RELU) resident_write<T, ONE, U, KAD_ACT_RELU>(a, o, col, raw, xt, y, m, w, b);
  else resident_write<T, ONE, U, KAD_ACT_NONE>(a, o, col, raw, xt, y, m, w, b);
}

// ---------------------------------------------------------------------------- split forward
// A tile's rows, R at a time: `whole` times all of them, then `rest` threads' rows, in `count` rounds.
struct Tile {
  int64_t first;
  int whole, rest, count;
  bool tail;
  __device__ __forceinline__ Tile(const Geo& o, int t) {
    tail = t == o.tiles - 1;
    first = (int64_t)t * o.rows;
    whole = tail ? o.last : o.whole;
    rest = tail ? o.rest : 0;
    count = whole + (rest ? 1 : 0);
  }
  // The i-th round of a walk from the end: the whole ones backwards, then the partial one.
  __device__ __forceinline__ int back(int i) const { return i < whole ? whole - 1 - i : i; }
};
// Pixels of the t-th tile of the first launch.
__device__ __forceinline__ int part_pixels(const Geo& o, int64_t P, int t) {
  const int64_t first = (int64_t)t * o.part_rows * o.k, next = first + (int64_t)o.part_rows * o.k;
  return (int)((t == o.parts - 1 ? P : next) - first);
}

// A map's rows as a thread meets them in a tile: an address that all threads share moves from round to round, the
// thread's own offset stays (32 bits of bytes: 512 rows of at most 2^20 elements apart).
template <typename T>
struct Lane {
  T* base;
  int64_t step;
  uint32_t off, edge;  // edge: in the last, partial round, where a thread may have no row
  template <typename C>
  __device__ __forceinline__ Lane(const Geo& o, const C& col, const Tile& rows, T* image, int64_t stride)
      : base(image + rows.first * stride), step(o.R * stride) {
    off = ((uint32_t)col.r * (uint32_t)stride + col.j * C::V) * (uint32_t)sizeof(T);
    edge = col.r < rows.rest ? off : 0;
  }
  __device__ __forceinline__ T* at(const Tile& rows, int round) const {
    return (T*)((char*)(base + round * step) + (round < rows.whole ? off : edge));
  }
};

// A tile's rounds, B at a time, the next B on their way while these are worked on.  load(i) reads the i-th;
// all(i, rows) takes B whole ones from the i-th on, some(i, rows, n) the n that are left, the partial one among them.
// Loads and stores stand outside of branches (past the end the last round is read again): with a branch around
// one, the compiler no longer knows how many are in flight and waits for all ([16, 128, 200, 200] bf16 forward
// and backward: 136 and 176 us).
template <typename Raw, int B>
struct Walk {
  int count;
  Raw next[B];
  template <typename Load>
  __device__ __forceinline__ void fetch(int i, Load load) {
#pragma unroll
    for (int k = 0; k < B; ++k) next[k] = load(i + k < count ? i + k : count - 1);
  }
  template <typename Load>
  __device__ __forceinline__ Walk(int rounds, Load load) : count(rounds) {
    if (count) fetch(0, load);
  }
  template <typename Load, typename All, typename Some>
  __device__ __forceinline__ void run(int whole, Load load, All all, Some some) {
    int i = 0;
    for (; i + B <= whole; i += B) {
      Raw now[B];
#pragma unroll
      for (int k = 0; k < B; ++k) now[k] = next[k];
      fetch(i + B, load);
      all(i, now);
    }
    if (i < count) some(i, next, count - i);
  }
};
struct Pair {
  intx4 x, d;
};

// The moments of a thread's values, for each channel or for all: as many of each.
template <int NG>
struct Running {
  float n, mean[NG], m2[NG];
  __device__ __forceinline__ Running() : n(0.f) {
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
__device__ __forceinline__ void add_rows(Running<ONE ? 1 : VEC<T>>& acc, const intx4 raw[B]) {
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

template <typename T, bool ONE, int MOST>
__global__ __launch_bounds__(MOST) void group_norm_stats_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V, B = 4;
  extern __shared__ float lds[];
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const Tile rows(o, tile);
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs;
  const Lane<const T> lane(o, col, rows, x, xs);
  Running<NG> acc;
  const auto load = [&](int i) { return load_vec(lane.at(rows, i)); };
  Walk<intx4, B> walk(rows.count, load);
  walk.run(
      rows.whole, load, [&](int, const intx4* raw) { add_rows<T, ONE, B>(acc, raw); },
      [&](int at, const intx4* raw, int left) {
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (i < left && (at + i < rows.whole || col.r < rows.rest)) add_rows<T, ONE, 1>(acc, raw + i);
      });
  // The short row's values are of a channel each, so counts differ from channel to channel.
  Moments mo[NG];
#pragma unroll
  for (int v = 0; v < NG; ++v) mo[v] = Moments{acc.n, acc.mean[v], acc.m2[v]};
  const int nt = rows.tail ? col.ntail : 0;
  if (nt) {
    float xt[V];
    load_some(x + o.full * xs + col.j * V, nt, xt);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nt) mo[ONE ? 0 : v] = mo[ONE ? 0 : v].join(Moments{1.f, xt[v], 0.f});
  }
  const bool vectors = ONE && o.q > 1;  // a group is D / V of the threads' values; the only group is all of them
  const int active = o.R * o.S, W = vectors ? o.S : ONE ? active : o.W, D = vectors ? o.D / V : ONE ? active : o.D;
  const int lines = vectors ? o.R : ONE ? 1 : o.R * o.k;
  Sums* part = (Sums*)a.work + ((int64_t)n * o.tiles + tile) * o.q;
  join_runs<NG>(mo, active, lines, W, o.q, D, o.tpg, (Moments*)lds, [&](int g, const Moments& e) { part[g] = Sums{e.mean, e.m2}; });
}

// Joins what the tiles of an image left for each group: thread t takes group t mod q of every per-th tile,
// consecutive threads consecutive groups, and quarters of the block join in LDS, in an order that the sizes alone
// decide.  The first two tiles' parts are asked for by the constructor, before the rows that a caller fetches
// meanwhile: loads return in order.
template <typename E>
struct TileJoin {
  const Sums* part;
  int per, l, g;
  Sums first[2];
  __device__ __forceinline__ TileJoin(const Geo& o, const Sums* p) : part(p) {
    const int t = threadIdx.x;
    per = o.per;
    l = over(t, o.inv_q);
    g = t - l * o.q;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (l < per && l + i * per < o.parts) first[i] = part[(l + i * per) * o.q + g];
  }
  // make(tile, part) gives a tile's E.
  template <typename Make, typename Done>
  __device__ __forceinline__ void run(const Geo& o, E* red, Make make, Done done) {
    const int t = threadIdx.x;
    if (o.q > (int)blockDim.x) {  // a group a thread, over and over
      for (int k = t; k < o.q; k += blockDim.x) {
        E acc = make(0, part[k]);
        for (int i = 1; i < o.parts; ++i) acc = acc.join(make(i, part[i * o.q + k]));
        done(k, acc);
      }
      __syncthreads();
      return;
    }
    E acc{};
    if (l < per) {
      acc = make(l, first[0]);
      if (l + per < o.parts) acc = acc.join(make(l + per, first[1]));
      for (int i = l + 2 * per; i < o.parts; i += per) acc = acc.join(make(i, part[i * o.q + g]));
    }
    red[t] = acc;
    for (int n = per; n > 1;) {  // quarters join
      const int part = (n + 3) / 4;
      __syncthreads();
      if (l < part) {
        E more[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const int from = l + (i + 1) * part;
          more[i] = E{};
          if (from < n) more[i] = red[t + (i + 1) * part * o.q];
        }
        acc = acc.join(more[0]).join(more[1].join(more[2]));
        if (part > 1) red[t] = acc;
      }
      n = part;
    }
    if (l == 0) done(g, acc);
    __syncthreads();
  }
};

template <typename T, bool ONE, int ACT, int B, typename Load>
__device__ __forceinline__ void apply_rows(const Columns<T, ONE>& col, const Tile& rows, const Lane<T>& out, const T* xt, T* yt,
                                           const float* mean, const float* w, const float* b, Walk<intx4, B>& walk, Load load) {
  constexpr int V = VEC<T>;
  const auto write = [&](int round, intx4 raw) {
    float f[V];
    unpack<T>(raw, f);
    norm_vec<T, ONE, ACT>(f, mean, w, b);
    stream_vec(out.at(rows, round), f);
  };
  walk.run(
      rows.whole, load,
      [&](int at, const intx4* raw) {
#pragma unroll
        for (int i = 0; i < B; ++i) write(rows.back(at + i), raw[i]);
      },
      [&](int at, const intx4* raw, int left) {
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (i < left && (at + i < rows.whole || col.r < rows.rest)) write(rows.back(at + i), raw[i]);
      });
  if (rows.tail && col.ntail) {
    float f[V];
    load_some(xt, col.ntail, f);
    norm_vec<T, ONE, ACT>(f, mean, w, b);
    store_some(yt, col.ntail, f);
  }
}

template <typename T, bool ONE, int MOST>
__global__ __launch_bounds__(MOST) void group_norm_apply_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V, B = 4;
  extern __shared__ float lds[];
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const Tile rows(o, tile);
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c, ys = (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs;
  T* y = (T*)a.out + n * P * a.c;
  const Lane<const T> lane(o, col, rows, x, xs);
  const Lane<T> out(o, col, rows, y, ys);
  float w[V], b[V], m[NG], rs[NG];
  TileJoin<Moments> join(o, (const Sums*)a.work + (int64_t)n * o.parts * o.q);
  col.params(o, a, w, b);
  // Backwards: what the statistics read last is in the cache before memory still.
  const auto load = [&](int i) { return load_vec(lane.at(rows, rows.back(i))); };
  Walk<intx4, B> walk(rows.count, load);
  float *mean = lds + 3 * blockDim.x, *rstd = mean + o.q;
  join.run(
      o, (Moments*)lds,
      [&](int t, const Sums& p) { return Moments{(float)part_pixels(o, P, t) * (float)o.D, p.a, p.b}; },
      [&](int g, const Moments& e) {
        const float r = 1.0f / sqrtf(e.m2 / e.n + a.eps);
        mean[g] = e.mean;
        rstd[g] = r;
        if (tile == 0) {
          a.mean[n * a.groups + g] = e.mean;
          a.rstd[n * a.groups + g] = r;
        }
      });
  if (!col.on) return;
  col.of_groups(o, mean, m);
  col.of_groups(o, rstd, rs);
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] *= rs[ONE ? 0 : v];
  const T* xt = x + o.full * xs + col.j * V;
  T* yt = y + o.full * ys + col.j * V;
  if (a.act == KAD_ACT_SILU) apply_rows<T, ONE, KAD_ACT_SILU, B>(col, rows, out, xt, yt, m, w, b, walk, load);
  else if (a.act == KAD_ACT_RELU) apply_rows<T, ONE, KAD_ACT_RELU, B>(col, rows, out, xt, yt, m, w, b, walk, load);
  else apply_rows<T, ONE, KAD_ACT_NONE, B>(col, rows, out, xt, yt, m, w, b, walk, load);
}

// ---------------------------------------------------------------------------- backward
// Two launches: the sums of dz and dz xhat of each channel in each tile, and of w times them in each group;
// then dx.  The last blocks of the second one sum the channels' parts to dw and db.
// With xm = x - mean and w times rstd: z = xm w + b, and the sums of dz and dz xm.
template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void sum_vec(const float x[VEC<T>], const float dy[VEC<T>], const float* mean, const float* w,
                                        const float* b, float* db, float* dw) {
#pragma unroll
  for (int v = 0; v < VEC<T>; ++v) {
    const float xm = x[v] - mean[ONE ? 0 : v];
    const float dz = act_grad<T, ACT>(xm * w[v] + b[v], dy[v]);
    db[v] += dz;
    dw[v] += dz * xm;
  }
}

template <typename T, bool ONE, int ACT, int B, typename Load>
__device__ __forceinline__ void sum_rows(const Columns<T, ONE>& col, const Tile& rows, const T* xt, const T* dt, const float* mean,
                                         const float* w, const float* b, float* db, float* dw, Walk<Pair, B>& walk, Load load) {
  constexpr int V = VEC<T>;
  const auto add = [&](const Pair& raw) {
    float f[V], g[V];
    unpack<T>(raw.x, f);
    unpack<T>(raw.d, g);
    sum_vec<T, ONE, ACT>(f, g, mean, w, b, db, dw);
  };
  walk.run(
      rows.whole, load,
      [&](int, const Pair* raw) {
#pragma unroll
        for (int i = 0; i < B; ++i) add(raw[i]);
      },
      [&](int at, const Pair* raw, int left) {
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (i < left && (at + i < rows.whole || col.r < rows.rest)) add(raw[i]);
      });
  if (rows.tail && col.ntail) {
    float f[V], g[V], d1[V], d2[V];
    load_some(xt, col.ntail, f);
    load_some(dt, col.ntail, g);
#pragma unroll
    for (int v = 0; v < V; ++v) d1[v] = d2[v] = 0.f;
    sum_vec<T, ONE, ACT>(f, g, mean, w, b, d1, d2);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      db[v] += v < col.ntail ? d1[v] : 0.f;
      dw[v] += v < col.ntail ? d2[v] : 0.f;
    }
  }
}

template <typename T, bool ONE, int MOST>
__global__ __launch_bounds__(MOST) void group_norm_bwd_sums_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V, B = MOST > 512 ? 2 : 4;
  extern __shared__ float lds[];
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const Tile rows(o, tile);
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t xs = o.k == 1 ? a.x_cs : (int64_t)o.k * a.c, ds = o.k == 1 ? a.dy_cs : (int64_t)o.k * a.c;
  const T* x = (const T*)a.x + n * P * a.x_cs;
  const T* dy = (const T*)a.dy + n * P * a.dy_cs;
  const Lane<const T> lx(o, col, rows, x, xs), ld(o, col, rows, dy, ds);
  float w[V], b[V], m[NG], rs[NG];
  col.params(o, a, w, b);
  col.of_groups(o, a.mean + n * o.q, m);
  col.of_groups(o, a.rstd + n * o.q, rs);
  const auto load = [&](int i) { return Pair{load_vec(lx.at(rows, i)), load_vec(ld.at(rows, i))}; };
  Walk<Pair, B> walk(rows.count, load);
  // The channels' sums, and their weights, for the groups' sums.
  Sums* red = (Sums*)lds;
  float *cb = lds + 2 * blockDim.x * V, *cw = cb + o.W, *weight = cw + o.W;
  if (col.on && col.r == 0) {
    int c = col.channel(o);
#pragma unroll
    for (int v = 0; v < V; ++v) {  // where a row is several pixels, its threads write the same weights
      weight[c] = w[v];
      c = c + 1 == o.W ? 0 : c + 1;
    }
  }
  float db[V], dw[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    db[v] = dw[v] = 0.f;
    w[v] *= rs[ONE ? 0 : v];
  }
  const T *xt = x + o.full * xs + col.j * V, *dt = dy + o.full * ds + col.j * V;
  if (a.act == KAD_ACT_SILU) sum_rows<T, ONE, KAD_ACT_SILU, B>(col, rows, xt, dt, m, w, b, db, dw, walk, load);
  else if (a.act == KAD_ACT_RELU) sum_rows<T, ONE, KAD_ACT_RELU, B>(col, rows, xt, dt, m, w, b, db, dw, walk, load);
  else sum_rows<T, ONE, KAD_ACT_NONE, B>(col, rows, xt, dt, m, w, b, db, dw, walk, load);
  Sums sums[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sums[v] = Sums{db[v], dw[v] * rs[ONE ? 0 : v]};
  const int64_t part = (int64_t)n * o.tiles + tile;
  Sums* chans = (Sums*)a.work + (int64_t)a.n * o.tiles * o.q + part * o.W;
  const bool keep = a.dweight || a.dbias;
  join_runs<V>(sums, o.R * o.S, o.R * o.k, o.W, o.W, 1, o.tpc, red, [&](int c, const Sums& e) {
    cb[c] = e.a;
    cw[c] = e.b;
    if (keep) chans[c] = e;
  });
  Sums* groups = (Sums*)a.work + part * o.q;
  const int per = o.tpg < 64 ? o.tpg : 64, l = threadIdx.x & (per - 1);
  for (int g = threadIdx.x / per; g < o.q; g += blockDim.x / per) {
    Sums acc{};
    for (int c = g * o.D + l; c < (g + 1) * o.D; c += per) acc = acc.join(Sums{weight[c] * cb[c], weight[c] * cw[c]});
    for (int k = 1; k < per; k <<= 1) acc = acc.join(acc.from(k));
    if (l == 0) groups[g] = acc;
  }
}

// dx = rstd (w dz - s1 - xhat s2) with w times rstd, c1 = rstd s1 and c2 = rstd^2 s2.
template <typename T, bool ONE, int ACT>
__device__ __forceinline__ void dx_vec(float x[VEC<T>], const float dy[VEC<T>], const float* mean, const float* w,
                                       const float* b, const float* c1, const float* c2) {
#pragma unroll
  for (int v = 0; v < VEC<T>; ++v) {
    const int g = ONE ? 0 : v;
    const float xm = x[v] - mean[g];
    const float dz = act_grad<T, ACT>(xm * w[v] + b[v], dy[v]);
    x[v] = w[v] * dz - (xm * c2[g] + c1[g]);
  }
}

template <typename T, bool ONE, int ACT, int B, typename Load>
__device__ __forceinline__ void dx_rows(const Columns<T, ONE>& col, const Tile& rows, const Lane<T>& out, const T* xt, const T* dt,
                                        T* ot, const float* mean, const float* w, const float* b, const float* c1, const float* c2,
                                        Walk<Pair, B>& walk, Load load) {
  constexpr int V = VEC<T>;
  const auto write = [&](int round, const Pair& raw) {
    float f[V], g[V];
    unpack<T>(raw.x, f);
    unpack<T>(raw.d, g);
    dx_vec<T, ONE, ACT>(f, g, mean, w, b, c1, c2);
    stream_vec(out.at(rows, round), f);
  };
  walk.run(
      rows.whole, load,
      [&](int at, const Pair* raw) {
#pragma unroll
        for (int i = 0; i < B; ++i) write(rows.back(at + i), raw[i]);
      },
      [&](int at, const Pair* raw, int left) {
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (i < left && (at + i < rows.whole || col.r < rows.rest)) write(rows.back(at + i), raw[i]);
      });
  if (rows.tail && col.ntail) {
    float f[V], g[V];
    load_some(xt, col.ntail, f);
    load_some(dt, col.ntail, g);
    dx_vec<T, ONE, ACT>(f, g, mean, w, b, c1, c2);
    store_some(ot, col.ntail, f);
  }
}

// dw and db of 16 channels from the tiles' parts: a thread in each 16 takes a channel, over rows of parts.
constexpr int PARAM_CHANNELS = 16;
__device__ __forceinline__ void param_sums(const kad_group_norm_args& a, const Geo& o, int block, float* lds) {
  const int c = block * PARAM_CHANNELS + (threadIdx.x & (PARAM_CHANNELS - 1));
  const int parts = a.n * o.parts, step = blockDim.x / PARAM_CHANNELS;
  const Sums* chans = (const Sums*)a.work + (int64_t)parts * o.q;
  float db = 0.f, dw = 0.f;
  if (c < o.W)
    for (int i = threadIdx.x / PARAM_CHANNELS; i < parts; i += step) {
      const Sums p = chans[(int64_t)i * o.W + c];
      db += p.a;
      dw += p.b;
    }
#pragma unroll
  for (int d = PARAM_CHANNELS; d < 64; d <<= 1) {
    db += __shfl_xor(db, d);
    dw += __shfl_xor(dw, d);
  }
  Sums* waves = (Sums*)lds;
  if ((threadIdx.x & 63) < PARAM_CHANNELS) waves[(threadIdx.x >> 6) * PARAM_CHANNELS + (threadIdx.x & 63)] = Sums{db, dw};
  __syncthreads();
  if (threadIdx.x < PARAM_CHANNELS && c < o.W) {
    db = dw = 0.f;
    for (int w = 0; w < blockDim.x >> 6; ++w) {
      db += waves[w * PARAM_CHANNELS + threadIdx.x].a;
      dw += waves[w * PARAM_CHANNELS + threadIdx.x].b;
    }
    if (a.dweight) store_param(a.dweight, c, a.param_dtype, dw);
    if (a.dbias) store_param(a.dbias, c, a.param_dtype, db);
  }
}

template <typename T, bool ONE, int MOST>
__global__ __launch_bounds__(MOST) void group_norm_dx_kernel(kad_group_norm_args a, Geo o) {
  constexpr int V = VEC<T>, NG = ONE ? 1 : V, B = 2;
  extern __shared__ float lds[];
  const int maps = a.out ? a.n : 0;  // the rows of blocks after the images' are the parameters'
  if ((int)blockIdx.y >= maps) return param_sums(a, o, (blockIdx.y - maps) * gridDim.x + blockIdx.x, lds);
  const int n = blockIdx.y, tile = blockIdx.x;
  const Columns<T, ONE> col(o, 0);
  const Tile rows(o, tile);
  const int64_t P = (int64_t)a.h * a.w;
  const int64_t os = (int64_t)o.k * a.c, xs = o.k == 1 ? a.x_cs : os, ds = o.k == 1 ? a.dy_cs : os;
  const T* x = (const T*)a.x + n * P * a.x_cs;
  const T* dy = (const T*)a.dy + n * P * a.dy_cs;
  T* dx = (T*)a.out + n * P * a.c;
  const Lane<const T> lx(o, col, rows, x, xs), ld(o, col, rows, dy, ds);
  const Lane<T> out(o, col, rows, dx, os);
  float w[V], b[V], m[NG], rs[NG], s1[NG], s2[NG];
  TileJoin<Sums> join(o, (const Sums*)a.work + (int64_t)n * o.parts * o.q);
  col.params(o, a, w, b);
  col.of_groups(o, a.mean + n * o.q, m);
  col.of_groups(o, a.rstd + n * o.q, rs);
  const auto load = [&](int i) {
    return Pair{load_vec(lx.at(rows, rows.back(i))), load_vec(ld.at(rows, rows.back(i)))};
  };
  Walk<Pair, B> walk(rows.count, load);
  float *l1 = lds + 2 * blockDim.x, *l2 = l1 + o.q;
  join.run(
      o, (Sums*)lds, [](int, const Sums& p) { return p; },
      [&](int g, const Sums& e) {
        const float inv = 1.0f / ((float)P * (float)o.D);
        l1[g] = e.a * inv;
        l2[g] = e.b * inv;
      });
  if (!col.on) return;
  col.of_groups(o, l1, s1);
  col.of_groups(o, l2, s2);
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] *= rs[ONE ? 0 : v];
#pragma unroll
  for (int v = 0; v < NG; ++v) {
    s1[v] *= rs[v];
    s2[v] *= rs[v] * rs[v];
  }
  const T *xt = x + o.full * xs + col.j * V, *dt = dy + o.full * ds + col.j * V;
  T* ot = dx + o.full * os + col.j * V;
  if (a.act == KAD_ACT_SILU)
    dx_rows<T, ONE, KAD_ACT_SILU, B>(col, rows, out, xt, dt, ot, m, w, b, s1, s2, walk, load);
  else if (a.act == KAD_ACT_RELU)
    dx_rows<T, ONE, KAD_ACT_RELU, B>(col, rows, out, xt, dt, ot, m, w, b, s1, s2, walk, load);
  else
    dx_rows<T, ONE, KAD_ACT_NONE, B>(col, rows, out, xt, dt, ot, m, w, b, s1, s2, walk, load);
}

// ---------------------------------------------------------------------------- any width
// Rows of more than 1024 vectors (C over 8192, or over 1024 and odd, for 16-bit types): a block takes a group's
// columns of a tile of pixels, a value a thread at a time: L threads beside each other on a pixel's D channels,
// 256 / L pixels at once.  Sums and joins as above, an (image, group) for itself.  Loads of single values bound it:
// [2, 9000, 40, 40] fp16 in 30 groups takes 138 us forward and 196 backward, 0.8 and 0.9 TB/s.
struct Wide {
  int L, at_once;     // min(D, 256), 256 / L
  float inv;          // 1 / L
  int rows, tiles;    // pixels of a tile, tiles of an image
};
struct WidePlace {
  int r, l;
  bool on;
  int64_t first, last;  // the tile's pixels
  __device__ __forceinline__ WidePlace(const Wide& o, int64_t P) {
    r = over(threadIdx.x, o.inv);
    l = threadIdx.x - r * o.L;
    on = r < o.at_once;
    first = (int64_t)blockIdx.z * o.rows;
    last = first + o.rows < P ? first + o.rows : P;
  }
};
template <typename T>
__device__ __forceinline__ float wide_act(float z, int act) {
  return act == KAD_ACT_SILU ? act_of<T, KAD_ACT_SILU>(z) : act == KAD_ACT_RELU ? act_of<T, KAD_ACT_RELU>(z) : z;
}
template <typename T>
__device__ __forceinline__ float wide_grad(float z, float dy, int act) {
  return act == KAD_ACT_SILU ? act_grad<T, KAD_ACT_SILU>(z, dy) : act == KAD_ACT_RELU ? act_grad<T, KAD_ACT_RELU>(z, dy) : dy;
}

// What the block's 256 threads have, joined, for all of them.
template <typename E>
__device__ __forceinline__ E block_join(E e) {
  __shared__ E waves[4];
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) e = e.join(e.from(m));
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = e;
  __syncthreads();
  e = waves[0].join(waves[1]).join(waves[2].join(waves[3]));
  __syncthreads();
  return e;
}
// The parts that the tiles of an (image, group) left, joined, for all threads.
template <typename E, typename Make>
__device__ __forceinline__ E wide_join(const kad_group_norm_args& a, const Wide& o, int n, int g, Make make) {
  E e{};
  for (int t = threadIdx.x; t < o.tiles; t += 256) e = e.join(make(t, ((const Sums*)a.work)[((int64_t)n * o.tiles + t) * a.groups + g]));
  return block_join(e);
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_stats_kernel(kad_group_norm_args a, Wide o) {
  const int g = blockIdx.x, n = blockIdx.y, D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w;
  const WidePlace at(o, P);
  const T* x = (const T*)a.x + n * P * a.x_cs + (int64_t)g * D;
  Moments acc{};
  if (at.on)
    for (int64_t p = at.first + at.r; p < at.last; p += o.at_once)
      for (int d = at.l; d < D; d += 4 * o.L) {
        float v[4], n4 = 0.f, s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = d + i * o.L < D;
          v[i] = to_f32(x[p * a.x_cs + (in ? d + i * o.L : d)]);
          n4 += in ? 1.f : 0.f;
          s += in ? v[i] : 0.f;
        }
        s /= n4;
#pragma unroll
        for (int i = 0; i < 4; ++i) q += d + i * o.L < D ? (v[i] - s) * (v[i] - s) : 0.f;
        acc = acc.join(Moments{n4, s, q});
      }
  acc = block_join(acc);
  if (threadIdx.x == 0) ((Sums*)a.work)[((int64_t)n * o.tiles + blockIdx.z) * a.groups + g] = Sums{acc.mean, acc.m2};
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_apply_kernel(kad_group_norm_args a, Wide o) {
  const int g = blockIdx.x, n = blockIdx.y, D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w;
  const WidePlace at(o, P);
  const Moments e = wide_join<Moments>(a, o, n, g, [&](int t, const Sums& p) {
    const int64_t left = P - (int64_t)t * o.rows;
    return Moments{(float)(left < o.rows ? left : o.rows) * (float)D, p.a, p.b};
  });
  const float mean = e.mean, rstd = 1.0f / sqrtf(e.m2 / e.n + a.eps);
  if (blockIdx.z == 0 && threadIdx.x == 0) {
    a.mean[n * a.groups + g] = mean;
    a.rstd[n * a.groups + g] = rstd;
  }
  if (!at.on) return;
  const T* x = (const T*)a.x + n * P * a.x_cs + (int64_t)g * D;
  T* y = (T*)a.out + n * P * a.c + (int64_t)g * D;
  for (int d = at.l; d < D; d += o.L) {
    const float w = load_param(a.weight, g * D + d, a.param_dtype, 1.f) * rstd;
    const float b = load_param(a.bias, g * D + d, a.param_dtype, 0.f);
#pragma unroll 4
    for (int64_t p = at.first + at.r; p < at.last; p += o.at_once)
      y[p * a.c + d] = from_f32<T>(wide_act<T>((to_f32(x[p * a.x_cs + d]) - mean) * w + b, a.act));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_sums_kernel(kad_group_norm_args a, Wide o) {
  __shared__ Sums red[256];
  const int g = blockIdx.x, n = blockIdx.y, D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w, part = (int64_t)n * o.tiles + blockIdx.z;
  const WidePlace at(o, P);
  const float mean = a.mean[n * a.groups + g], rstd = a.rstd[n * a.groups + g];
  const T* x = (const T*)a.x + n * P * a.x_cs + (int64_t)g * D;
  const T* dy = (const T*)a.dy + n * P * a.dy_cs + (int64_t)g * D;
  Sums* chans = (Sums*)a.work + (int64_t)a.n * o.tiles * a.groups + part * a.c + (int64_t)g * D;
  const bool keep = a.dweight || a.dbias;
  Sums group{};
  for (int d0 = 0; d0 < D; d0 += o.L) {  // L channels at a time, their pixels shared by 256 / L threads
    const int d = d0 + at.l;
    Sums s{};
    float w = 0.f;
    if (at.on && d < D) {
      w = load_param(a.weight, g * D + d, a.param_dtype, 1.f);
      const float b = load_param(a.bias, g * D + d, a.param_dtype, 0.f);
#pragma unroll 4
      for (int64_t p = at.first + at.r; p < at.last; p += o.at_once) {
        const float xhat = (to_f32(x[p * a.x_cs + d]) - mean) * rstd;
        const float dz = wide_grad<T>(xhat * w + b, to_f32(dy[p * a.dy_cs + d]), a.act);
        s.a += dz;
        s.b += dz * xhat;
      }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (at.on && at.r == 0 && d < D) {
      for (int r = 1; r < o.at_once; ++r) s = s.join(red[threadIdx.x + r * o.L]);
      if (keep) chans[d] = s;
      group = group.join(Sums{w * s.a, w * s.b});
    }
    __syncthreads();
  }
  group = block_join(group);
  if (threadIdx.x == 0) ((Sums*)a.work)[part * a.groups + g] = group;
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_wide_dx_kernel(kad_group_norm_args a, Wide o) {
  const int g = blockIdx.x, n = blockIdx.y, D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w;
  const WidePlace at(o, P);
  const Sums e = wide_join<Sums>(a, o, n, g, [](int, const Sums& p) { return p; });
  const float mean = a.mean[n * a.groups + g], rstd = a.rstd[n * a.groups + g], inv = 1.0f / ((float)P * (float)D);
  const float s1 = e.a * inv, s2 = e.b * inv;
  if (!at.on) return;
  const T* x = (const T*)a.x + n * P * a.x_cs + (int64_t)g * D;
  const T* dy = (const T*)a.dy + n * P * a.dy_cs + (int64_t)g * D;
  T* dx = (T*)a.out + n * P * a.c + (int64_t)g * D;
  for (int d = at.l; d < D; d += o.L) {
    const float w = load_param(a.weight, g * D + d, a.param_dtype, 1.f);
    const float b = load_param(a.bias, g * D + d, a.param_dtype, 0.f);
#pragma unroll 4
    for (int64_t p = at.first + at.r; p < at.last; p += o.at_once) {
      const float xhat = (to_f32(x[p * a.x_cs + d]) - mean) * rstd;
      const float dz = wide_grad<T>(xhat * w + b, to_f32(dy[p * a.dy_cs + d]), a.act);
      dx[p * a.c + d] = from_f32<T>(rstd * (w * dz - s1 - xhat * s2));
    }
  }
}

__global__ __launch_bounds__(256) void group_norm_wide_param_kernel(kad_group_norm_args a, Geo o) {
  __shared__ float lds[4 * PARAM_CHANNELS * 2];
  param_sums(a, o, blockIdx.x, lds);
}

// ---------------------------------------------------------------------------- host
constexpr int MOST_THREADS = 1024, MOST_GROUPS = 2048;

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
  o.inv_s = 1.0f / (float)o.S;
  o.inv_w = 1.0f / (float)o.W;
  o.inv_d = 1.0f / (float)o.D;
  o.inv_q = 1.0f / (float)o.q;
  o.full = (int)(P / o.k);
  o.tail = (int)(P % o.k) * o.W;
  return true;
}
void count_threads(Geo& o, int rows, int& threads) {
  o.R = rows < 1 ? 1 : rows;
  threads = round_up(o.R * o.S, 64);
  o.tpg = pow2_at_most(threads / o.q, threads);
  o.tpc = pow2_at_most(threads / o.W, threads);
}

// Blocks go round the 8 XCDs by their number: those whose sets share 128-byte lines of a pixel are kept on one.
dim3 resident_grid(const kad_group_norm_args& a, const Geo& o) {
  const int line = 128 / (o.W * dtype_size(a.dtype)), share = line > 1 && o.sets % line == 0 ? line : 1;
  const int64_t blocks = (int64_t)a.n * o.sets;
  return dim3(8, share, (unsigned)((blocks + 8 * share - 1) / (8 * share)));
}

// The resident kernel's layout; false: the split kernels' case.
bool resident(const kad_group_norm_args& a, Geo& o, int& threads) {
  const int V = 16 / dtype_size(a.dtype), D = a.c / a.groups;
  int q = a.c % V ? a.groups : V / gcd(D, V);  // groups whose channels are whole vectors together
  if (a.groups % q) q = a.groups;
  if (!lay_out(a, q, o)) return false;
  // One launch, but a block's columns of D or few channels are pieces of lines that other blocks fetch too, and
  // one CU reads them.  One launch against the split kernels' two, in us: up to 32 KB a block 4.8 against 8.1
  // ([1, 64, 20, 20] fp16), 4.5 against 7.4 ([2, 48, 13, 17] fp32), 13 against 15 ([16, 512, 25, 25] in 16 groups); at
  // 64 KB 11.1 against 8.9 with 8 blocks, 13.8 against 17.0 with 256; at 256 KB twice theirs.  So the limit is where one
  // launch wins whatever the number of blocks; what many blocks of 33 to 64 KB would gain by it is left.
  if ((int64_t)o.full * o.S * 16 > 32 * 1024) return false;
  int rows = ceil_div(o.full, MOST_RESIDENT);
  if (rows < ceil_div(64, o.S)) rows = ceil_div(64, o.S);
  if (rows > o.full) rows = o.full;
  if (rows * o.S > MOST_THREADS) return false;
  count_threads(o, rows, threads);
  o.sets = a.groups / q;
  return resident_grid(a, o).z <= 65535;  // a grid's layers
}

// Cuts an image's rows into about `tiles` tiles.
void cut(Geo& o, int tiles) {
  o.rows = round_up(ceil_div(o.full, tiles), o.R);
  if (o.rows < 1) o.rows = o.R;
  o.tiles = o.full ? ceil_div(o.full, o.rows) : 1;
  o.whole = o.rows / o.R;
  o.last = (o.full - (o.tiles - 1) * o.rows) / o.R;
  o.rest = (o.full - (o.tiles - 1) * o.rows) % o.R;
}

// The split kernels' layouts, of the launch that sums and of the one that writes; false: the any-width kernels' case.
bool split(const kad_group_norm_args& a, bool backward, Geo& sums, Geo& writes, int& threads) {
  Geo o;
  if (!lay_out(a, a.groups, o)) return false;
  // One block of 512 threads a CU: what a block does beside its rows (places, weights, the join of what it and
  // others left) is microseconds, so that more blocks lose more than their loads in flight gain ([8, 256, 100, 100]
  // fp16, forward and backward: 27 and 46 us where this was tried; 32 and 54 with two blocks a CU, 44 and 70 with
  // four; 27 and 47 with 256 threads).  Threads of under 8 rows are halved ([3, 86, 67, 41] fp32: 9.6 and 12.0 us
  // against 10.4 and 12.7).
  const int most = (int64_t)a.n * o.full * o.S < 8 * 256 * 512 ? 256 : 512;
  count_threads(o, most / o.S < o.full ? most / o.S : o.full, threads);
  int tiles = a.n < 256 ? 256 / a.n : 1;
  // An image of over 256 rows a thread and tile is cut finer, up to 256 tiles, whatever the batch.
  const int64_t fine = o.full / (256 * o.R);
  if (tiles < fine) tiles = fine < 256 ? (int)fine : 256;
  const int least = ceil_div(o.full, 4 * o.R);  // 4 rows a thread
  if (tiles > least) tiles = least;
  if (tiles < 1) tiles = 1;
  sums = writes = o;
  cut(writes, tiles);
  // Every block of the second launch joins all parts of its image: few images with many groups are summed in fewer
  // tiles than they are written in, 8 parts a thread to join forward and 16 backward, where the sums take longer
  // ([1, 384, 18, 166] fp32 in 32 groups: 12.4 and 16.3 us, 19.0 and 21.0 with as many parts as tiles, 14.3 and 22.8
  // with 64 rows a thread; [1, 128, 100, 100] fp16: 13.4 and 19.1, 15.4 and 19.2, 18.5 and 33.7).
  int parts = (backward ? 16 : 8) * threads / o.q;
  const int busy = ceil_div(o.full, 32 * o.R);
  if (parts < busy) parts = busy;
  cut(sums, parts < tiles ? parts : tiles);
  sums.parts = writes.parts = sums.tiles;
  sums.part_rows = writes.part_rows = sums.rows;
  writes.per = threads / o.q < 1 ? 1 : threads / o.q < writes.parts ? threads / o.q : writes.parts;
  return true;
}

// The any-width kernels' layout: four blocks a CU over all images and groups, 16 pixels a thread at least.
Wide wide(const kad_group_norm_args& a) {
  const int D = a.c / a.groups;
  const int64_t P = (int64_t)a.h * a.w;
  Wide o;
  o.L = D < 256 ? D : 256;
  o.at_once = 256 / o.L;
  o.inv = 1.0f / (float)o.L;
  const int64_t cells = (int64_t)a.n * a.groups, least = 16 * o.at_once;
  int64_t tiles = cells < 1024 ? 1024 / cells : 1;
  if (tiles * least > P) tiles = (P + least - 1) / least;
  o.rows = (int)((P + tiles - 1) / tiles);
  o.tiles = (int)((P + o.rows - 1) / o.rows);
  return o;
}

int check_args(const kad_group_norm_args* a, const char* what) {
  KAD_CHECK_ARG(a, "%s: null pointer", what);
  KAD_CHECK_ARG(a->dtype == KAD_F32 || a->dtype == KAD_F16 || a->dtype == KAD_BF16, "%s: bad dtype", what);
  KAD_CHECK_ARG(a->param_dtype == KAD_F32 || a->param_dtype == a->dtype, "%s: param_dtype must be float or dtype", what);
  KAD_CHECK_ARG(a->n > 0 && a->h > 0 && a->w > 0 && a->c > 0 && a->groups > 0 && a->c % a->groups == 0,
                "%s: sizes must be positive and groups divide c", what);
  KAD_CHECK_ARG(a->n <= 65535 && a->c <= (1 << 20) && (int64_t)a->h * a->w <= INT32_MAX,
                "%s: at most 65535 images, 2^20 channels and 2^31 - 1 pixels", what);
  // (image, group) pairs are numbered in 32 bits, up to 64 blocks past the last
  KAD_CHECK_ARG((int64_t)a->n * a->groups <= (1 << 30), "%s: at most 2^30 groups in all images together", what);
  KAD_CHECK_ARG(a->act == KAD_ACT_NONE || a->act == KAD_ACT_RELU || a->act == KAD_ACT_SILU, "%s: unknown activation", what);
  KAD_CHECK_ARG(a->eps >= 0.f, "%s: eps must be >= 0", what);
  return KAD_OK;
}

int check_call(const kad_group_norm_args* a, bool backward, const char* what) {
  if (int rc = check_args(a, what)) return rc;
  KAD_CHECK_ARG(a->x && a->mean && a->rstd && (backward ? a->dy : a->out), "%s: null pointer", what);
  const int v = 16 / dtype_size(a->dtype);
  KAD_CHECK_ARG(a->x_cs <= (1 << 20) && (!backward || a->dy_cs <= (1 << 20)), "%s: pixels lie at most 2^20 elements apart", what);
  KAD_CHECK_ARG(a->x_cs == a->c || (a->x_cs > a->c && a->c % v == 0), "%s: x_cs does not fit c", what);
  KAD_CHECK_ARG(!backward || a->dy_cs == a->c || (a->dy_cs > a->c && a->c % v == 0), "%s: dy_cs does not fit c", what);
  KAD_CHECK_ARG(a->work || kad_group_norm_work_elems(a, backward) == 0, "%s: work is missing", what);
  return KAD_OK;
}

template <typename T, bool ONE>
void launch_resident(const kad_group_norm_args& a, const Geo& o, int threads, hipStream_t st) {
  const size_t lds = threads * (ONE ? 1 : VEC<T>) * sizeof(Moments) + 2 * o.q * sizeof(float);
  allow_lds(group_norm_resident_kernel<T, ONE>, lds);
  group_norm_resident_kernel<T, ONE><<<resident_grid(a, o), threads, lds, st>>>(a, o);
}

template <typename T, bool ONE, int MOST>
void launch_split(const kad_group_norm_args& a, const Geo& first, const Geo& o, int threads, hipStream_t st) {
  const size_t stats = threads * (ONE ? 1 : VEC<T>) * sizeof(Moments);
  allow_lds(group_norm_stats_kernel<T, ONE, MOST>, stats);
  group_norm_stats_kernel<T, ONE, MOST><<<dim3(first.tiles, a.n), threads, stats, st>>>(a, first);
  group_norm_apply_kernel<T, ONE, MOST><<<dim3(o.tiles, a.n), threads, threads * sizeof(Moments) + 2 * o.q * sizeof(float), st>>>(a, o);
}

template <typename T>
void forward(const kad_group_norm_args& a, hipStream_t st) {
  Geo o, first;
  int threads;
  if (resident(a, o, threads)) {
    if (o.q == 1) launch_resident<T, true>(a, o, threads, st);
    else launch_resident<T, false>(a, o, threads, st);
  } else if (split(a, false, first, o, threads)) {
    const bool one = o.q == 1 || o.D % VEC<T> == 0;
    if (one) threads > 512 ? launch_split<T, true, 1024>(a, first, o, threads, st) : launch_split<T, true, 512>(a, first, o, threads, st);
    else threads > 512 ? launch_split<T, false, 1024>(a, first, o, threads, st) : launch_split<T, false, 512>(a, first, o, threads, st);
  } else {
    const Wide v = wide(a);
    group_norm_wide_stats_kernel<T><<<dim3(a.groups, a.n, v.tiles), 256, 0, st>>>(a, v);
    group_norm_wide_apply_kernel<T><<<dim3(a.groups, a.n, v.tiles), 256, 0, st>>>(a, v);
  }
}

template <typename T, bool ONE, int MOST>
void launch_backward(const kad_group_norm_args& a, const Geo& first, const Geo& o, int threads, hipStream_t st) {
  const size_t sums = threads * VEC<T> * sizeof(Sums) + 3 * o.W * sizeof(float);
  allow_lds(group_norm_bwd_sums_kernel<T, ONE, MOST>, sums);
  group_norm_bwd_sums_kernel<T, ONE, MOST><<<dim3(first.tiles, a.n), threads, sums, st>>>(a, first);
  const int params = a.dweight || a.dbias ? ceil_div(ceil_div(o.W, PARAM_CHANNELS), o.tiles) : 0;
  const int waves = threads / 64 * PARAM_CHANNELS * 2, join = 2 * threads + 2 * o.q;
  if (a.out && a.n + params > 65535) {  // more rows of blocks than a grid has
    kad_group_norm_args only = a;
    only.out = nullptr;
    group_norm_dx_kernel<T, ONE, MOST><<<dim3(o.tiles, params), threads, (join > waves ? join : waves) * sizeof(float), st>>>(only, o);
    group_norm_dx_kernel<T, ONE, MOST><<<dim3(o.tiles, a.n), threads, (join > waves ? join : waves) * sizeof(float), st>>>(a, o);
    return;
  }
  group_norm_dx_kernel<T, ONE, MOST><<<dim3(o.tiles, (a.out ? a.n : 0) + params), threads, (join > waves ? join : waves) * sizeof(float), st>>>(a, o);
}

template <typename T>
void backward(const kad_group_norm_args& a, hipStream_t st) {
  Geo o, first;
  int threads;
  if (!a.out && !a.dweight && !a.dbias) return;
  if (split(a, true, first, o, threads)) {
    const bool one = o.q == 1 || o.D % VEC<T> == 0;
    if (one) threads > 512 ? launch_backward<T, true, 1024>(a, first, o, threads, st) : launch_backward<T, true, 512>(a, first, o, threads, st);
    else threads > 512 ? launch_backward<T, false, 1024>(a, first, o, threads, st) : launch_backward<T, false, 512>(a, first, o, threads, st);
    return;
  }
  const Wide v = wide(a);
  const dim3 grid(a.groups, a.n, v.tiles);
  group_norm_wide_sums_kernel<T><<<grid, 256, 0, st>>>(a, v);
  if (a.out) group_norm_wide_dx_kernel<T><<<grid, 256, 0, st>>>(a, v);
  if (a.dweight || a.dbias) {
    o = Geo{};
    o.q = a.groups;
    o.W = a.c;
    o.parts = v.tiles;
    group_norm_wide_param_kernel<<<dim3(ceil_div(a.c, PARAM_CHANNELS)), 256, 0, st>>>(a, o);
  }
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_group_norm_work_elems(const kad_group_norm_args* a, int backward) {
  if (int rc = check_args(a, "kad_group_norm_work_elems")) return rc;
  Geo o, first;
  int threads;
  if (!backward && resident(*a, o, threads)) return 0;
  if (!split(*a, backward, first, o, threads)) return (int64_t)a->n * wide(*a).tiles * 2 * (a->groups + (backward ? a->c : 0));
  return (int64_t)a->n * o.parts * 2 * (o.q + (backward ? o.W : 0));
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
