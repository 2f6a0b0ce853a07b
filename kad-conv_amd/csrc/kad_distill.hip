// Distillation from a teacher's top logits: the loss of rows of logits, and its gradient.
//
//   p = softmax(t / T) over a row's entries (t_e at class i_e), q = softmax(z / T)
//   loss = T^2 sum_e p_e (log p_e - log q[i_e]) = T^2 (sum_e e_e ((t_e - tm) - (z_i - zm)) / T / S + log(Z / S))
//          with e_e = exp((t_e - tm) / T), S = sum e, Z = sum_j exp((z_j - zm) / T), tm and zm the largest of each
//   dz_j = dloss T (q_j - sum of p_e with i_e = j)
//
// Memory bounds it: forward reads z once (the largest value and the sum in one pass), backward reads z and writes dz;
// what the classes of the entries are is looked up in z, a few values a row.
//
// Two forms, and one in 64 bits for high temperatures (below).  Up to 1024 classes a row stays in the registers of up to 64
// lanes (kad_rows.h), many rows a wave; beyond, a wave or a block walks a row, or a block a part of one where rows are few:
// forward these parts are joined in a second launch, backward each writes its own classes.
//
// 4096 rows of 32768 classes, bf16, 64 entries: 159 us a pass, 58 forward (4.7 TB/s), 5 for the join and 98 backward (5.8, part of z
// from the cache that holds the logits, past which gradients are written: 183 a pass through it).  537600 rows of 16 classes,
// fp16, 16 entries: 25 us (3.0 TB/s) and 29 (3.1).
//
// An index may come twice: its p add up, in no order that could change them: of small rows in LDS as whole numbers of
// 2^-62 (a p of 2^-38 and more keeps its 24 bits; of what is smaller, no more than 2^-62 of the row's weight is lost),
// of large ones by the entry that comes first, in the entries' order.
#include "kad_rows.h"

namespace kad {
namespace {

constexpr int MOST_WAVE = KAD_DISTILL_MOST / 4;  // entries of a row that is a wave's
constexpr int MOST_HELD = 8;  // entries of a lane in registers
constexpr int MOST_BLOCKS = 1 << 20;  // a grid has at most 2^32 threads
constexpr float INF = __builtin_inff();

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// One 32-bit multiplication: what both are at most is checked.
__device__ __forceinline__ int64_t product(uint32_t n, int64_t stride) { return (int64_t)((uint64_t)n * (uint32_t)stride); }

// A row's entries.
struct Entries {
  const kad_distill_args& a;
  int64_t t0, i0;
  __device__ __forceinline__ Entries(const kad_distill_args& args, uint32_t row) : a(args) {
    if (a.inner < a.rows) {
      const uint32_t n = row / (uint32_t)a.inner, p = row - n * (uint32_t)a.inner;
      t0 = (int64_t)n * a.t_sn + product(p, a.t_sp);
      i0 = (int64_t)n * a.i_sn + product(p, a.i_sp);
    } else {
      t0 = product(row, a.t_sp);
      i0 = product(row, a.i_sp);
    }
  }
  // Whether entry e counts; its class and logit.
  __device__ __forceinline__ bool get(int e, int& at, float& t) const {
    const int64_t i = i0 + product(e, a.i_sk), ti = t0 + product(e, a.t_sk);
    const int64_t c = a.index_bits == 32 ? (int64_t)((const int32_t*)a.index)[i] : ((const int64_t*)a.index)[i];
    t = a.teacher_dtype == KAD_F32 ? ((const float*)a.teacher)[ti]
        : a.teacher_dtype == KAD_F16 ? (float)((const half_t*)a.teacher)[ti] : (float)((const bf16_t*)a.teacher)[ti];
    at = (int)c;
    return c >= 0 && c < a.v && t != -INF;
  }
};

struct Scales {
  float inv_t, c2;  // 1 / T, log2(e) / T
  __device__ __forceinline__ explicit Scales(float t) : inv_t(1.0f / t), c2(1.44269504f / t) {}
};

// One entry's part of S and of sum e ((t - tm) - (z - zm)).  An entry that weighs nothing does not meet log q = -inf.
__device__ __forceinline__ void add_entry(float t, float tm, float z, float zm, float c2, float& s, float& d) {
  const float e = exp2_((t - tm) * c2);
  s += e;
  d += e == 0.f ? 0.f : e * ((t - tm) - (z - zm));
}
__device__ __forceinline__ float row_loss(float T, float s, float d, float zsum, const Scales& c) {
  return T * T * (d / s * c.inv_t + logf(zsum / s));
}

// A block's losses and rows that count, as a pair of work.
__device__ __forceinline__ void leave_part(const kad_distill_args& a, float loss, unsigned count) {
  __shared__ float red[32];
  if (a.reduction == KAD_REDUCE_NONE) return;
  float n = (float)count;
  loss = lanes_sum(loss, 64);
  n = lanes_sum(n, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[2 * (threadIdx.x >> 6)] = loss;
    red[2 * (threadIdx.x >> 6) + 1] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < (int)blockDim.x >> 6; ++w) {
    loss += red[2 * w];
    n += red[2 * w + 1];
  }
  a.work[2 * blockIdx.x] = loss;
  a.work[2 * blockIdx.x + 1] = n;  // a whole number under 2^24: a block has fewer rows
}

__device__ __forceinline__ void leave_row(const kad_distill_args& a, int64_t row, bool counts, float zm, float zsum, float loss) {
  if (a.stats) {
    a.stats[2 * row] = zm;
    a.stats[2 * row + 1] = counts ? 1.0f / zsum : 0.f;
  }
  if (a.reduction == KAD_REDUCE_NONE) a.loss[row] = loss;
}

__global__ __launch_bounds__(1024) void distill_join_kernel(kad_distill_args a, int parts) {
  __shared__ float red[16];
  __shared__ unsigned nred[16];
  float s = 0.f;
  unsigned n = 0;
  for (int i = threadIdx.x; i < parts; i += 1024) {
    s += a.work[2 * i];
    n += (unsigned)a.work[2 * i + 1];
  }
  s = lanes_sum(s, 64);
  for (int m = 1; m < 64; m <<= 1) n += __shfl_xor(n, m);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = s;
    nred[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) {
    s += red[w];
    n += nred[w];
  }
  const float share = n ? 1.0f / (float)n : 0.f;
  if (a.reduction == KAD_REDUCE_MEAN) {
    if (a.share) *a.share = share;
    *a.loss = n ? s / (float)n : 0.f;
  } else {
    *a.loss = s;
  }
}

// What dlogits are multiplied by, and 0 or NaN where a row's are.
__device__ __forceinline__ float row_factor(const kad_distill_args& a, int64_t row) {
  const float g = a.dloss[a.reduction == KAD_REDUCE_NONE ? row : 0];
  return g * a.temperature * (a.reduction == KAD_REDUCE_MEAN ? *a.share : 1.f);
}

// ---------------------------------------------------------------------------- rows in registers

// A lane's entries: `chunk` that follow each other, at most HELD (1 or 8); those that do not count have class -1.
template <int HELD>
struct Own {
  int at[HELD];
  float t[HELD];
  int chunk;
  __device__ __forceinline__ explicit Own(int c) : chunk(c) {}
  template <typename Q>
  __device__ __forceinline__ void logits(const Q* p) {
    constexpr int V = VEC<Q>;
#pragma unroll
    for (int i = 0; i < HELD; i += V) unpack<Q>(load_vec(p + i), t + i);
  }
  __device__ __forceinline__ void load(const Entries& en, int l) {
    const kad_distill_args& a = en.a;
    const int e = l * chunk;
    if (HELD == 1) {
      t[0] = 0.f;
      at[0] = -1;
      if (l < a.k && !en.get(l, at[0], t[0])) at[0] = -1;
      return;
    }
    if (chunk == HELD && e + HELD <= a.k && a.t_sk == 1 && a.i_sk == 1) {
      if (a.index_bits == 32) {
        const int32_t* p = (const int32_t*)a.index + en.i0 + e;
#pragma unroll
        for (int i = 0; i < HELD; ++i) at[i] = p[i];
      } else {
        const int64_t* p = (const int64_t*)a.index + en.i0 + e;
#pragma unroll
        for (int i = 0; i < HELD; ++i) at[i] = p[i] >= 0 && p[i] < a.v ? (int)p[i] : -1;
      }
      if (a.teacher_dtype == KAD_F32) logits((const float*)a.teacher + en.t0 + e);
      else if (a.teacher_dtype == KAD_F16) logits((const half_t*)a.teacher + en.t0 + e);
      else logits((const bf16_t*)a.teacher + en.t0 + e);
#pragma unroll
      for (int i = 0; i < HELD; ++i) at[i] = (uint32_t)at[i] < (uint32_t)a.v && t[i] != -INF ? at[i] : -1;
      return;
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      t[i] = 0.f;
      at[i] = -1;
      if (i < chunk && e + i < a.k && !en.get(e + i, at[i], t[i])) at[i] = -1;
    }
  }
  __device__ __forceinline__ float largest() const {
    float m = -INF;
#pragma unroll
    for (int i = 0; i < HELD; ++i) m = at[i] >= 0 ? fmaxf(m, t[i]) : m;
    return m;
  }
  __device__ __forceinline__ bool any() const {
    int m = -1;
#pragma unroll
    for (int i = 0; i < HELD; ++i) m = m > at[i] ? m : at[i];
    return m >= 0;
  }
};

// HELD: entries of a lane that stay in registers too, where a row has HELD G at most (1 or 8); 0: they are read again for each
// use.
template <typename T, int VV, int U, bool RAGGED, int HELD>
__global__ __launch_bounds__(256) void distill_small_fwd_kernel(kad_distill_args a, int G) {
  const int sub = threadIdx.x / G, l = threadIdx.x & (G - 1), per = 256 / G;
  const Place<VV, U, RAGGED> o(l, G, a.v);
  const Scales c(a.temperature);
  const uint32_t step = gridDim.x * per, rows = (uint32_t)a.rows, last = rows - 1;  // rows + step < 2^32
  Own<HELD> own(HELD == 1 ? 1 : (a.k + G - 1) / G);
  float total = 0.f;
  unsigned count = 0;
  for (uint32_t base = blockIdx.x * per; base < rows; base += step) {
    const bool live = base + sub <= last;
    const uint32_t row = live ? base + sub : last;
    const T* z = (const T*)a.logits + product(row, a.z_rs);
    Piece<T, VV> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].load(z + o.at[u]);
    const Entries en(a, row);
    float tm = -INF, any = 0.f, t;
    int at;
    float zi[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
      own.load(en, l);
#pragma unroll
      for (int i = 0; i < HELD; ++i) zi[i] = i < own.chunk && own.at[i] >= 0 ? to_f32(z[own.at[i]]) : 0.f;
      tm = own.largest();
      any = own.any() ? 1.f : 0.f;
    } else {
      for (int e = l; e < a.k; e += G)
        if (en.get(e, at, t)) {
          any = 1.f;
          tm = fmaxf(tm, t);
        }
    }
    any = lanes_max(any, G);
    tm = lanes_max(tm, G);
    float x[U][VV], zm = -INF, zsum = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u].get(x[u]);
#pragma unroll
      for (int e = 0; e < VV; ++e) zm = fmaxf(zm, x[u][e]);
    }
    zm = lanes_max(zm, G);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < VV; ++e) x[u][e] = exp2_((x[u][e] - zm) * c.c2);
      zsum += o.own(u, x[u]);
    }
    zsum = lanes_sum(zsum, G);
    float s = 0.f, d = 0.f;
    if constexpr (HELD > 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (i < own.chunk && own.at[i] >= 0) add_entry(own.t[i], tm, zi[i], zm, c.c2, s, d);
    } else {
      for (int e = l; e < a.k; e += G)
        if (en.get(e, at, t)) add_entry(t, tm, to_f32(z[at]), zm, c.c2, s, d);
    }
    s = lanes_sum(s, G);
    d = lanes_sum(d, G);
    if (l == 0 && live) {
      const float loss = any != 0.f ? row_loss(a.temperature, s, d, zsum, c) : 0.f;
      leave_row(a, row, any != 0.f, zm, zsum, loss);
      total += loss;
      count += any != 0.f;
    }
  }
  leave_part(a, total, count);
}

// Sums of weights as whole numbers of 2^-62; `unit` is 2^62 of the weights' own unit.
__device__ __forceinline__ void add_weight(unsigned long long* sum, float weight, float unit) {
  const float u = weight * unit, hi = floorf(u * 0x1p-32f), lo = __builtin_fmaf(hi, -0x1p32f, u);  // both exact
  atomicAdd(sum, (unsigned long long)(uint32_t)hi << 32 | (uint32_t)lo);
}
__device__ __forceinline__ float weight_of(unsigned long long sum) {
  return __builtin_fmaf((float)(uint32_t)(sum >> 32), 0x1p-30f, (float)(uint32_t)sum * 0x1p-62f);
}
template <typename T, int VV, int U, bool RAGGED, int HELD>
__global__ __launch_bounds__(256) void distill_small_bwd_kernel(kad_distill_args a, int G) {
  extern __shared__ unsigned long long sums[];  // [rows of the block][v]; a row's are its own wave's
  const int sub = threadIdx.x / G, l = threadIdx.x & (G - 1), per = 256 / G;
  const Place<VV, U, RAGGED> o(l, G, a.v);
  const Scales c(a.temperature);
  const uint32_t step = gridDim.x * per, rows = (uint32_t)a.rows, last = rows - 1;  // rows + step < 2^32
  Own<HELD> own(HELD == 1 ? 1 : (a.k + G - 1) / G);
  unsigned long long* mine = sums + sub * a.v;
  for (int i = threadIdx.x; i < per * a.v; i += 256) sums[i] = 0;
  __syncthreads();
  for (uint32_t base = blockIdx.x * per; base < rows; base += step) {
    const bool live = base + sub <= last;
    const uint32_t row = live ? base + sub : last;
    const T* z = (const T*)a.logits + product(row, a.z_rs);
    Piece<T, VV> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].load(z + o.at[u]);
    const float2 stats = ((const float2*)a.stats)[row];
    const float zm = stats.x, inv = stats.y, f = row_factor(a, row);
    const Entries en(a, row);
    float tm = -INF, s = 0.f, t;
    int at;
    if constexpr (HELD > 0) {
      own.load(en, l);
      tm = lanes_max(own.largest(), G);
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (i < own.chunk) {
          own.t[i] = exp2_((own.t[i] - tm) * c.c2);
          s += own.at[i] >= 0 ? own.t[i] : 0.f;
        }
    } else {
      for (int e = l; e < a.k; e += G)
        if (en.get(e, at, t)) tm = fmaxf(tm, t);
      tm = lanes_max(tm, G);
      for (int e = l; e < a.k; e += G)
        if (en.get(e, at, t)) s += exp2_((t - tm) * c.c2);
    }
    s = lanes_sum(s, G);
    const float unit = 0x1p62f / s;
    if (s == s) {
      if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
          if (i < own.chunk && own.at[i] >= 0) add_weight(mine + own.at[i], own.t[i], unit);
      } else {
        for (int e = l; e < a.k; e += G)
          if (en.get(e, at, t)) add_weight(mine + at, exp2_((t - tm) * c.c2), unit);
      }
    }
    wave_order();
    float x[U][VV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u].get(x[u]);
#pragma unroll
      for (int e = 0; e < VV; ++e) {
        const float q = exp2_((x[u][e] - zm) * c.c2) * inv, p = weight_of(mine[o.at[u] + e]);
        x[u][e] = inv == 0.f ? 0.f : f * (s == s ? q - p : s);
      }
    }
    wave_order();  // what two vectors share is read twice before it is cleared
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!o.on[u]) continue;
#pragma unroll
      for (int e = 0; e < VV; ++e) mine[o.at[u] + e] = 0;
      if (live) put<T, VV>((T*)a.dlogits + product(row, a.v) + o.at[u], x[u]);
    }
    wave_order();
  }
}

// ---------------------------------------------------------------------------- rows of any length
// A thread's largest value and sum of exp((z - largest) / T).
struct Soft {
  float m = -INF, s = 0.f;
  // The base of differences: 0 while all values are -inf, whose exponentials are 0.
  static __device__ __forceinline__ float base(float m) { return m == -INF ? 0.f : m; }
  template <int N>
  __device__ __forceinline__ void add(const float* v, float c2) {  // what does not count is -inf
    float n = m;
#pragma unroll
    for (int e = 0; e < N; ++e) n = fmaxf(n, v[e]);
    const float b = base(n);
    s *= exp2_((m - b) * c2);
    float more = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) more += exp2_((v[e] - b) * c2);
    s += more;
    m = n;
  }
  __device__ __forceinline__ void join(float om, float os, float c2) {
    const float n = fmaxf(m, om), b = base(n);
    s = s * exp2_((m - b) * c2) + os * exp2_((om - b) * c2);
    m = n;
  }
};

// A row's threads are WAVES waves of a block of four: its own place in shared memory, its threads' order.
template <int WAVES> __device__ __forceinline__ int row_lane() { return threadIdx.x & (64 * WAVES - 1); }
template <int WAVES> __device__ __forceinline__ int row_of_block() { return threadIdx.x / (64 * WAVES); }
template <int WAVES> __device__ __forceinline__ void row_barrier() {
  if constexpr (WAVES > 1) __syncthreads();
  else wave_order();
}

// Joined over a row's threads.
template <int WAVES>
__device__ __forceinline__ Soft join_row(Soft v, float c2) {
  __shared__ float red[8];
  const float m = lanes_max(v.m, 64), b = Soft::base(m);
  const float s = lanes_sum(v.s * exp2_((v.m - b) * c2), 64);
  Soft r;
  r.m = m;
  r.s = s;
  if constexpr (WAVES > 1) {
    static_assert(WAVES == 4, "a row has one wave or a block");
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red[2 * (threadIdx.x >> 6)] = m;
      red[2 * (threadIdx.x >> 6) + 1] = s;
    }
    __syncthreads();
    r.m = red[0];
    r.s = red[1];
    for (int w = 1; w < 4; ++w) r.join(red[2 * w], red[2 * w + 1], c2);
  }
  return r;
}

template <int WAVES>
__device__ __forceinline__ float sum_of_row(float v) {
  __shared__ float red[4];
  v = lanes_sum(v, 64);
  if constexpr (WAVES == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
template <int WAVES>
__device__ __forceinline__ float max_of_row(float v) {
  __shared__ float red[4];
  v = lanes_max(v, 64);
  if constexpr (WAVES == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// What the entries come to, before the row's largest logit zm is known: with zr the largest logit of the entries' classes,
// d = sum e ((t - tm) - (z_i - zr)), to which S (zm - zr) is added.
struct Teacher {
  float s, d, zr;
  bool counts;
};
template <typename T, int WAVES>
__device__ __forceinline__ Teacher teacher_of(const kad_distill_args& a, const Entries& en, const T* z, const Scales& c) {
  constexpr int MOST = KAD_DISTILL_MOST / 256;  // a wave's rows have MOST_WAVE entries at most
  float t[MOST], zi[MOST], tm = -INF, zr = -INF, any = 0.f;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int e = row_lane<WAVES>() + 64 * WAVES * i;
    t[i] = -INF;
    zi[i] = 0.f;
    int at;
    float v;
    if (e < a.k && en.get(e, at, v)) {
      t[i] = v;
      zi[i] = to_f32(z[at]);
      tm = fmaxf(tm, v);
      zr = fmaxf(zr, zi[i]);
      any = 1.f;
    }
  }
  tm = max_of_row<WAVES>(tm);
  zr = max_of_row<WAVES>(zr);
  any = max_of_row<WAVES>(any);
  if (zr == -INF) zr = 0.f;  // no entry's class has weight: d is infinite
  Teacher r{0.f, 0.f, zr, any != 0.f};
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (t[i] != -INF) add_entry(t[i], tm, zi[i], zr, c.c2, r.s, r.d);
  r.s = sum_of_row<WAVES>(r.s);
  r.d = sum_of_row<WAVES>(r.d);
  return r;
}
__device__ __forceinline__ float large_loss(const kad_distill_args& a, const Teacher& t, const Soft& soft, const Scales& c) {
  return t.counts ? row_loss(a.temperature, t.s, t.d + t.s * (soft.m - t.zr), soft.s, c) : 0.f;
}

// A thread's share of values [begin, end), which are VEC<T> at least: the next vectors are on their way while some are added,
// the first ones from the start.
template <typename T, int WAVES>
struct Stream {
  static constexpr int V = VEC<T>, AT_ONCE = 4, N = 64 * WAVES;
  const T* z;
  int begin, end;
  intx4 next[AT_ONCE];
  __device__ __forceinline__ Stream(const T* p, int from, int to) : z(p), begin(from), end(to) { fetch(row_lane<WAVES>()); }
  __device__ __forceinline__ void fetch(int j) {
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = begin + (j + u * N) * V;
      next[u] = load_vec(z + (i < end - V ? i : end - V));
    }
  }
  __device__ __forceinline__ Soft soft(float c2) {
    Soft r;
    const int l = row_lane<WAVES>(), n = (end - begin + V - 1) / V;
    for (int j = l; j - l < n; j += AT_ONCE * N) {
      float v[AT_ONCE][V];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = begin + (j + u * N) * V;
        unpack<T>(next[u], v[u]);
        if (i > end - V) {  // moved back to end with the row: its first values are another thread's, or all are
#pragma unroll
          for (int e = 0; e < V; ++e) v[u][e] = e >= i - (end - V) ? v[u][e] : -INF;
        }
      }
      fetch(j + AT_ONCE * N);
      r.add<AT_ONCE * V>(v[0], c2);
    }
    return r;
  }
};

// sum and largest of no values, or of -inf alone: the softmax is not defined
__device__ __forceinline__ Soft settled(Soft v) {
  if (!(v.s > 0.f)) v.s = __builtin_nanf("");
  return v;
}

template <typename T, int WAVES>
__global__ __launch_bounds__(256) void distill_large_fwd_kernel(kad_distill_args a) {
  constexpr int ROWS = 4 / WAVES;
  const Scales c(a.temperature);
  float total = 0.f;
  unsigned count = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + row_of_block<WAVES>(); row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    const T* z = (const T*)a.logits + row * a.z_rs;
    Stream<T, WAVES> stream(z, 0, a.v);
    const Teacher teacher = teacher_of<T, WAVES>(a, Entries(a, row), z, c);
    const Soft soft = settled(join_row<WAVES>(stream.soft(c.c2), c.c2));
    if (row_lane<WAVES>() == 0) {
      const float loss = large_loss(a, teacher, soft, c);
      leave_row(a, row, teacher.counts, soft.m, soft.s, loss);
      total += loss;
      count += teacher.counts;
    }
  }
  leave_part(a, total, count);
}

// Where rows are few: a part of one a block, [rows][parts][2] behind the blocks' losses in work.
template <typename T>
__global__ __launch_bounds__(256) void distill_part_kernel(kad_distill_args a, int part, float* softs) {
  const Scales c(a.temperature);
  const int64_t row = blockIdx.x;
  const int begin = blockIdx.y * part, end = begin + part < a.v ? begin + part : a.v;
  const Soft soft = join_row<4>(Stream<T, 4>((const T*)a.logits + row * a.z_rs, begin, end).soft(c.c2), c.c2);
  if (threadIdx.x) return;
  softs[2 * (row * gridDim.y + blockIdx.y)] = soft.m;
  softs[2 * (row * gridDim.y + blockIdx.y) + 1] = soft.s;
}
template <typename T>
__global__ __launch_bounds__(256) void distill_parts_fwd_kernel(kad_distill_args a, int parts, const float* softs) {
  const Scales c(a.temperature);
  const int64_t row = blockIdx.x;
  Soft mine;
  if ((int)threadIdx.x < parts) {
    mine.m = softs[2 * (row * parts + threadIdx.x)];
    mine.s = softs[2 * (row * parts + threadIdx.x) + 1];
  }
  const Soft soft = settled(join_row<4>(mine, c.c2));
  const Teacher teacher = teacher_of<T, 4>(a, Entries(a, row), (const T*)a.logits + row * a.z_rs, c);
  const float loss = large_loss(a, teacher, soft, c);
  if (threadIdx.x == 0) leave_row(a, row, teacher.counts, soft.m, soft.s, loss);
  leave_part(a, threadIdx.x ? 0.f : loss, threadIdx.x == 0 && teacher.counts);
}

// Rows from the last to the first: the forward pass left the last ones in the memory-side cache.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void distill_large_bwd_kernel(kad_distill_args a, int part) {
  constexpr int V = VEC<T>, AT_ONCE = 4, N = 64 * WAVES, ROWS = 4 / WAVES;
  __shared__ int at_of_rows[KAD_DISTILL_MOST];
  __shared__ float p_of_rows[KAD_DISTILL_MOST];
  const int l = row_lane<WAVES>();
  int* at_of = at_of_rows + row_of_block<WAVES>() * (KAD_DISTILL_MOST / ROWS);
  float* p_of = p_of_rows + row_of_block<WAVES>() * (KAD_DISTILL_MOST / ROWS);
  const Scales c(a.temperature);
  const int begin = blockIdx.y * part, end = begin + part < a.v ? begin + part : a.v, n = (end - begin + V - 1) / V;
  for (int64_t turn = (int64_t)blockIdx.x * ROWS + row_of_block<WAVES>(); turn < a.rows; turn += (int64_t)gridDim.x * ROWS) {
    const int64_t row = a.rows - 1 - turn;
    const T* z = (const T*)a.logits + row * a.z_rs;
    T* dz = (T*)a.dlogits + row * a.v;
    const float zm = a.stats[2 * row], inv = a.stats[2 * row + 1], f = row_factor(a, row);
    const Entries en(a, row);
    float tm = -INF, s = 0.f, t;
    int at;
    for (int e = l; e < a.k; e += N)
      if (en.get(e, at, t)) tm = fmaxf(tm, t);
    tm = max_of_row<WAVES>(tm);
    row_barrier<WAVES>();  // the row before is done with its entries
    for (int e = l; e < a.k; e += N) {
      const bool counts = en.get(e, at, t);
      const float w = counts ? exp2_((t - tm) * c.c2) : 0.f;
      at_of[e] = counts ? at : -1;
      p_of[e] = w;
      s += w;
    }
    s = sum_of_row<WAVES>(s);  // NaN, or a row that counts: 1 at least
    const float norm = 1.0f / s, scale = s == s ? f * inv : s;
    for (int j = l; j < n; j += AT_ONCE * N) {
      intx4 raw[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = begin + (j + u * N) * V;
        raw[u] = load_vec(z + (i < end - V ? i : end - V));
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = begin + (j + u * N) * V;
        float v[V];
        unpack<T>(raw[u], v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = inv == 0.f ? 0.f : scale * exp2_((v[e] - zm) * c.c2);
        if (i < end) stream_vec(dz + (i < end - V ? i : end - V), v);
      }
    }
    if (inv == 0.f) continue;
    // The entries' classes again, once all of the row's stores are done.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    row_barrier<WAVES>();
    for (int e = l; e < a.k; e += N) {
      const int mine = at_of[e];
      if (mine < begin || mine >= end) continue;
      float p = 0.f;
      bool again = false;
      for (int i = 0; i < a.k; ++i) {
        const bool same = at_of[i] == mine;
        p += same ? p_of[i] : 0.f;
        again |= same && i < e;
      }
      if (!again) dz[mine] = from_f32<T>(f * (exp2_((to_f32(z[mine]) - zm) * c.c2) * inv - p * norm));
    }
  }
}

// ---------------------------------------------------------------------------- high temperatures
// Loss and gradient are T^2 and T times what is left of logarithms and weights of order 1 that agree in all but 1 / T^2 and 1 / T
// of themselves, where the entries have nearly all of the row's weight.  So 32 bits are off by T^2 2^-24 and T 2^-24 times a
// row's sums' own errors (16 classes, all of them entries, losses of 0.04: 2e-5 of a loss at T of 4, 7e-5 at 8, 1e-2 at 100, all
// of it at 1000): up to MOST_32 that is the arithmetic above, beyond it is in 64 bits.  There too the logarithms' own size is kept
// out of the loss:
//   log(Z / S) = log1p((Z - S) / S),  Z - S from exponentials less 1, which are of the arguments' size, 1 / T:
// T 2^-53 is what the loss is off by, 1e-10 at T of 10^6.
//
// One row to 16, 64 or 256 lanes, z read twice in either direction.  64-bit exponentials and one row's loads after another bound it:
// 4096 rows of 32768 classes, bf16, 64 entries, forward 356 us (614 a value at a time; 49 in 32 bits) and backward 381 (474; 106);
// 537600 of 16, fp16, 16 entries, 177 (31) and 162 (29); of few long rows each is one block's: 4 of 150000, bf16, 201 (12) and 171
// (9).  A series for e^x - 1 in (-1, 0] took 395 and 427.
constexpr float MOST_32 = 8.f;

template <int G>
__device__ __forceinline__ float max_of_lanes(float v) {
  if constexpr (G > 64) return max_of_row<G / 64>(v);
  else return lanes_max(v, G);
}
template <int G>
__device__ __forceinline__ double sum_of_lanes(double v) {
#pragma unroll
  for (int m = 1; m < (G < 64 ? G : 64); m <<= 1) v += __shfl_xor(v, m);
  if constexpr (G > 64) {
    __shared__ double red[G / 64];
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < G / 64; ++i) v += red[i];
  }
  return v;
}

// f(class, value) of a row's values, each by one of its lanes: 16 bytes at a time where that keeps all of them busy, the next ones
// on their way.
template <typename T, int G, typename F>
__device__ __forceinline__ void each_value(const T* z, int v, F&& f) {
  constexpr int V = VEC<T>;
  const int l = threadIdx.x & (G - 1);
  if (v < G * V) {
    for (int j = l; j < v; j += G) f(j, to_f32(z[j]));
    return;
  }
  const auto at = [&](int i) { return i < v - V ? i : v - V; };  // the last vector ends with the row
  intx4 next = load_vec(z + at(l * V));
  for (int i = l * V; i < v; i += G * V) {
    float x[V];
    unpack<T>(next, x);
    next = load_vec(z + at(i + G * V));
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e >= i - at(i)) f(at(i) + e, x[e]);
  }
}

// A sum of exponentials of x <= 0: how many x are above -1, the sum of e^x - 1 over these, and that of the others' e^x.
struct Mass {
  double near = 0., less = 0., far = 0.;
  __device__ __forceinline__ void add(double x) {
    if (x > -1.) {
      near += 1.;
      less += expm1(x);
    } else {
      far += exp(x);
    }
  }
  template <int G>
  __device__ __forceinline__ void join() {
    near = sum_of_lanes<G>(near);
    less = sum_of_lanes<G>(less);
    far = sum_of_lanes<G>(far);
  }
  __device__ __forceinline__ double whole() const { return near + far + less; }
  __device__ __forceinline__ double over(const Mass& o) const { return (near - o.near) + (far - o.far) + (less - o.less); }
};

template <typename T, int G>
__global__ __launch_bounds__(256) void distill_high_fwd_kernel(kad_distill_args a) {
  constexpr int ROWS = 256 / G;
  const int l = threadIdx.x & (G - 1);
  const double heat = a.temperature, c = 1. / heat;
  float total = 0.f;
  unsigned count = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    const T* z = (const T*)a.logits + row * a.z_rs;
    const Entries en(a, row);
    float tm = -INF, zm = -INF, any = 0.f, t;
    int at;
    for (int e = l; e < a.k; e += G)
      if (en.get(e, at, t)) {
        any = 1.f;
        tm = fmaxf(tm, t);
      }
    each_value<T, G>(z, a.v, [&](int, float x) { zm = fmaxf(zm, x); });
    any = max_of_lanes<G>(any);
    tm = max_of_lanes<G>(tm);
    zm = max_of_lanes<G>(zm);
    Mass of_z, of_t;
    double d = 0.;
    each_value<T, G>(z, a.v, [&](int, float x) { of_z.add(((double)x - zm) * c); });
    for (int e = l; e < a.k; e += G)
      if (en.get(e, at, t)) {
        const double y = ((double)t - tm) * c, w = exp(y);
        of_t.add(y);
        d += w == 0. ? 0. : w * (y - ((double)to_f32(z[at]) - zm) * c);  // as in add_entry
      }
    of_z.join<G>();
    of_t.join<G>();
    d = sum_of_lanes<G>(d);
    if (l == 0) {
      const double s = of_t.whole();
      const float loss = any != 0.f ? (float)(heat * heat * (d / s + log1p(of_z.over(of_t) / s))) : 0.f;
      leave_row(a, row, any != 0.f, zm, (float)of_z.whole(), loss);
      total += loss;
      count += any != 0.f;
    }
  }
  leave_part(a, total, count);
}

template <typename T, int G>
__global__ __launch_bounds__(256) void distill_high_bwd_kernel(kad_distill_args a) {
  constexpr int ROWS = 256 / G;
  __shared__ int at_of_rows[KAD_DISTILL_MOST];
  __shared__ double p_of_rows[KAD_DISTILL_MOST];
  const int l = threadIdx.x & (G - 1), sub = threadIdx.x / G;
  int* at_of = at_of_rows + sub * (KAD_DISTILL_MOST / ROWS);
  double* p_of = p_of_rows + sub * (KAD_DISTILL_MOST / ROWS);
  const double heat = a.temperature, c = 1. / heat;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    const T* z = (const T*)a.logits + row * a.z_rs;
    T* dz = (T*)a.dlogits + row * a.v;
    const float zm = a.stats[2 * row];
    const bool live = a.stats[2 * row + 1] != 0.f;
    const double f = a.dloss[a.reduction == KAD_REDUCE_NONE ? row : 0] * heat * (a.reduction == KAD_REDUCE_MEAN ? *a.share : 1.f);
    const Entries en(a, row);
    float tm = -INF, t;
    int at;
    for (int e = l; e < a.k; e += G)
      if (en.get(e, at, t)) tm = fmaxf(tm, t);
    tm = max_of_lanes<G>(tm);
    row_barrier<(G > 64 ? G / 64 : 1)>();  // the row before is done with its entries
    double s = 0., zsum = 0.;
    for (int e = l; e < a.k; e += G) {
      const bool counts = en.get(e, at, t);
      const double w = counts ? exp(((double)t - tm) * c) : 0.;
      at_of[e] = counts ? at : -1;
      p_of[e] = w;
      s += w;
    }
    each_value<T, G>(z, a.v, [&](int, float x) { zsum += exp(((double)x - zm) * c); });
    s = sum_of_lanes<G>(s);
    zsum = sum_of_lanes<G>(zsum);
    const double inv = 1. / zsum, norm = 1. / s, scale = s == s ? f * inv : s;
    each_value<T, G>(z, a.v, [&](int j, float x) { dz[j] = from_f32<T>(live ? (float)(scale * exp(((double)x - zm) * c)) : 0.f); });
    // The entries' classes again, once all of the row's stores are done.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    row_barrier<(G > 64 ? G / 64 : 1)>();
    for (int e = l; e < a.k; e += G) {
      const int mine = at_of[e];
      if (mine < 0 || !live) continue;
      double p = 0.;
      bool again = false;
      for (int i = 0; i < a.k; ++i) {
        const bool same = at_of[i] == mine;
        p += same ? p_of[i] : 0.;
        again |= same && i < e;
      }
      if (!again) dz[mine] = from_f32<T>((float)(f * (exp(((double)to_f32(z[mine]) - zm) * c) * inv - p * norm)));
    }
  }
}

// ---------------------------------------------------------------------------- host
struct Shape {
  int lanes;       // of a row, at high temperatures; else 0
  int vv, u, G;
  int64_t blocks;  // whose losses are joined
  bool wave_rows;  // large rows: a wave each
  int part, parts; // large rows: classes of a block, blocks of a row
};

Shape shape_of(const kad_distill_args& a, bool backward) {
  Shape s{};
  if (a.temperature > MOST_32) {  // a block's rows have KAD_DISTILL_MOST entries
    s.lanes = a.v <= 256 && a.k <= 64 ? 16 : a.v <= 4096 && a.k <= 256 ? 64 : 256;
    const int64_t turns = (a.rows + 256 / s.lanes - 1) / (256 / s.lanes), most = backward ? MOST_BLOCKS : 2048;
    s.blocks = turns < most ? turns : most;
    return s;
  }
  const int v = 16 / dtype_size(a.dtype);
  // Rows in registers or not, us, 131072 rows of 1024 classes, 32 entries: forward bf16 134 and 134, fp32 140 and 129,
  // backward fp32 208 and 303, but bf16 244 and 173 (and 266 against 274 at 512 classes, twice the rows).
  const int most_small = backward && dtype_size(a.dtype) == 2 ? 512 : 1024;
  if (a.v <= most_small) {
    s.vv = a.v >= v ? v : 1;
    const int vecs = ceil_div(a.v, s.vv);
    s.u = 1;
    while (vecs > 64 * s.u) s.u *= 2;
    s.G = 1;
    while (s.G * s.u < vecs || (s.G < 64 && s.G * MOST_HELD < a.k)) s.G *= 2;
    const int64_t turns = (a.rows + 256 / s.G - 1) / (256 / s.G);
    s.blocks = turns < 2048 ? turns : 2048;
    return s;
  }
  // A row a wave, or a block, us: forward, bf16, 65536 rows of 2048 classes 76 against 263, 16384 of 8192 54 against 77;
  // backward 150 against 204 at 2048, 126 against 123 at 4096, where a block's loads reach further ahead.
  s.wave_rows = a.rows >= 1024 && a.k <= MOST_WAVE && (backward ? a.v * dtype_size(a.dtype) <= 6144 : a.v <= 8192);
  const int64_t turns = s.wave_rows ? (a.rows + 3) / 4 : a.rows, most_blocks = backward ? MOST_BLOCKS : 2048;
  s.blocks = turns < most_blocks ? turns : most_blocks;
  s.parts = 1;
  s.part = a.v;
  const int64_t wanted = backward ? 2048 : 1024;
  if (a.rows * 2 <= wanted && a.v >= 8192) {
    int64_t parts = wanted / a.rows, most = a.v / 4096;
    parts = parts < most ? parts : most;
    if (parts > 256) parts = 256;
    s.part = round_up((int)((a.v + parts - 1) / parts), v);
    // a last part shorter than a vector could not be read in one
    while (s.parts = ceil_div(a.v, s.part), s.parts > 1 && a.v - (s.parts - 1) * s.part < v) s.part += v;
  }
  return s;
}

int check_args(const kad_distill_args* a, const char* what) {
  const auto is_dtype = [](int t) { return t == KAD_F32 || t == KAD_F16 || t == KAD_BF16; };
  KAD_CHECK_ARG(a, "%s: null pointer", what);
  KAD_CHECK_ARG(is_dtype(a->dtype) && is_dtype(a->teacher_dtype), "%s: bad dtype", what);
  KAD_CHECK_ARG(a->index_bits == 32 || a->index_bits == 64, "%s: index_bits must be 32 or 64", what);
  KAD_CHECK_ARG(a->rows > 0 && a->rows <= INT32_MAX, "%s: 1 to 2^31 - 1 rows expected", what);
  KAD_CHECK_ARG(a->v > 0 && a->v <= 1 << 30, "%s: 1 to 2^30 classes expected", what);
  KAD_CHECK_ARG(a->k > 0 && a->k <= KAD_DISTILL_MOST, "%s: 1 to %d entries expected", what, KAD_DISTILL_MOST);
  KAD_CHECK_ARG(a->temperature >= 1e-6f && a->temperature <= 1e6f, "%s: temperature must lie in 1e-6 to 1e6", what);
  KAD_CHECK_ARG(a->reduction >= KAD_REDUCE_NONE && a->reduction <= KAD_REDUCE_MEAN, "%s: unknown reduction", what);
  return KAD_OK;
}

int check_call(const kad_distill_args* a, bool backward, const char* what) {
  if (int rc = check_args(a, what)) return rc;
  KAD_CHECK_ARG(a->logits && a->teacher && a->index, "%s: null pointer", what);
  KAD_CHECK_ARG(backward ? a->dloss && a->dlogits && a->stats : a->loss != nullptr, "%s: null pointer", what);
  KAD_CHECK_ARG(!backward || a->reduction != KAD_REDUCE_MEAN || a->share, "%s: share is missing", what);
  KAD_CHECK_ARG(backward || a->work || kad_distill_work_elems(a) == 0, "%s: work is missing", what);
  KAD_CHECK_ARG(a->z_rs >= a->v && a->z_rs <= INT32_MAX, "%s: z_rs does not fit v", what);
  KAD_CHECK_ARG(a->inner >= 1, "%s: inner must be at least 1", what);
  KAD_CHECK_ARG(a->t_sp <= UINT32_MAX && a->t_sk <= UINT32_MAX && a->i_sp <= UINT32_MAX && a->i_sk <= UINT32_MAX,
                "%s: strides from pixel to pixel and entry to entry must be below 2^32", what);
  KAD_CHECK_ARG(a->t_sn >= 0 && a->t_sp >= 0 && a->t_sk >= 0 && a->i_sn >= 0 && a->i_sp >= 0 && a->i_sk >= 0,
                "%s: strides must not be negative", what);
  return KAD_OK;
}

template <typename T, int VV, int U, bool RAGGED, int HELD>
void launch_small(const kad_distill_args& a, const Shape& s, bool backward, hipStream_t st) {
  if (backward) {
    if constexpr (sizeof(T) == 4 || U == 1)  // others have too many classes
      distill_small_bwd_kernel<T, VV, U, RAGGED, HELD><<<s.blocks, 256, (256 / s.G) * a.v * sizeof(unsigned long long), st>>>(a, s.G);
    return;
  }
  distill_small_fwd_kernel<T, VV, U, RAGGED, HELD><<<s.blocks, 256, 0, st>>>(a, s.G);
}

template <typename T, int VV, int U, bool RAGGED>
void launch_small(const kad_distill_args& a, const Shape& s, bool backward, hipStream_t st) {
  if (a.k <= s.G) launch_small<T, VV, U, RAGGED, 1>(a, s, backward, st);
  else if (a.k <= MOST_HELD * s.G) launch_small<T, VV, U, RAGGED, MOST_HELD>(a, s, backward, st);
  else launch_small<T, VV, U, RAGGED, 0>(a, s, backward, st);
}

template <typename T, int U>
void launch_small(const kad_distill_args& a, const Shape& s, bool backward, hipStream_t st) {
  if (a.v % VEC<T>) launch_small<T, VEC<T>, U, true>(a, s, backward, st);
  else launch_small<T, VEC<T>, U, false>(a, s, backward, st);
}

template <typename T, int G>
void launch_high(const kad_distill_args& a, const Shape& s, bool backward, hipStream_t st) {
  if (backward) distill_high_bwd_kernel<T, G><<<s.blocks, 256, 0, st>>>(a);
  else distill_high_fwd_kernel<T, G><<<s.blocks, 256, 0, st>>>(a);
}

template <typename T>
void launch(const kad_distill_args& a, bool backward, hipStream_t st) {
  const Shape s = shape_of(a, backward);
  if (s.lanes) {
    if (s.lanes == 16) launch_high<T, 16>(a, s, backward, st);
    else if (s.lanes == 64) launch_high<T, 64>(a, s, backward, st);
    else launch_high<T, 256>(a, s, backward, st);
  } else if (s.G) {
    if (s.vv == 1) launch_small<T, 1, 1, false>(a, s, backward, st);
    else if (s.u == 1) launch_small<T, 1>(a, s, backward, st);
    else if (s.u == 2) launch_small<T, 2>(a, s, backward, st);
    else if constexpr (sizeof(T) == 4) launch_small<T, 4>(a, s, backward, st);
  } else if (backward) {
    if (s.wave_rows) distill_large_bwd_kernel<T, 1><<<s.blocks, 256, 0, st>>>(a, s.part);
    else distill_large_bwd_kernel<T, 4><<<dim3(s.blocks, s.parts), 256, 0, st>>>(a, s.part);
  } else if (s.parts > 1) {
    float* softs = a.work + 2 * s.blocks;
    distill_part_kernel<T><<<dim3(a.rows, s.parts), 256, 0, st>>>(a, s.part, softs);
    distill_parts_fwd_kernel<T><<<a.rows, 256, 0, st>>>(a, s.parts, softs);
  } else {
    if (s.wave_rows) distill_large_fwd_kernel<T, 1><<<s.blocks, 256, 0, st>>>(a);
    else distill_large_fwd_kernel<T, 4><<<s.blocks, 256, 0, st>>>(a);
  }
  if (!backward && a.reduction != KAD_REDUCE_NONE) distill_join_kernel<<<1, 1024, 0, st>>>(a, (int)s.blocks);
}

int run(const kad_distill_args* a, bool backward, void* stream, const char* what) {
  if (int rc = check_call(a, backward, what)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) launch<float>(*a, backward, st);
  else if (a->dtype == KAD_F16) launch<half_t>(*a, backward, st);
  else launch<bf16_t>(*a, backward, st);
  return check_launch(what);
}

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_distill_work_elems(const kad_distill_args* a) {
  if (int rc = check_args(a, "kad_distill_work_elems")) return rc;
  const Shape s = shape_of(*a, false);
  return (a->reduction == KAD_REDUCE_NONE && s.parts <= 1 ? 0 : 2 * s.blocks) + (s.parts > 1 ? 2 * a->rows * s.parts : 0);
}

extern "C" int kad_distill_fwd(const kad_distill_args* a, void* stream) { return run(a, false, stream, "kad_distill_fwd"); }

extern "C" int kad_distill_bwd(const kad_distill_args* a, void* stream) { return run(a, true, stream, "kad_distill_bwd"); }
