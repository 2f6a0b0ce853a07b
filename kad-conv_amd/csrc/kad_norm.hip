// Group norm with an activation on NHWC maps, forward and backward: one block an (image, group), the
// group's values read once for each sum and once for the result.
//
//   forward   z = w (x - mean) rstd + b, y = act(z)
//   backward  dz = dy act'(z), xhat = (x - mean) rstd
//             db = sum dz, dw = sum dz xhat        over images and pixels
//             dx = rstd (w dz - (s1 + xhat s2) / M), s1 = sum w dz, s2 = sum w dz xhat over the group's M values
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

// act(z), and act'(z) times dy.
__device__ __forceinline__ float act_of(float z, int act) {
  return act == KAD_ACT_SILU ? z * sigmoidf_(z) : act == KAD_ACT_RELU ? (z > 0.f ? z : z != z ? z : 0.f) : z;
}
__device__ __forceinline__ float act_grad(float z, float dy, int act) {
  if (act == KAD_ACT_SILU) {
    const float s = sigmoidf_(z);
    return dy * s * (1.f + z * (1.f - s));
  }
  return act == KAD_ACT_RELU ? (z > 0.f ? dy : 0.f) : dy;
}

// Sum over the block's 256 threads, for all of them.
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_fwd_kernel(kad_group_norm_args a) {
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
    y[i / D * a.c + c] = from_f32<T>(act_of((to_f32(x[i / D * a.x_cs + c]) - mean) * rstd * w + b, a.act));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void group_norm_dx_kernel(kad_group_norm_args a) {
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
      const float wdz = w * act_grad(xhat * w + b, to_f32(dy[p * a.dy_cs + c]), a.act);
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
__global__ __launch_bounds__(256) void group_norm_dparam_kernel(kad_group_norm_args a) {
  __shared__ float lds[4];
  const int c = blockIdx.x, g = c / (a.c / a.groups);
  const int64_t P = (int64_t)a.h * a.w, rows = P * a.n;
  const float w = load_param(a.weight, c, a.param_dtype, 1.f), b = load_param(a.bias, c, a.param_dtype, 0.f);
  float dw = 0.f, db = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 256) {
    const int k = (int)(r / P) * a.groups + g;
    const float xhat = (to_f32(((const T*)a.x)[r * a.x_cs + c]) - a.mean[k]) * a.rstd[k];
    const float dz = act_grad(xhat * w + b, to_f32(((const T*)a.dy)[r * a.dy_cs + c]), a.act);
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

}  // namespace
}  // namespace kad

using namespace kad;

extern "C" int64_t kad_group_norm_work_elems(const kad_group_norm_args* a, int backward) {
  (void)backward;
  if (int rc = check_args(a, "kad_group_norm_work_elems")) return rc;
  return 0;
}

extern "C" int kad_group_norm_fwd(const kad_group_norm_args* a, void* stream) {
  if (int rc = check_call(a, false, "kad_group_norm_fwd")) return rc;
  const dim3 grid(a->groups, a->n);
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) group_norm_fwd_kernel<float><<<grid, 256, 0, st>>>(*a);
  else if (a->dtype == KAD_F16) group_norm_fwd_kernel<half_t><<<grid, 256, 0, st>>>(*a);
  else group_norm_fwd_kernel<bf16_t><<<grid, 256, 0, st>>>(*a);
  return check_launch("kad_group_norm_fwd");
}

template <typename T>
static void backward(const kad_group_norm_args& a, hipStream_t st) {
  if (a.out) group_norm_dx_kernel<T><<<dim3(a.groups, a.n), 256, 0, st>>>(a);
  if (a.dweight || a.dbias) group_norm_dparam_kernel<T><<<dim3(a.c), 256, 0, st>>>(a);
}

extern "C" int kad_group_norm_bwd(const kad_group_norm_args* a, void* stream) {
  if (int rc = check_call(a, true, "kad_group_norm_bwd")) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == KAD_F32) backward<float>(*a, st);
  else if (a->dtype == KAD_F16) backward<half_t>(*a, st);
  else backward<bf16_t>(*a, st);
  return check_launch("kad_group_norm_bwd");
}
