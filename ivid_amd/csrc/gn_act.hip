// GroupNorm + FiLM + activation + dropout over channels-last tensors, forward and backward (include/ivid_hip.h ivid_gn_act_*).
//
//   xc = x - mean, xhat = xc * rstd, u = xhat * gamma + beta, v = u * (1 + s) + t, y = drop(act(v))
//   gv = drop(dy) * act'(v);  per (n, c): A = sum_p gv, B = sum_p gv * xhat
//   dshift = A, dscale = gamma * B + beta * A, dgamma = sum_n (1 + s) * B, dbeta = sum_n (1 + s) * A
//   with g = gv * gamma * (1 + s), M = HW * C / G:  dx = rstd * (g - sum(g) / M - xhat * sum(g * xhat) / M), sums over the group
#include <math.h>
#include "common.h"
#include "internal.h"
#include "philox.h"

int ivid_drop_rng(double p, unsigned long long seed, unsigned long long stream_id, const unsigned long long* rng, DropRng* out);

namespace {
constexpr int NT = 256;

struct GnArgs {
  const char *src0, *src1;
  long long ld0, sn0, ld1, sn1;
  int HW, C0, C, G, Cg, act, film_kind;  // film_kind: 0 none, 1 fp32, 2 the tensors' type
  const float *gamma, *beta;
  const char* film;
  long long film_ld;
  float eps;
  bool drop;
  DropRng rng;
};

template <typename T>
__device__ __forceinline__ float film_at(const GnArgs& a, long long i) {
  return a.film_kind == 1 ? ((const float*)a.film)[i] : (float)((const T*)a.film)[i];
}
template <typename T>
__device__ __forceinline__ float load_x(const GnArgs& a, int n, int p, int c) {
  return c < a.C0 ? (float)((const T*)a.src0)[n * a.sn0 + p * a.ld0 + c] : (float)((const T*)a.src1)[n * a.sn1 + p * a.ld1 + c - a.C0];
}

// a * b rounded: not contracted into a following addition (with one value a group, g - sum(g) / M has to cancel exactly)
__device__ __forceinline__ float mul_rounded(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < NT / 64; ++w) v += red[w];
  return v;
}

// one workgroup per (group, sample): mean, centred sum of squares, result
template <typename T>
__global__ __launch_bounds__(NT) void gn_act_fwd_kernel(GnArgs a, T* out, float* stats) {
  __shared__ float red[NT / 64];
  drop_resolve(a.rng);
  const int g = blockIdx.x, n = blockIdx.y;
  const long long M = (long long)a.HW * a.Cg;
  float s = 0.f;
  for (long long i = threadIdx.x; i < M; i += NT) s += load_x<T>(a, n, (int)(i / a.Cg), g * a.Cg + (int)(i % a.Cg));
  const float mean = block_sum(s, red) / (float)M;
  s = 0.f;
  for (long long i = threadIdx.x; i < M; i += NT) {
    const float d = load_x<T>(a, n, (int)(i / a.Cg), g * a.Cg + (int)(i % a.Cg)) - mean;
    s += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, red) / (float)M + a.eps);
  if (threadIdx.x == 0) {
    stats[((long long)n * a.G + g) * 2] = mean;
    stats[((long long)n * a.G + g) * 2 + 1] = rstd;
  }
  for (long long i = threadIdx.x; i < M; i += NT) {
    const int p = (int)(i / a.Cg), c = g * a.Cg + (int)(i % a.Cg);
    float f[1] = {(load_x<T>(a, n, p, c) - mean) * rstd * a.gamma[c] + a.beta[c]};
    if (a.film_kind) f[0] = f[0] * (1.0f + film_at<T>(a, n * a.film_ld + c)) + film_at<T>(a, n * a.film_ld + a.C + c);
    if (a.act) f[0] = silu_f(f[0]);
    const long long o = ((long long)n * a.HW + p) * a.C + c;
    if (a.drop) drop_apply<1>(a.rng, o, f);
    out[o] = (T)f[0];
  }
}

template <typename T>
struct BwdElem {
  const GnArgs& a;
  const T* dy;
  int n;
  float mean, rstd;
  __device__ __forceinline__ void at(int p, int c, float& gv, float& xhat) const {
    xhat = (load_x<T>(a, n, p, c) - mean) * rstd;
    float v = xhat * a.gamma[c] + a.beta[c];
    if (a.film_kind) v = v * (1.0f + film_at<T>(a, n * a.film_ld + c)) + film_at<T>(a, n * a.film_ld + a.C + c);
    const long long o = ((long long)n * a.HW + p) * a.C + c;
    float f[1] = {(float)dy[o]};
    if (a.drop) drop_apply<1>(a.rng, o, f);
    if (a.act) {
      const float sg = __builtin_amdgcn_rcpf(1.0f + __expf(-v));
      f[0] *= sg * (1.0f + v * (1.0f - sg));
    }
    gv = f[0];
  }
};

// one workgroup per (group, sample); part[n][c] = A, B
template <typename T>
__global__ __launch_bounds__(NT) void gn_act_bwd_kernel(GnArgs a, const float* stats, const T* dy, T* d0, T* d1, float* part, char* dfilm) {
  __shared__ float red[NT / 64];
  drop_resolve(a.rng);
  const int g = blockIdx.x, n = blockIdx.y;
  const long long M = (long long)a.HW * a.Cg;
  const BwdElem<T> el{a, dy, n, stats[((long long)n * a.G + g) * 2], stats[((long long)n * a.G + g) * 2 + 1]};
  float m1 = 0.f, m2 = 0.f;
  for (int c = g * a.Cg; c < (g + 1) * a.Cg; ++c) {
    float A = 0.f, B = 0.f;
    for (int p = threadIdx.x; p < a.HW; p += NT) {
      float gv, xh;
      el.at(p, c, gv, xh);
      A += gv;
      B += gv * xh;
    }
    A = block_sum(A, red);
    B = block_sum(B, red);
    const float gain = a.film_kind ? 1.0f + film_at<T>(a, n * a.film_ld + c) : 1.0f;
    m1 += mul_rounded(A, a.gamma[c] * gain);
    m2 += mul_rounded(B, a.gamma[c] * gain);
    if (threadIdx.x == 0) {
      part[((long long)n * a.C + c) * 2] = A * gain;
      part[((long long)n * a.C + c) * 2 + 1] = B * gain;
      if (dfilm) {
        const float ds = a.gamma[c] * B + a.beta[c] * A;
        const long long i = (long long)n * 2 * a.C + c;
        if (a.film_kind == 1) { ((float*)dfilm)[i] = ds; ((float*)dfilm)[i + a.C] = A; }
        else { ((T*)dfilm)[i] = (T)ds; ((T*)dfilm)[i + a.C] = (T)A; }
      }
    }
  }
  m1 /= (float)M;
  m2 /= (float)M;
  for (long long i = threadIdx.x; i < M; i += NT) {
    const int p = (int)(i / a.Cg), c = g * a.Cg + (int)(i % a.Cg);
    float gv, xh;
    el.at(p, c, gv, xh);
    const float gain = a.film_kind ? 1.0f + film_at<T>(a, n * a.film_ld + c) : 1.0f;
    const T d = (T)(el.rstd * (mul_rounded(gv, a.gamma[c] * gain) - m1 - xh * m2));
    if (c < a.C0) d0[((long long)n * a.HW + p) * a.C0 + c] = d;
    else d1[((long long)n * a.HW + p) * (a.C - a.C0) + c - a.C0] = d;
  }
}

__global__ __launch_bounds__(NT) void gn_act_param_kernel(const float* part, int N, int C, float* dgamma, float* dbeta) {
  const int c = blockIdx.x * NT + threadIdx.x;
  if (c >= C) return;
  float A = 0.f, B = 0.f;
  for (int n = 0; n < N; ++n) {
    A += part[((long long)n * C + c) * 2];
    B += part[((long long)n * C + c) * 2 + 1];
  }
  dgamma[c] = B;
  dbeta[c] = A;
}

int fill_args(const ivid_gn_act_desc* d, GnArgs* a) {
  if (!d) return ivid_set_error("gn_act: no descriptor", hipSuccess);
  const int esz = d->dtype == IVID_BF16X3 ? 0 : ivid_esz(d->dtype);
  if (!esz) return ivid_set_error("gn_act: dtype must be IVID_F32, IVID_BF16 or IVID_F16", hipSuccess);
  if (d->N < 0 || d->HW < 0 || d->C0 <= 0 || d->C1 < 0 || (long long)d->C0 + d->C1 > (1 << 30))
    return ivid_set_error("gn_act: bad sizes", hipSuccess);
  if (d->groups <= 0 || (d->C0 + d->C1) % d->groups) return ivid_set_error("gn_act: C must be divisible by groups", hipSuccess);
  if ((d->C1 > 0) != (d->src1 != nullptr)) return ivid_set_error("gn_act: src1 and C1 go together", hipSuccess);
  if (d->act != 0 && d->act != 1) return ivid_set_error("gn_act: bad act", hipSuccess);
  if (!(d->eps > 0.0)) return ivid_set_error("gn_act: eps must be positive", hipSuccess);
  if (d->film && d->film_dtype != IVID_F32 && d->film_dtype != d->dtype) return ivid_set_error("gn_act: film must be fp32 or of the tensors' dtype", hipSuccess);
  if (d->N > 0 && d->HW > 0 &&
      (!d->src0 || !d->gamma || !d->beta || ((uintptr_t)d->src0 | (uintptr_t)d->src1) % esz || ((uintptr_t)d->gamma | (uintptr_t)d->beta) % 4 ||
       (uintptr_t)d->film % (d->film_dtype == IVID_F32 ? 4 : esz) || (uintptr_t)d->rng % 8))
    return ivid_set_error("gn_act: NULL or misaligned pointer", hipSuccess);
  *a = GnArgs{(const char*)d->src0, (const char*)d->src1, d->ld0, d->sn0, d->ld1, d->sn1, d->HW, d->C0, d->C0 + d->C1, d->groups,
              (d->C0 + d->C1) / d->groups, d->act, d->film ? (d->film_dtype == IVID_F32 ? 1 : 2) : 0, d->gamma, d->beta,
              (const char*)d->film, d->film_ld, (float)d->eps, false, {}};
  if (int e = ivid_drop_rng(d->p, d->seed, d->stream_id, d->rng, &a->rng)) return e;
  a->drop = a->rng.thr > 0;
  if (d->N > 65535) return ivid_set_error("gn_act: N too large", hipSuccess);
  return 0;
}
}  // namespace

extern "C" long long ivid_gn_act_scratch_bytes(const ivid_gn_act_desc* d, int backward) {
  GnArgs a;
  if (fill_args(d, &a)) return -1;
  return backward ? (long long)d->N * a.C * 8 : 0;
}

extern "C" int ivid_gn_act_forward(const ivid_gn_act_desc* d, void* out, float* stats, void* scratch, long long scratch_bytes, void* stream) {
  GnArgs a;
  if (int e = fill_args(d, &a)) return e;
  if (!d->N || !d->HW) return 0;
  if (!out || !stats) return ivid_set_error("gn_act: out / stats missing", hipSuccess);
  dim3 grid(a.G, d->N);
#define LAUNCH(T) hipLaunchKernelGGL(gn_act_fwd_kernel<T>, grid, dim3(NT), 0, (hipStream_t)stream, a, (T*)out, stats)
  if (d->dtype == IVID_F32) LAUNCH(float); else if (d->dtype == IVID_F16) LAUNCH(_Float16); else LAUNCH(__bf16);
#undef LAUNCH
  return ivid_check_launch("gn_act_forward");
}

extern "C" int ivid_gn_act_backward(const ivid_gn_act_desc* d, const float* stats, const void* dy, void* dsrc0, void* dsrc1, float* dgamma,
                                    float* dbeta, void* dfilm, void* scratch, long long scratch_bytes, void* stream) {
  GnArgs a;
  if (int e = fill_args(d, &a)) return e;
  if (!dgamma || !dbeta || (d->C1 > 0) != (dsrc1 != nullptr) || (d->film != nullptr) != (dfilm != nullptr))
    return ivid_set_error("gn_act_backward: an output is missing or has no input", hipSuccess);
  if (d->N && d->HW && (!stats || !dy || !dsrc0)) return ivid_set_error("gn_act_backward: NULL pointer", hipSuccess);
  if (scratch_bytes < (long long)d->N * a.C * 8 || (!scratch && d->N)) return ivid_set_error("gn_act_backward: scratch too small", hipSuccess);
  dim3 grid(a.G, d->N);
#define LAUNCH(T)                                                                                                             \
  hipLaunchKernelGGL(gn_act_bwd_kernel<T>, grid, dim3(NT), 0, (hipStream_t)stream, a, stats, (const T*)dy, (T*)dsrc0, (T*)dsrc1, \
                     (float*)scratch, (char*)dfilm)
  if (d->N) {
    if (d->dtype == IVID_F32) LAUNCH(float); else if (d->dtype == IVID_F16) LAUNCH(_Float16); else LAUNCH(__bf16);
  }
#undef LAUNCH
  hipLaunchKernelGGL(gn_act_param_kernel, dim3((a.C + NT - 1) / NT), dim3(NT), 0, (hipStream_t)stream, (const float*)scratch, d->N, a.C, dgamma, dbeta);
  return ivid_check_launch("gn_act_backward");
}
