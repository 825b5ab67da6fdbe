// Dropout from the counter-based generator (philox.h): the draws are a function of (seed, stream, element index), so no mask is
// stored and the backward pass is the same kernel on the gradient.
//
// A thread takes whole generator blocks of eight elements, STEPS of them, all loads in front of the generator's rounds: bound by HBM,
// 188 us for 64 x 128 x 128 x 256 bf16 (537 MB in, 537 MB out: 5.7 TB/s; a copy 202 us), where one element a thread ran 558.
#include <math.h>
#include "common.h"
#include "internal.h"
#include "philox.h"

namespace {
constexpr int NT = 256, STEPS = 4;

template <typename T> struct Eight { typedef T vec __attribute__((ext_vector_type(8), aligned(16))); };

template <typename T>
__global__ __launch_bounds__(NT) void dropout_kernel(const T* x, T* out, long long n, DropRng r) {
  typedef typename Eight<T>::vec vec_t;
  drop_resolve(r);
  const long long blocks = n >> 3, b0 = (long long)blockIdx.x * (NT * STEPS) + threadIdx.x;
  vec_t v[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
    if (b0 + i * NT < blocks) v[i] = *(const vec_t*)(x + (b0 + i * NT) * 8);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const long long b = b0 + i * NT;
    if (b < blocks) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)v[i][e];
      drop_apply<8>(r, (unsigned long long)b * 8, f);
      vec_t o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = (T)f[e];
      *(vec_t*)(out + b * 8) = o;
    } else if (b == blocks) {
      for (long long j = b * 8; j < n; ++j) {
        float f[1] = {(float)x[j]};
        drop_apply<1>(r, (unsigned long long)j, f);
        out[j] = (T)f[0];
      }
    }
  }
}

// pointers that are aligned to an element only
template <typename T>
__global__ __launch_bounds__(NT) void dropout_scalar_kernel(const T* x, T* out, long long n, DropRng r) {
  drop_resolve(r);
  const long long i = (long long)blockIdx.x * NT + threadIdx.x;
  if (i < n) {
    float f[1] = {(float)x[i]};
    drop_apply<1>(r, (unsigned long long)i, f);
    out[i] = (T)f[0];
  }
}

template <typename T>
int launch(const void* x, void* out, long long n, const DropRng& r, hipStream_t s) {
  const bool wide = !(((uintptr_t)x | (uintptr_t)out) & 15);
  const long long per = wide ? NT * STEPS * 8 : NT, blocks = (n + per - 1) / per;
  if (blocks >= (1 << 24)) return ivid_set_error("dropout: n too large for one launch", hipSuccess);   // 2^32 threads is the limit
  if (wide)
    hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)blocks), dim3(NT), 0, s, (const T*)x, (T*)out, n, r);
  else
    hipLaunchKernelGGL(dropout_scalar_kernel<T>, dim3((unsigned)blocks), dim3(NT), 0, s, (const T*)x, (T*)out, n, r);
  return ivid_check_launch("dropout");
}
}  // namespace

int ivid_drop_rng(double p, unsigned long long seed, unsigned long long stream_id, const unsigned long long* rng, DropRng* out) {
  if (!(p >= 0.0 && p <= 1.0)) return ivid_set_error("dropout: p must be in [0, 1]", hipSuccess);
  out->seed = seed;
  out->stream = stream_id;
  out->dev = rng;
  out->thr = (uint32_t)floor(p * 65536.0 + 0.5);
  out->scale = out->thr < 65536u ? (float)(65536.0 / (65536.0 - (double)out->thr)) : 0.f;
  return 0;
}

extern "C" int ivid_dropout(int dtype, const void* x, void* out, long long n, double p, unsigned long long seed,
                            unsigned long long stream_id, const unsigned long long* rng, void* stream) {
  const int esz = dtype == IVID_BF16X3 ? 0 : ivid_esz(dtype);
  if (!esz) return ivid_set_error("dropout: bad dtype", hipSuccess);
  DropRng r;
  if (int e = ivid_drop_rng(p, seed, stream_id, rng, &r)) return e;
  if (n < 0) return ivid_set_error("dropout: n < 0", hipSuccess);
  if (n == 0) return 0;
  if (!x || !out || (((uintptr_t)x | (uintptr_t)out) % esz) || ((uintptr_t)rng & 7))
    return ivid_set_error("dropout: NULL or misaligned pointer", hipSuccess);
  const uintptr_t px = (uintptr_t)x, po = (uintptr_t)out;
  if (px != po && (px < po ? po - px : px - po) / esz < (unsigned long long)n)
    return ivid_set_error("dropout: x and out overlap and are not the same", hipSuccess);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == IVID_F32) return launch<float>(x, out, n, r, s);
  return dtype == IVID_F16 ? launch<_Float16>(x, out, n, r, s) : launch<__bf16>(x, out, n, r, s);
}
