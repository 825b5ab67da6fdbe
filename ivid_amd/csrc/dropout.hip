// Dropout from the counter-based generator (philox.h): the draws are a function of (seed, stream, element index), so no mask is
// stored and the backward pass is the same kernel on the gradient.
#include <math.h>
#include "common.h"
#include "internal.h"
#include "philox.h"

namespace {
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, T* out, long long n, DropRng r) {
  drop_resolve(r);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float f[1] = {(float)x[i]};
    drop_apply<1>(r, (unsigned long long)i, f);
    out[i] = (T)f[0];
  }
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
  const long long blocks = (n + 255) / 256 < 65536 ? (n + 255) / 256 : 65536;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == IVID_F32)
    hipLaunchKernelGGL(dropout_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, (const float*)x, (float*)out, n, r);
  else if (dtype == IVID_F16)
    hipLaunchKernelGGL(dropout_kernel<_Float16>, dim3((unsigned)blocks), dim3(256), 0, s, (const _Float16*)x, (_Float16*)out, n, r);
  else
    hipLaunchKernelGGL(dropout_kernel<__bf16>, dim3((unsigned)blocks), dim3(256), 0, s, (const __bf16*)x, (__bf16*)out, n, r);
  return ivid_check_launch("dropout");
}
