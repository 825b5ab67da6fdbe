// GroupNorm + FiLM + activation + dropout over channels-last tensors, forward and backward (include/ivid_hip.h ivid_gn_act_*).
//
//   xc = x - mean, xhat = xc * rstd, u = xhat * gamma + beta, v = u * (1 + s) + t, y = drop(act(v))
//   gv = drop(dy) * act'(v);  per (n, c): A = sum_p gv, B = sum_p gv * xhat
//   dshift = A, dscale = gamma * B + beta * A, dgamma = sum_n (1 + s) * B, dbeta = sum_n (1 + s) * A
//   with g = gv * gamma * (1 + s), M = HW * C / G:  dx = rstd * (g - sum(g) / M - xhat * sum(g * xhat) / M), sums over the group
//
// Bound by HBM: a forward has to read x and write y, a backward to read x and dy and write dx, and both need the whole group's sums
// before the first result.  So that nothing is read twice, a workgroup keeps its tile IN REGISTERS between the sums and the result.
// A tile is a range of pixels x a slab of whole groups (at least 128 bytes of channels, so that every line is read by one workgroup);
// the K tiles of one (sample, slab) form a cluster that exchanges its sums through memory:
//   * a sum is published as one 64-bit word {value, 1} by a relaxed agent-scope store: value and arrival in one, no fences.  The words
//     are zeroed by a launch in front (none for K = 1);
//   * every workgroup of the cluster adds the K partial sums itself, in the same order, in 64 bits: equal results, no atomics;
//   * a wait ends after a bounded number of polls: the workgroup then computes the missing tile's sums itself -- by the same code, so
//     bit for bit the same -- publishes them and goes on.  No workgroup depends on another one being resident.
// A cluster of more than MAX_K tiles would not be resident at once: it takes two launches, sums and results (PH_SUMS, PH_RESULT), with
// a small one between them that adds the words, and reads its inputs twice.
// Sums inside a tile are two-pass (mean, then centred squares) over the registers: a large mean costs no digits.
#include <math.h>
#include <utility>
#include "common.h"
#include "internal.h"
#include "philox.h"

int ivid_drop_rng(double p, unsigned long long seed, unsigned long long stream_id, const unsigned long long* rng, DropRng* out);

namespace {
constexpr int NT = 256;
constexpr int MAX_GS = 64;        // groups of a slab: one of the 256 threads' 4-lane teams each
constexpr int MAX_POLLS = 512;    // ~ 0.3 ms
constexpr int MAX_K = 128;        // tiles of a cluster that runs as one launch
enum { PH_ALL = 0, PH_SUMS = 1, PH_RESULT = 2 };

// A piece of VE elements as it is kept in registers: 32-bit words.
template <int BYTES> struct Words;
template <> struct Words<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); typedef type mem; };
template <> struct Words<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); typedef type mem; };
template <> struct Words<4> { typedef uint32_t type; typedef type mem; };
template <> struct Words<2> { typedef uint32_t type; typedef uint16_t mem; };
template <typename T, int VE> struct Piece {
  typedef typename Words<VE * sizeof(T)>::type reg;
  typedef typename Words<VE * sizeof(T)>::mem mem;
  typedef T vec __attribute__((ext_vector_type(VE)));
};

template <typename T, int VE>
__device__ __forceinline__ void unpack(typename Piece<T, VE>::reg v, float* f) {
  if constexpr (VE == 1) f[0] = (float)__builtin_bit_cast(T, (typename Piece<T, VE>::mem)v);
  else {
    const auto u = __builtin_bit_cast(typename Piece<T, VE>::vec, v);
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = (float)u[e];
  }
}
template <typename T, int VE>
__device__ __forceinline__ typename Piece<T, VE>::mem pack(const float* f) {
  if constexpr (VE == 1) return __builtin_bit_cast(typename Piece<T, VE>::mem, (T)f[0]);
  else {
    typename Piece<T, VE>::vec v;
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = (T)f[e];
    return __builtin_bit_cast(typename Piece<T, VE>::mem, v);
  }
}
// The compiler must not carry a piece's fp32 values from one pass over the registers to the next: they would need twice the registers.
template <typename R>
__device__ __forceinline__ void forget(R& v) { asm volatile("" : "+v"(v)); }

// f(0), f(1), ... f(N - 1) as straight-line code: the sweeps of a tile live in registers, which cannot be indexed by a loop
template <typename F, int... I>
__device__ __forceinline__ void sweeps_of(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void sweeps(F&& f) { sweeps_of(f, std::make_integer_sequence<int, N>{}); }

// How the work is cut (see cut_up()); part of the kernel arguments.
struct Cut {
  int S, nslab;             // channels of a slab (a multiple of the group and of the piece), slabs of a sample
  int PP, kcols;            // pieces of a tile's row; column chunks of a slab (1 unless a slab's row is wider than the workgroup)
  int RPI, nv, rows, krows; // pixels per sweep of the workgroup, sweeps, pixels of a tile, tiles down a sample
  int K, GS, W;             // tiles of a cluster, groups of a slab, lanes per group in the reductions (a power of two)
  int polls, phase;
};

struct GnArgs {
  const char *src0, *src1;
  long long ld0, sn0, ld1, sn1;
  int HW, C0, C, G, Cg, act, film_kind;  // film_kind: 0 none, 1 fp32, 2 the tensors' type
  const float *gamma, *beta;
  const char* film;
  long long film_ld;
  float eps;
  int drop;
  DropRng rng;
  Cut cut;
};

template <typename T>
__device__ __forceinline__ float film_at(const GnArgs& a, long long i) {
  return a.film_kind == 1 ? ((const float*)a.film)[i] : (float)((const T*)a.film)[i];
}

// a * b rounded: not contracted into a following addition (with one value a group, g - sum(g) / M has to cancel exactly)
__device__ __forceinline__ float mul_rounded(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

__device__ __forceinline__ void publish(unsigned long long* w, float v) {
  __hip_atomic_store(w, (1ull << 32) | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* w) {
  return __hip_atomic_load(const_cast<unsigned long long*>(w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// One tile as a thread sees it.
struct Tile {
  int row0, nrow;      // first pixel, pixels
  int cb, ce;          // channels [cb, ce)
  int r0, piece, c;    // this thread's first row, piece and channel
  bool active;
};
template <int VE>
__device__ __forceinline__ Tile tile_of(const GnArgs& a, int slab, int k) {
  const Cut& q = a.cut;
  const int kr = q.kcols == 1 ? k : k / q.kcols, kc = q.kcols == 1 ? 0 : k - kr * q.kcols;
  Tile t;
  const int cs = slab * q.S, cend = min(cs + q.S, a.C);
  t.cb = cs + kc * q.PP * VE;
  t.ce = min(t.cb + q.PP * VE, cend);
  t.row0 = kr * q.rows;
  t.nrow = min(q.rows, a.HW - t.row0);
  t.r0 = threadIdx.x / q.PP;
  t.piece = threadIdx.x - t.r0 * q.PP;
  t.c = t.cb + t.piece * VE;
  t.active = t.r0 < q.RPI && t.c < t.ce;
  return t;
}
// values of group g (of the slab) in tile k
__device__ __forceinline__ int columns_of(const GnArgs& a, int slab, int kc, int g, int VE) {
  const int cs = slab * a.cut.S;
  const int cb = cs + kc * a.cut.PP * VE, ce = min(cb + a.cut.PP * VE, min(cs + a.cut.S, a.C));
  const int lo = max(cs + g * a.Cg, cb), hi = min(cs + (g + 1) * a.Cg, ce);
  return max(hi - lo, 0);
}
__device__ __forceinline__ int groups_of(const GnArgs& a, int slab) { return min(a.cut.GS, a.G - slab * a.cut.GS); }

// per-thread channel sums s[VE] -> group sums of the tile in gs[] (LDS), the same order for every workgroup
template <int VE>
__device__ __forceinline__ void reduce_groups(const GnArgs& a, const Tile& t, int slab, const float* s, float* red, float* gs) {
  const Cut& q = a.cut;
  const int RS = q.PP * VE + 8;     // padded rows: the lanes of a team read several rows at once
  if (t.r0 < q.RPI) {
#pragma unroll
    for (int e = 0; e < VE; ++e) red[t.r0 * RS + t.piece * VE + e] = s[e];
  }
  __syncthreads();
  const int g = threadIdx.x / q.W, l = threadIdx.x - g * q.W;
  const int c0 = slab * q.S + g * a.Cg;
  const int lo = max(c0, t.cb), hi = min(c0 + a.Cg, t.ce), w = hi - lo;
  float sum = 0.f;
  if (g < groups_of(a, slab) && w > 0) {
    const int dr = q.W / w, dj = q.W - dr * w;
    int row = l / w, j = l - row * w;
    while (row < q.RPI) {
      sum += red[row * RS + lo - t.cb + j];
      row += dr;
      j += dj;
      if (j >= w) { j -= w; ++row; }
    }
  }
  for (int o = q.W >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (l == 0 && g < q.GS) gs[g] = sum;
  __syncthreads();
}

// The cluster's words of this (sample, slab): [K][GS][2].  Adds them per group, in 64 bits, in a fixed order: weight(k, g) * first [+
// second + weight * first^2 for the forward pass].  Returns the first tile whose words have not come, or -1 with the sums in out[].
template <int VE, bool MOMENTS>
__device__ __forceinline__ int gather(const GnArgs& a, int slab, const unsigned long long* words, int* missing, double2* out) {
  const Cut& q = a.cut;
  const int g = threadIdx.x / q.W, l = threadIdx.x - g * q.W;
  if (threadIdx.x == 0) *missing = 0x7fffffff;
  __syncthreads();
  double s1 = 0.0, s2 = 0.0;
  if (g < groups_of(a, slab)) {
    for (int k = l; k < q.K; k += q.W) {
      const int kr = q.kcols == 1 ? k : k / q.kcols, kc = q.kcols == 1 ? 0 : k - kr * q.kcols;
      const unsigned long long* w = words + ((size_t)k * q.GS + g) * 2;
      unsigned long long w0, w1;
      bool there = false;
      for (int i = 0; i < q.polls; ++i) {
        w0 = peek(w);
        w1 = peek(w + 1);
        there = (w0 >> 32) && (w1 >> 32);
        if (there) break;
        __builtin_amdgcn_s_sleep(4);
      }
      if (!there) {
        atomicMin(missing, k);
        break;
      }
      const double x0 = (double)__uint_as_float((unsigned)w0), x1 = (double)__uint_as_float((unsigned)w1);
      if constexpr (MOMENTS) {
        const double cnt = (double)min(q.rows, a.HW - kr * q.rows) * (double)columns_of(a, slab, kc, g, VE);
        s1 += cnt * x0;
        s2 += x1 + cnt * x0 * x0;
      } else {
        s1 += x0;
        s2 += x1;
      }
    }
  }
  for (int o = q.W >> 1; o > 0; o >>= 1) {
    s1 += __shfl_xor(s1, o);
    s2 += __shfl_xor(s2, o);
  }
  if (l == 0 && g < q.GS) out[g] = make_double2(s1, s2);
  __syncthreads();
  const int m = *missing;
  __syncthreads();
  return m == 0x7fffffff ? -1 : m;
}

// gamma * (1 + s) and beta * (1 + s) + t of one channel
template <typename T>
__device__ __forceinline__ float2 affine(const GnArgs& a, int n, int c) {
  float w = a.gamma[c], b = a.beta[c];
  if (a.film_kind) {
    const float gain = 1.0f + film_at<T>(a, (long long)n * a.film_ld + c);
    w *= gain;
    b = b * gain + film_at<T>(a, (long long)n * a.film_ld + a.C + c);
  }
  return make_float2(w, b);
}
template <int VE>
__device__ __forceinline__ void read_channels(const float* ch, int piece, float* f) {
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = ch[piece * VE + e];
}

template <typename T, int VE>
__device__ __forceinline__ const char* source(const GnArgs& a, int n, const Tile& t, long long& step) {
  const bool second = t.c >= a.C0;
  const long long ld = second ? a.ld1 : a.ld0, sn = second ? a.sn1 : a.sn0;
  step = ld * a.cut.RPI * (long long)sizeof(T);
  return (second ? a.src1 : a.src0) + ((long long)n * sn + (long long)(t.row0 + t.r0) * ld + (t.c - (second ? a.C0 : 0))) * (long long)sizeof(T);
}

template <typename T, int VE, int NV>
__global__ __launch_bounds__(NT, 4) void gn_act_fwd_kernel(GnArgs a, char* __restrict__ out, float* __restrict__ stats,
                                                           unsigned long long* words, const double2* __restrict__ totals) {
  typedef typename Piece<T, VE>::reg reg_t;
  typedef typename Piece<T, VE>::mem mem_t;
  __shared__ __attribute__((aligned(16))) float red[NT * (VE + 8)];
  __shared__ __attribute__((aligned(16))) float chM[NT * VE];
  float *const chW = red, *const chB = red + NT * VE;      // per channel mean, scale, offset: the last two once the sums are done
  __shared__ float gs[MAX_GS], gmean[MAX_GS], grstd[MAX_GS];
  __shared__ double2 tot[MAX_GS];
  __shared__ int missing;
  const Cut& q = a.cut;
  drop_resolve(a.rng);
  const int slab = blockIdx.x % q.nslab, rest = blockIdx.x / q.nslab;
  const int me = rest % q.K, n = rest / q.K;
  unsigned long long* const cluster = words + ((size_t)n * q.nslab + slab) * q.K * q.GS * 2;
  const int GS = groups_of(a, slab);
  const float Mf = (float)a.HW * (float)a.Cg;

  reg_t x[NV];
  Tile t;
  bool again = false;
  for (int k = me;;) {
    // ---- the tile into registers, its groups' means and centred squares ----
    t = tile_of<VE>(a, slab, k);
    const int mine = t.active ? t.nrow - t.r0 : 0;
    long long step;
    const char* p = source<T, VE>(a, n, t, step);
    int left = mine;      // (running pointers and counts: products with the sweep's number would all be kept across the loop)
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      x[i] = reg_t{};      // (so that no earlier tile's value stays alive behind the condition)
      if (left > 0) x[i] = *(const mem_t*)p;
      p += step;
      left -= q.RPI;
    });
    float s[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) s[e] = 0.f;
    left = mine;
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      if (left > 0) {
        float f[VE];
        forget(x[i]);
        unpack<T, VE>(x[i], f);
#pragma unroll
        for (int e = 0; e < VE; ++e) s[e] += f[e];
      }
      left -= q.RPI;
    });
    reduce_groups<VE>(a, t, slab, s, red, gs);
    const int kc = q.kcols == 1 ? 0 : k % q.kcols;
    if (threadIdx.x < GS) gmean[threadIdx.x] = gs[threadIdx.x] / fmaxf((float)t.nrow * (float)columns_of(a, slab, kc, threadIdx.x, VE), 1.f);
    __syncthreads();
    for (int j = threadIdx.x; j < t.ce - t.cb; j += NT) chM[j] = gmean[(t.cb + j) / a.Cg - slab * q.GS];
    __syncthreads();
    float m[VE];
    read_channels<VE>(chM, t.piece, m);
#pragma unroll
    for (int e = 0; e < VE; ++e) s[e] = 0.f;
    left = mine;
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      if (left > 0) {
        float f[VE];
        forget(x[i]);
        unpack<T, VE>(x[i], f);
#pragma unroll
        for (int e = 0; e < VE; ++e) { const float d = f[e] - m[e]; s[e] += d * d; }
      }
      left -= q.RPI;
    });
    reduce_groups<VE>(a, t, slab, s, red, gs);
    if (q.K == 1 || q.phase == PH_RESULT) break;
    if (threadIdx.x < GS) {
      publish(cluster + ((size_t)k * q.GS + threadIdx.x) * 2, gmean[threadIdx.x]);
      publish(cluster + ((size_t)k * q.GS + threadIdx.x) * 2 + 1, gs[threadIdx.x]);
    }
    if (q.phase == PH_SUMS) return;
    if (again) break;
    const int miss = gather<VE, true>(a, slab, cluster, &missing, tot);
    if (miss >= 0) k = miss;
    else if (k == me) break;
    else { k = me; again = true; }
  }
  __syncthreads();
  if (q.K == 1) {
    if (threadIdx.x < GS) grstd[threadIdx.x] = 1.0f / sqrtf(gs[threadIdx.x] / Mf + a.eps);
  } else {
    if (threadIdx.x < GS) {
      if (q.phase == PH_RESULT) tot[threadIdx.x] = totals[((size_t)n * q.nslab + slab) * q.GS + threadIdx.x];
      const double M = (double)a.HW * (double)a.Cg, mean = tot[threadIdx.x].x / M;
      const double var = fmax(tot[threadIdx.x].y / M - mean * mean, 0.0);
      gmean[threadIdx.x] = (float)mean;
      // a NaN sum stays one: fmax would drop it
      grstd[threadIdx.x] = tot[threadIdx.x].y == tot[threadIdx.x].y ? (float)(1.0 / sqrt(var + (double)a.eps)) : __builtin_nanf("");
    }
  }
  __syncthreads();
  if (me == 0 && threadIdx.x < GS) {
    const size_t i = ((size_t)n * a.G + slab * q.GS + threadIdx.x) * 2;
    stats[i] = gmean[threadIdx.x];
    stats[i + 1] = grstd[threadIdx.x];
  }
  for (int j = threadIdx.x; j < t.ce - t.cb; j += NT) {
    const int g = (t.cb + j) / a.Cg - slab * q.GS;
    const float2 wb = affine<T>(a, n, t.cb + j);
    chM[j] = gmean[g];
    chW[j] = wb.x * grstd[g];
    chB[j] = wb.y;
  }
  __syncthreads();
  if (!t.active) return;
  float m[VE], sc[VE], bb[VE];
  read_channels<VE>(chM, t.piece, m);
  read_channels<VE>(chW, t.piece, sc);
  read_channels<VE>(chB, t.piece, bb);
  long long o = ((long long)n * a.HW + t.row0 + t.r0) * a.C + t.c;
  const long long ostep = (long long)q.RPI * a.C;
  int left = t.nrow - t.r0;
  sweeps<NV>([&](auto i) __attribute__((always_inline)) {
    if (left > 0) {
      float f[VE];
      forget(x[i]);
      unpack<T, VE>(x[i], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = (f[e] - m[e]) * sc[e] + bb[e];
      if (a.act) {
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = silu_f(f[e]);
      }
      if (a.drop) drop_apply<VE>(a.rng, (unsigned long long)o, f);
      *(mem_t*)(out + o * (long long)sizeof(T)) = pack<T, VE>(f);
    }
    o += ostep;
    left -= q.RPI;
  });
}

// dscale, dshift of one (n, c) and its share of dgamma, dbeta
template <typename T>
__device__ __forceinline__ void channel_done(const GnArgs& a, int n, int c, float A, float B, float2* ab, char* dfilm) {
  float gain = 1.0f;
  if (a.film_kind) {
    gain += film_at<T>(a, (long long)n * a.film_ld + c);
    const float ds = a.gamma[c] * B + a.beta[c] * A;
    const long long i = (long long)n * 2 * a.C + c;
    if (a.film_kind == 1) { ((float*)dfilm)[i] = ds; ((float*)dfilm)[i + a.C] = A; }
    else { ((T*)dfilm)[i] = (T)ds; ((T*)dfilm)[i + a.C] = (T)A; }
  }
  ab[(long long)n * a.C + c] = make_float2(gain * A, gain * B);
}

template <typename T, int VE, int NV>
__global__ __launch_bounds__(NT, 2) void gn_act_bwd_kernel(GnArgs a, const float* __restrict__ stats, const char* __restrict__ dy,
                                                           char* __restrict__ d0, char* __restrict__ d1, unsigned long long* words,
                                                           const double2* __restrict__ totals, float2* __restrict__ part,
                                                           float2* __restrict__ ab, char* __restrict__ dfilm) {
  typedef typename Piece<T, VE>::reg reg_t;
  typedef typename Piece<T, VE>::mem mem_t;
  __shared__ __attribute__((aligned(16))) float redA[NT * (VE + 8)], redB[NT * (VE + 8)];
  // per channel: mean, gamma * (1 + s), the offset (then A), B
  __shared__ __attribute__((aligned(16))) float chM[NT * VE], chW[NT * VE], chA[NT * VE], chB[NT * VE];
  __shared__ float gmean[MAX_GS], grstd[MAX_GS], gm1[MAX_GS], gm2[MAX_GS];
  __shared__ double2 tot[MAX_GS];
  __shared__ int missing;
  const Cut& q = a.cut;
  drop_resolve(a.rng);
  const int slab = blockIdx.x % q.nslab, rest = blockIdx.x / q.nslab;
  const int me = rest % q.K, n = rest / q.K;
  unsigned long long* const cluster = words + ((size_t)n * q.nslab + slab) * q.K * q.GS * 2;
  const int GS = groups_of(a, slab);
  const float Mf = (float)a.HW * (float)a.Cg;
  if (threadIdx.x < GS) {
    const size_t i = ((size_t)n * a.G + slab * q.GS + threadIdx.x) * 2;
    gmean[threadIdx.x] = stats[i];
    grstd[threadIdx.x] = stats[i + 1];
  }
  __syncthreads();

  reg_t x[NV];
  float gv[NV][VE];
  Tile t;
  bool again = false;
  for (int k = me;;) {
    t = tile_of<VE>(a, slab, k);
    const int mine = t.active ? t.nrow - t.r0 : 0;
    const long long o0 = ((long long)n * a.HW + t.row0 + t.r0) * a.C + t.c, ostep = (long long)q.RPI * a.C;
    long long step;
    const char* p = source<T, VE>(a, n, t, step);
    reg_t g[NV];
    int left = mine;
    const char* pd = dy + o0 * (long long)sizeof(T);
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      x[i] = g[i] = reg_t{};      // (so that no earlier tile's value stays alive behind the condition)
      if (left > 0) {
        x[i] = *(const mem_t*)p;
        g[i] = *(const mem_t*)pd;
      }
      p += step;
      pd += ostep * (long long)sizeof(T);
      left -= q.RPI;
    });
    for (int j = threadIdx.x; j < t.ce - t.cb; j += NT) {
      const int gj = (t.cb + j) / a.Cg - slab * q.GS;
      const float2 wb = affine<T>(a, n, t.cb + j);
      chM[j] = gmean[gj];
      chW[j] = wb.x;
      chA[j] = wb.y;
      chB[j] = wb.x * grstd[gj];
    }
    __syncthreads();
    float m[VE], bb[VE], sc[VE], A[VE], B[VE];
    read_channels<VE>(chM, t.piece, m);
    read_channels<VE>(chA, t.piece, bb);
    read_channels<VE>(chB, t.piece, sc);
#pragma unroll
    for (int e = 0; e < VE; ++e) A[e] = B[e] = 0.f;
    left = mine;
    long long o = o0;
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      if (left > 0) {
        float f[VE], d[VE];
        forget(x[i]);
        unpack<T, VE>(x[i], f);
        unpack<T, VE>(g[i], d);
        if (a.drop) drop_apply<VE>(a.rng, (unsigned long long)o, d);
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] -= m[e];
        if (a.act) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float v = f[e] * sc[e] + bb[e];
            const float sg = __builtin_amdgcn_rcpf(1.0f + __expf(-v));
            d[e] *= sg * (1.0f + v * (1.0f - sg));
          }
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          gv[i][e] = d[e];
          A[e] += d[e];
          B[e] += d[e] * f[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) gv[i][e] = 0.f;
      }
      o += ostep;
      left -= q.RPI;
    });
    // ---- channel sums over the tile's pixels ----
    const int RS = q.PP * VE + 8, ncol = t.ce - t.cb;
    if (t.r0 < q.RPI) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        redA[t.r0 * RS + t.piece * VE + e] = A[e];
        redB[t.r0 * RS + t.piece * VE + e] = B[e];
      }
    }
    __syncthreads();
    const int parts = ncol < NT ? NT / ncol : 1;
    if (parts > 1) {
      const int h = threadIdx.x / ncol, j = threadIdx.x - h * ncol;
      float sa = 0.f, sb = 0.f;
      if (h < parts) {
        for (int r = h; r < q.RPI; r += parts) { sa += redA[r * RS + j]; sb += redB[r * RS + j]; }
      }
      __syncthreads();
      if (h < parts) { redA[h * ncol + j] = sa; redB[h * ncol + j] = sb; }
      __syncthreads();
    }
    const int nr = parts > 1 ? min(parts, q.RPI) : q.RPI, rs = parts > 1 ? ncol : RS;
    const int kr = q.kcols == 1 ? k : k / q.kcols;
    for (int j = threadIdx.x; j < ncol; j += NT) {
      float sa = 0.f, sb = 0.f;
      for (int r = 0; r < nr; ++r) { sa += redA[r * rs + j]; sb += redB[r * rs + j]; }
      sb *= grstd[(t.cb + j) / a.Cg - slab * q.GS];
      chA[j] = sa;
      chB[j] = sb;
      if (q.krows > 1) part[((size_t)n * q.krows + kr) * a.C + t.cb + j] = make_float2(sa, sb);
      else channel_done<T>(a, n, t.cb + j, sa, sb, ab, dfilm);
    }
    __syncthreads();
    // ---- the groups' sums of g and g * xhat ----
    {
      const int g2 = threadIdx.x / q.W, l = threadIdx.x - g2 * q.W;
      const int c0 = slab * q.S + g2 * a.Cg;
      float s1 = 0.f, s2 = 0.f;
      if (g2 < GS) {
        for (int j = max(c0, t.cb) - t.cb + l; j < min(c0 + a.Cg, t.ce) - t.cb; j += q.W) {
          s1 += mul_rounded(chA[j], chW[j]);
          s2 += mul_rounded(chB[j], chW[j]);
        }
      }
      for (int o = q.W >> 1; o > 0; o >>= 1) {
        s1 += __shfl_xor(s1, o);
        s2 += __shfl_xor(s2, o);
      }
      if (l == 0 && g2 < GS) {
        gm1[g2] = s1 / Mf;
        gm2[g2] = s2 / Mf;
        if (q.K > 1 && q.phase != PH_RESULT) {
          publish(cluster + ((size_t)k * q.GS + g2) * 2, s1);
          publish(cluster + ((size_t)k * q.GS + g2) * 2 + 1, s2);
        }
      }
    }
    if (q.phase == PH_SUMS) return;
    if (q.K == 1 || q.phase == PH_RESULT || again) break;
    const int miss = gather<VE, false>(a, slab, cluster, &missing, tot);
    if (miss >= 0) k = miss;
    else if (k == me) break;
    else { k = me; again = true; }
  }
  __syncthreads();
  if (q.K > 1) {
    if (threadIdx.x < GS) {
      if (q.phase == PH_RESULT) tot[threadIdx.x] = totals[((size_t)n * q.nslab + slab) * q.GS + threadIdx.x];
      const double M = (double)a.HW * (double)a.Cg;
      gm1[threadIdx.x] = (float)(tot[threadIdx.x].x / M);
      gm2[threadIdx.x] = (float)(tot[threadIdx.x].y / M);
    }
    __syncthreads();
  }
  for (int j = threadIdx.x; j < t.ce - t.cb; j += NT) {
    const int g = (t.cb + j) / a.Cg - slab * q.GS;
    chA[j] = gm1[g];
    chB[j] = gm2[g] * grstd[g];
    redA[j] = grstd[g];
  }
  __syncthreads();
  if (!t.active) return;
  const bool second = t.c >= a.C0;
  const long long ld = second ? a.C - a.C0 : a.C0;
  char* o = (second ? d1 : d0) + (((long long)n * a.HW + t.row0 + t.r0) * ld + (t.c - (second ? a.C0 : 0))) * (long long)sizeof(T);
  const long long ostep = ld * q.RPI * (long long)sizeof(T);
  int left = t.nrow - t.r0;
  float m[VE], gw[VE], m1[VE], m2[VE], rs[VE];
  read_channels<VE>(chM, t.piece, m);
  read_channels<VE>(chW, t.piece, gw);
  read_channels<VE>(chA, t.piece, m1);
  read_channels<VE>(chB, t.piece, m2);
  read_channels<VE>(redA, t.piece, rs);
  sweeps<NV>([&](auto i) __attribute__((always_inline)) {
    if (left > 0) {
      float f[VE];
      forget(x[i]);
      unpack<T, VE>(x[i], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = rs[e] * ((mul_rounded(gv[i][e], gw[e]) - m1[e]) - (f[e] - m[e]) * m2[e]);
      *(mem_t*)o = pack<T, VE>(f);
    }
    o += ostep;
    left -= q.RPI;
  });
}

// the words of one cluster added up, between PH_SUMS and PH_RESULT: one workgroup per (sample, slab)
template <int VE, bool MOMENTS>
__global__ __launch_bounds__(NT) void gn_act_total_kernel(GnArgs a, const unsigned long long* words, double2* __restrict__ totals) {
  __shared__ double2 tot[MAX_GS];
  __shared__ int missing;
  const Cut& q = a.cut;
  const int slab = blockIdx.x % q.nslab;
  gather<VE, MOMENTS>(a, slab, words + (size_t)blockIdx.x * q.K * q.GS * 2, &missing, tot);
  if (threadIdx.x < groups_of(a, slab)) totals[(size_t)blockIdx.x * q.GS + threadIdx.x] = tot[threadIdx.x];
}

// zeroes the clusters' words (a kernel, so that it may be captured)
__global__ __launch_bounds__(NT) void gn_act_clear_kernel(ulonglong2* words, long long n) {
  const long long i = (long long)blockIdx.x * NT + threadIdx.x;
  if (i < n) words[i] = make_ulonglong2(0, 0);
}

// part [N][krows][C] -> ab [N][C], dfilm: 64 channels a workgroup, four threads a channel
template <typename T>
__global__ __launch_bounds__(NT) void gn_act_film_kernel(GnArgs a, const float2* __restrict__ part, float2* __restrict__ ab, char* __restrict__ dfilm) {
  __shared__ float2 red[NT];
  const int cblk = (a.C + 63) / 64;
  const int n = blockIdx.x / cblk, c = (blockIdx.x - n * cblk) * 64 + (threadIdx.x & 63), h = threadIdx.x >> 6;
  float A = 0.f, B = 0.f;
  if (c < a.C) {
    for (int k = h; k < a.cut.krows; k += NT / 64) {
      const float2 v = part[((size_t)n * a.cut.krows + k) * a.C + c];
      A += v.x;
      B += v.y;
    }
  }
  red[threadIdx.x] = make_float2(A, B);
  __syncthreads();
  if (h == 0 && c < a.C) {
#pragma unroll
    for (int j = 1; j < NT / 64; ++j) { A += red[threadIdx.x + 64 * j].x; B += red[threadIdx.x + 64 * j].y; }
    channel_done<T>(a, n, c, A, B, ab, dfilm);
  }
}

// ab [N][C] -> dgamma, dbeta: 16 channels a workgroup, 16 threads a channel
__global__ __launch_bounds__(NT) void gn_act_param_kernel(const float2* __restrict__ ab, int N, int C, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float2 red[NT];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), h = threadIdx.x >> 4;
  float A = 0.f, B = 0.f;
  if (c < C) {
    for (int n = h; n < N; n += 16) {
      const float2 v = ab[(size_t)n * C + c];
      A += v.x;
      B += v.y;
    }
  }
  red[threadIdx.x] = make_float2(A, B);
  __syncthreads();
  if (h == 0 && c < C) {
#pragma unroll
    for (int j = 1; j < 16; ++j) { A += red[threadIdx.x + 16 * j].x; B += red[threadIdx.x + 16 * j].y; }
    dgamma[c] = B;
    dbeta[c] = A;
  }
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// register-resident sweeps per type of piece
constexpr int NV_FWD = 16, NV_BWD = 12, NV_NARROW = 32;
int max_sweeps(int ve, bool backward) { return ve <= 2 ? NV_NARROW : (backward ? NV_BWD : NV_FWD); }

int cut_up(const ivid_gn_act_desc* d, bool backward, GnArgs* a, int* ve_out) {
  const int esz = ivid_esz(d->dtype);
  // the widest piece that every row of every tensor is a whole number of
  int ve = 16 / esz;
  auto fits = [&](int v) {
    const long long mask = v - 1;
    return !((d->C0 | d->C1 | d->ld0 | d->sn0 | (d->C1 ? d->ld1 | d->sn1 : 0)) & mask) && !((uintptr_t)d->src0 % (v * esz)) &&
           !((uintptr_t)d->src1 % (v * esz));
  };
  while (ve > 1 && !fits(ve)) ve >>= 1;
  const int C = a->C, Cg = a->Cg;
  const long long unit = (long long)Cg / gcd(Cg, ve) * ve;     // whole groups and whole pieces
  Cut& q = a->cut;
  long long S = unit;
  while (S < C && S * esz < 128 && (S + unit) / Cg <= MAX_GS && (S + unit) / ve <= NT) S += unit;
  // whole 128-byte lines, if a few more groups make them
  for (long long s = S; s <= 4 * S && s <= C && s / Cg <= MAX_GS && s / ve <= NT; s += unit)
    if (s * esz % 128 == 0) { S = s; break; }
  if (S > C) S = C;            // C is a multiple of the unit
  q.S = (int)S;
  q.nslab = (int)((C + S - 1) / S);
  q.GS = (int)(S / Cg);
  if (q.GS > MAX_GS) return ivid_set_error("gn_act: internal: too many groups in a slab", hipSuccess);
  const int pieces = (int)(S / ve);
  q.kcols = (pieces + NT - 1) / NT;
  q.PP = (pieces + q.kcols - 1) / q.kcols;
  q.RPI = NT / q.PP;
  q.W = 64;
  while (q.W * q.GS > NT) q.W >>= 1;
  const int most = max_sweeps(ve, backward);
  q.nv = (int)(((long long)d->HW + q.RPI - 1) / q.RPI);
  if (q.nv > most) q.nv = most;
  q.rows = q.RPI * q.nv;
  q.krows = (int)(((long long)d->HW + q.rows - 1) / q.rows);
  q.polls = d->max_polls > 0 ? d->max_polls : MAX_POLLS;
  *ve_out = ve;
  const double tiles = (double)d->N * q.nslab * q.krows * q.kcols;
  q.K = tiles < (1 << 24) ? q.krows * q.kcols : 0;
  if (!q.K || (long long)d->N * ((C + 63) / 64) >= (1 << 24))
    return ivid_set_error("gn_act: too many tiles for one launch", hipSuccess);
  return 0;
}

int fill_args(const ivid_gn_act_desc* d, bool backward, GnArgs* a, int* ve) {
  if (!d) return ivid_set_error("gn_act: no descriptor", hipSuccess);
  const int esz = d->dtype == IVID_BF16X3 ? 0 : ivid_esz(d->dtype);
  if (!esz) return ivid_set_error("gn_act: dtype must be IVID_F32, IVID_BF16 or IVID_F16", hipSuccess);
  if (d->N < 1 || d->HW < 1 || d->C0 < 1 || d->C1 < 0 || (long long)d->C0 + d->C1 > (1 << 24))
    return ivid_set_error("gn_act: bad sizes", hipSuccess);
  if (d->groups <= 0 || (d->C0 + d->C1) % d->groups) return ivid_set_error("gn_act: C must be divisible by groups", hipSuccess);
  if ((d->C1 > 0) != (d->src1 != nullptr)) return ivid_set_error("gn_act: src1 and C1 go together", hipSuccess);
  if (d->ld0 < 0 || d->sn0 < 0 || d->ld1 < 0 || d->sn1 < 0 || d->film_ld < 0) return ivid_set_error("gn_act: negative stride", hipSuccess);
  if (d->act != 0 && d->act != 1) return ivid_set_error("gn_act: bad act", hipSuccess);
  if (!(d->eps > 0.0)) return ivid_set_error("gn_act: eps must be positive", hipSuccess);
  if (d->film && d->film_dtype != IVID_F32 && d->film_dtype != d->dtype) return ivid_set_error("gn_act: film must be fp32 or of the tensors' dtype", hipSuccess);
  if (!d->src0 || !d->gamma || !d->beta || ((uintptr_t)d->src0 | (uintptr_t)d->src1) % esz || ((uintptr_t)d->gamma | (uintptr_t)d->beta) % 4 ||
      (uintptr_t)d->film % (d->film_dtype == IVID_F32 ? 4 : esz) || (uintptr_t)d->rng % 8)
    return ivid_set_error("gn_act: NULL or misaligned pointer", hipSuccess);
  *a = GnArgs{(const char*)d->src0, (const char*)d->src1, d->ld0, d->sn0, d->ld1, d->sn1, d->HW, d->C0, d->C0 + d->C1, d->groups,
              (d->C0 + d->C1) / d->groups, d->act, d->film ? (d->film_dtype == IVID_F32 ? 1 : 2) : 0, d->gamma, d->beta,
              (const char*)d->film, d->film_ld, (float)d->eps, 0, {}, {}};
  if (int e = ivid_drop_rng(d->p, d->seed, d->stream_id, d->rng, &a->rng)) return e;
  a->drop = a->rng.thr > 0;
  return cut_up(d, backward, a, ve);
}

// scratch: the clusters' words, (K > MAX_K) their totals, then (backward) ab [N][C] and part [N][krows][C]
struct Scratch { long long words, totals, ab, part, total; };
Scratch layout(const ivid_gn_act_desc* d, const GnArgs& a, bool backward) {
  Scratch s{};
  const Cut& q = a.cut;
  if (q.K > 1) s.words = (long long)d->N * q.nslab * q.K * q.GS * 16;
  if (q.K > MAX_K) s.totals = (long long)d->N * q.nslab * q.GS * 16;
  if (backward) {
    s.ab = (long long)d->N * a.C * 8;
    if (q.krows > 1) s.part = (long long)d->N * q.krows * a.C * 8;
  }
  s.total = s.words + s.totals + s.ab + s.part;
  return s;
}

int clear_words(const Scratch& s, void* scratch, hipStream_t stream) {
  if (!s.words || s.totals) return 0;      // two launches: every word is written before any is read
  const long long n = s.words / 16, blocks = (n + NT - 1) / NT;
  if (blocks >= (1 << 24)) return ivid_set_error("gn_act: too many tiles for one launch", hipSuccess);
  hipLaunchKernelGGL(gn_act_clear_kernel, dim3((unsigned)blocks), dim3(NT), 0, stream, (ulonglong2*)scratch, n);
  return 0;
}

// `run` launches the kernel once, or as sums - totals - results
template <bool MOMENTS, typename Run>
void run_phases(GnArgs& a, const ivid_gn_act_desc* d, int ve, const Scratch& s, void* scratch, hipStream_t st, Run run) {
  if (!s.totals) {
    run();
    return;
  }
  a.cut.phase = PH_SUMS;
  run();
  const dim3 grid((unsigned)((long long)d->N * a.cut.nslab));
  double2* totals = (double2*)((char*)scratch + s.words);
#define TOTAL(VE) hipLaunchKernelGGL((gn_act_total_kernel<VE, MOMENTS>), grid, dim3(NT), 0, st, a, (const unsigned long long*)scratch, totals)
  if (ve == 8) TOTAL(8); else if (ve == 4) TOTAL(4); else if (ve == 2) TOTAL(2); else TOTAL(1);
#undef TOTAL
  a.cut.phase = PH_RESULT;
  run();
}
}  // namespace

extern "C" long long ivid_gn_act_scratch_bytes(const ivid_gn_act_desc* d, int backward) {
  GnArgs a;
  int ve;
  if (fill_args(d, backward != 0, &a, &ve)) return -1;
  return layout(d, a, backward != 0).total;
}

extern "C" int ivid_gn_act_forward(const ivid_gn_act_desc* d, void* out, float* stats, void* scratch, long long scratch_bytes, void* stream) {
  GnArgs a;
  int ve;
  if (int e = fill_args(d, false, &a, &ve)) return e;
  if (!out || !stats || ((uintptr_t)out & 15) || ((uintptr_t)stats & 3)) return ivid_set_error("gn_act: out / stats missing or misaligned", hipSuccess);
  const Scratch s = layout(d, a, false);
  if (scratch_bytes < s.total || (s.total && (!scratch || ((uintptr_t)scratch & 15)))) return ivid_set_error("gn_act: scratch too small or misaligned", hipSuccess);
  hipStream_t st = (hipStream_t)stream;
  if (int e = clear_words(s, scratch, st)) return e;
  const dim3 grid((unsigned)((long long)d->N * a.cut.nslab * a.cut.K));
#define LAUNCH(T, VE, NV) \
  hipLaunchKernelGGL((gn_act_fwd_kernel<T, VE, NV>), grid, dim3(NT), 0, st, a, (char*)out, stats, (unsigned long long*)scratch, \
                     (const double2*)((char*)scratch + s.words))
#define LAUNCH16(T)                                   \
  do {                                                \
    if (ve == 8) LAUNCH(T, 8, NV_FWD);                \
    else if (ve == 4) LAUNCH(T, 4, NV_FWD);           \
    else if (ve == 2) LAUNCH(T, 2, NV_NARROW);        \
    else LAUNCH(T, 1, NV_NARROW);                     \
  } while (0)
  run_phases<true>(a, d, ve, s, scratch, st, [&] {
    if (d->dtype == IVID_F32) {
      if (ve == 4) LAUNCH(float, 4, NV_FWD);
      else if (ve == 2) LAUNCH(float, 2, NV_NARROW);
      else LAUNCH(float, 1, NV_NARROW);
    } else if (d->dtype == IVID_BF16) {
      LAUNCH16(__bf16);
    } else {
      LAUNCH16(_Float16);
    }
  });
#undef LAUNCH16
#undef LAUNCH
  return ivid_check_launch("gn_act_forward");
}

extern "C" int ivid_gn_act_backward(const ivid_gn_act_desc* d, const float* stats, const void* dy, void* dsrc0, void* dsrc1, float* dgamma,
                                    float* dbeta, void* dfilm, void* scratch, long long scratch_bytes, void* stream) {
  GnArgs a;
  int ve;
  if (int e = fill_args(d, true, &a, &ve)) return e;
  if (!dgamma || !dbeta || (d->C1 > 0) != (dsrc1 != nullptr) || (d->film != nullptr) != (dfilm != nullptr))
    return ivid_set_error("gn_act_backward: an output is missing or has no input", hipSuccess);
  if (!stats || !dy || !dsrc0 || (((uintptr_t)dy | (uintptr_t)dsrc0 | (uintptr_t)dsrc1) & 15) ||
      (((uintptr_t)stats | (uintptr_t)dgamma | (uintptr_t)dbeta | (uintptr_t)dfilm) & 3))
    return ivid_set_error("gn_act_backward: NULL or misaligned pointer", hipSuccess);
  const Scratch s = layout(d, a, true);
  if (scratch_bytes < s.total || !scratch || ((uintptr_t)scratch & 15)) return ivid_set_error("gn_act_backward: scratch too small or misaligned", hipSuccess);
  hipStream_t st = (hipStream_t)stream;
  if (int e = clear_words(s, scratch, st)) return e;
  float2* ab = (float2*)((char*)scratch + s.words + s.totals);
  float2* part = (float2*)((char*)scratch + s.words + s.totals + s.ab);
  const dim3 grid((unsigned)((long long)d->N * a.cut.nslab * a.cut.K));
#define LAUNCH(T, VE, NV)                                                                                              \
  hipLaunchKernelGGL((gn_act_bwd_kernel<T, VE, NV>), grid, dim3(NT), 0, st, a, stats, (const char*)dy, (char*)dsrc0,   \
                     (char*)dsrc1, (unsigned long long*)scratch, (const double2*)((char*)scratch + s.words), part, ab, (char*)dfilm)
#define LAUNCH16(T)                                   \
  do {                                                \
    if (ve == 8) LAUNCH(T, 8, NV_BWD);                \
    else if (ve == 4) LAUNCH(T, 4, NV_BWD);           \
    else if (ve == 2) LAUNCH(T, 2, NV_NARROW);        \
    else LAUNCH(T, 1, NV_NARROW);                     \
  } while (0)
  run_phases<false>(a, d, ve, s, scratch, st, [&] {
    if (d->dtype == IVID_F32) {
      if (ve == 4) LAUNCH(float, 4, NV_BWD);
      else if (ve == 2) LAUNCH(float, 2, NV_NARROW);
      else LAUNCH(float, 1, NV_NARROW);
    } else if (d->dtype == IVID_BF16) {
      LAUNCH16(__bf16);
    } else {
      LAUNCH16(_Float16);
    }
  });
#undef LAUNCH16
#undef LAUNCH
  if (s.part) {
    const dim3 g2((unsigned)((long long)d->N * ((a.C + 63) / 64)));
#define FILM(T) hipLaunchKernelGGL(gn_act_film_kernel<T>, g2, dim3(NT), 0, st, a, (const float2*)part, ab, (char*)dfilm)
    if (d->dtype == IVID_F32) FILM(float); else if (d->dtype == IVID_BF16) FILM(__bf16); else FILM(_Float16);
#undef FILM
  }
  hipLaunchKernelGGL(gn_act_param_kernel, dim3((unsigned)((a.C + 15) / 16)), dim3(NT), 0, st, (const float2*)ab, d->N, a.C, dgamma, dbeta);
  return ivid_check_launch("gn_act_backward");
}
