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
//   * a wait ends after a bounded number of polls: the workgroup then computes the missing tile's sums itself, in the same order and
//     so bit for bit the same, publishes them and goes on.  No workgroup depends on another one being resident.
// A cluster of more than MAX_K tiles would not be resident at once: it takes two launches, sums and results (PH_SUMS, PH_RESULT), with
// a small one between them that adds the words.  The second is the same code: it reads its inputs again and computes its tile's sums
// again, which it then does not use.
// The channels' sums of the tiles (backward) are added in 64 bits too, by launches behind the kernel.
// Squares are centred on the tile's own means: a large mean costs no digits.
//
// Choices and what they measured (MI355X; 64 x 128 x 128 x 256 bf16; copying that tensor takes 202 us, 5.3 TB/s).  A variant's
// time stands next to that of the form it was compared with, on the same card: several steps lie between some of them.
//   * now: forward 238 us (4.5 TB/s; with dropout 272), backward 374 (4.3 TB/s; 421).  One workgroup per (sample, group) with three
//     passes over memory: forward 2793, a training step with dropout 15699 (now 690);
//   * forward: 512 threads x 16 pieces (128 KB of x a workgroup) 293; 256 threads x 16 pieces 298, 1024 x 16: 322, 512 x 8: 323.
//     Backward: 256 threads x 12 pieces, x and the fp32 gradient behind the activation kept, 464; 512 threads 582; 10 pieces 522,
//     16: 527;
//   * a cluster's workgroups next to each other in the grid: forward 337 -> 309, backward 571 -> 506;
//   * loads without branches around them and coefficients in front of the tile, so that the compiler waits for one piece after the
//     other while the sums run, with lighter joins: forward 317 -> 255, backward 570 -> 433;
//   * the group sums published in front of the channel sums: backward 425 -> 374;
//   * slabs of 64 bytes 255 / 488 where 128 ran 238 / 426; of 256 bytes 302 / 528 where 128 ran 309 / 506 (forward / backward);
//   * what is left: the vector units are busy 64 % of the forward's and 68 % of the backward's time by the counters (78 and 72 % with
//     dropout: 9 more instructions an element, of 20 and 28), and a workgroup reads, sums, waits and writes in turn, so that these
//     overlap with memory between workgroups only.
#include <math.h>
#include <utility>
#include "common.h"
#include "internal.h"
#include "philox.h"

int ivid_drop_rng(double p, unsigned long long seed, unsigned long long stream_id, const unsigned long long* rng, DropRng* out);

#pragma clang fp contract(off)      // every fused multiply-add below is written out: a sum has the same bits wherever it is computed

namespace {
constexpr int NT_FWD = 512, NT_BWD = 256, NT_AUX = 256;
constexpr int MAX_GS = 64;        // groups of a slab: at least four lanes each in the reductions
constexpr int MAX_COL = 1024;     // channels of a tile
constexpr int MAX_POLLS = 512;    // ~ 1 ms
// Tiles of a cluster that runs as one launch: half of the 512 workgroups of a backward pass that the chip holds at once.  8 x 256 x 256 x
// 128 bf16, one launch against two (the second with its unused sums): backward (171 tiles) 134 us against 151, forward (64 tiles) 63
// against 84.
constexpr int MAX_K = 256;
constexpr int MIN_TILES = 16;     // of a sample, once it is cut
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
// The compiler must not carry a piece's fp32 values, or the counts that tell which pieces there are, from one pass over the registers to
// the next: they would need more registers than the data.
template <typename R>
__device__ __forceinline__ void forget(R& v) { asm volatile("" : "+v"(v)); }

// threadIdx.x as a value of its own: what is computed from it is not shared with, and so not kept for, another part of the kernel
__device__ __forceinline__ int fresh_thread() {
  int t = threadIdx.x;
  forget(t);
  return t;
}

// Every load has come back (s_waitcnt vmcnt(0)).  Behind the conditions around its pieces the compiler cannot know, and would wait for
// "all but the last few" memory operations in front of each piece -- which by then are the results' own stores, of the same counter.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// f(0), f(1), ... f(N - 1) as straight-line code: the sweeps of a tile live in registers, which cannot be indexed by a loop.  No branch
// around them either: the loads have to be unconditional for the compiler to wait for one after the other.
template <typename F, int... I>
__device__ __forceinline__ void sweeps_of(F& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void sweeps(F f) { sweeps_of(f, std::make_integer_sequence<int, N>{}); }

// n / d for n < 2^24 as a multiplication: the kernels divide by run-time sizes in front of their first load
struct Div {
  uint32_t m, s;
  __device__ __forceinline__ int of(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> s); }
};

// How the work is cut (see cut_up()); part of the kernel arguments.
struct Cut {
  int S, nslab;             // channels of a slab (a multiple of the group and of the piece), slabs of a sample
  int PP, kcols;            // pieces of a tile's row; column chunks of a slab (1 unless a slab's row is wider than the workgroup)
  int RPI, nv, rows, krows; // pixels per sweep of the workgroup, sweeps, pixels of a tile, tiles down a sample
  int K, GS, logW;          // tiles of a cluster, groups of a slab, log2 of the lanes per group (a team) in the reductions
  int seg, logseg;          // channels of a run: the largest power of two that divides the group and the piece
  int polls;
  int phase;                // PH_* in the low two bits, above them (forward) the first workgroup of this launch: a word of its own took
                            // the scalar registers of others (1 x 2^21 x 2 bf16: 13.9 us, so 13.6, without it 13.6)
  Div by_nslab, by_K, by_PP, by_Cg, by_runs;
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

__device__ __forceinline__ void publish(unsigned long long* w, float v) {
  __hip_atomic_store(w, (1ull << 32) | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* w) {
  return __hip_atomic_load(const_cast<unsigned long long*>(w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// One tile as a thread sees it.
struct Tile {
  int kc, row0, nrow;  // column chunk, first pixel, pixels
  int cb, ce;          // channels [cb, ce)
  int r0, piece, c;    // this thread's first row, piece and channel
  int mine;            // its rows are r0, r0 + RPI, ... while this, less RPI a sweep, stays positive; 0: it has none
};
template <int VE>
__device__ __forceinline__ Tile tile_of(const GnArgs& a, int slab, int k, int thread) {
  const Cut& q = a.cut;
  Tile t;
  int kr = k;
  t.kc = 0;
  if (q.kcols > 1) {
    kr = k / q.kcols;
    t.kc = k - kr * q.kcols;
  }
  const int cs = slab * q.S, cend = min(cs + q.S, a.C);
  t.cb = cs + t.kc * q.PP * VE;
  t.ce = min(t.cb + q.PP * VE, cend);
  t.row0 = kr * q.rows;
  t.nrow = min(q.rows, a.HW - t.row0);
  t.r0 = q.by_PP.of(thread);
  t.piece = thread - t.r0 * q.PP;
  t.c = t.cb + t.piece * VE;
  const bool active = t.r0 < q.RPI && t.c < t.ce;
  t.mine = active ? t.nrow - t.r0 : 0;
  return t;
}
// channels of group g (of the slab) in column chunk kc
__device__ __forceinline__ int columns_of(const GnArgs& a, int slab, int kc, int g, int VE) {
  const int cs = slab * a.cut.S;
  const int cb = cs + kc * a.cut.PP * VE, ce = min(cb + a.cut.PP * VE, min(cs + a.cut.S, a.C));
  const int lo = max(cs + g * a.Cg, cb), hi = min(cs + (g + 1) * a.Cg, ce);
  return max(hi - lo, 0);
}
__device__ __forceinline__ int groups_of(const GnArgs& a, int slab) { return min(a.cut.GS, a.G - slab * a.cut.GS); }

// Where a thread's first piece is; rows it does not have are read from the tile's last one (unconditional loads: all in flight at once).
template <typename T, int VE>
struct Source {
  const char* p;
  long long step;
  __device__ __forceinline__ Source(const GnArgs& a, int n, const Tile& t) {
    const int c = t.c < t.ce ? t.c : t.cb;
    const bool second = c >= a.C0;
    const long long ld = second ? a.ld1 : a.ld0, sn = second ? a.sn1 : a.sn0;
    step = ld * (a.cut.RPI * (int)sizeof(T));
    p = (second ? a.src1 : a.src0) + ((long long)n * sn + (long long)(t.row0 + min(t.r0, t.nrow - 1)) * ld + (c - (second ? a.C0 : 0))) * (long long)sizeof(T);
  }
};

// The cluster's words of this (sample, slab): [K][GS][2].  Adds them per group, in 64 bits, in a fixed order: for the forward pass
// (MOMENTS) count * mean and squares + count * mean^2.  Returns the first tile whose words have not come, or -1 with the sums in out[].
template <int VE, bool MOMENTS>
__device__ __forceinline__ int gather(const GnArgs& a, int slab, const unsigned long long* words, int* missing, double2* out) {
  const Cut& q = a.cut;
  const int thread = fresh_thread();
  const int g = thread >> q.logW, W = 1 << q.logW, l = thread & (W - 1);
  if (thread == 0) *missing = 0x7fffffff;
  __syncthreads();
  double s1 = 0.0, s2 = 0.0;
  if (g < groups_of(a, slab)) {
    constexpr int U = 2;      // tiles asked for at once
#pragma unroll 1
    for (int k0 = l; k0 < q.K; k0 += U * W) {
      unsigned long long w0[U], w1[U];
      int miss = 0;
      for (int i = 0; i < q.polls; ++i) {
        miss = 0x7fffffff;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (k0 + u * W < q.K) {
            const unsigned long long* w = words + ((size_t)(k0 + u * W) * q.GS + g) * 2;
            w0[u] = peek(w);
            w1[u] = peek(w + 1);
          }
        }
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
          if (k0 + u * W < q.K && !((w0[u] >> 32) && (w1[u] >> 32))) miss = k0 + u * W;
        if (miss == 0x7fffffff) break;
        __builtin_amdgcn_s_sleep(1);
      }
      if (miss != 0x7fffffff) {
        atomicMin(missing, miss);
        break;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * W;
        if (k < q.K) {
          const double x0 = (double)__uint_as_float((unsigned)w0[u]), x1 = (double)__uint_as_float((unsigned)w1[u]);
          if constexpr (MOMENTS) {
            int kr = k, kc = 0;
            if (q.kcols > 1) {
              kr = k / q.kcols;
              kc = k - kr * q.kcols;
            }
            const double cnt = (double)min(q.rows, a.HW - kr * q.rows) * (double)columns_of(a, slab, kc, g, VE);
            s1 += cnt * x0;
            s2 += x1 + cnt * x0 * x0;
          } else {
            s1 += x0;
            s2 += x1;
          }
        }
      }
    }
  }
  for (int o = W >> 1; o > 0; o >>= 1) {
    s1 += __shfl_xor(s1, o);
    s2 += __shfl_xor(s2, o);
  }
  if (l == 0 && g < q.GS) out[g] = make_double2(s1, s2);
  __syncthreads();
  const int m = *missing;
  __syncthreads();
  return m == 0x7fffffff ? -1 : m;
}

// gamma * (1 + s) and beta * (1 + s) + t of one channel, in two steps: the loads are issued in front of the tile's (they come back in
// order: behind them they would be waited for together with the whole tile), the arithmetic is done later
template <typename T>
struct Affine {
  float w, b;
  uint32_t s, t;      // as stored
  __device__ __forceinline__ void load(const GnArgs& a, int n, int c) {
    w = a.gamma[c];
    b = a.beta[c];
    s = t = 0;
    const long long i = (long long)n * a.film_ld + c;
    if (a.film_kind == 1) {
      s = ((const uint32_t*)a.film)[i];
      t = ((const uint32_t*)a.film)[i + a.C];
    } else if (a.film_kind == 2) {
      s = ((const typename Piece<T, 1>::mem*)a.film)[i];
      t = ((const typename Piece<T, 1>::mem*)a.film)[i + a.C];
    }
  }
  __device__ __forceinline__ float2 get(int film_kind) const {
    typedef typename Piece<T, 1>::mem mem_t;
    const float gain = 1.0f + (film_kind == 2 ? (float)__builtin_bit_cast(T, (mem_t)s) : __uint_as_float(s));
    const float shift = film_kind == 2 ? (float)__builtin_bit_cast(T, (mem_t)t) : __uint_as_float(t);
    return make_float2(w * gain, __builtin_fmaf(b, gain, shift));
  }
};
// that of the thread's own first channel of the tile (channel threadIdx.x; any other one's where there is none)
template <typename T>
__device__ __forceinline__ Affine<T> first_affine(const GnArgs& a, int n, const Tile& t) {
  Affine<T> f;
  f.load(a, n, t.cb + min((int)threadIdx.x, t.ce - t.cb - 1));
  return f;
}
template <int VE>
__device__ __forceinline__ void read_channels(const float* ch, int piece, float* f) {
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = ch[piece * VE + e];
}
// f(j, coefficients) for this thread's channels of the tile; `first` = those of channel threadIdx.x, loaded long before
template <int NT, typename T, typename F>
__device__ __forceinline__ void each_channel(const GnArgs& a, int n, const Tile& t, const Affine<T>& first, F f) {
  const int ncol = t.ce - t.cb;
  if ((int)threadIdx.x < ncol) f((int)threadIdx.x, first.get(a.film_kind));
  for (int j = threadIdx.x + NT; j < ncol; j += NT) {
    Affine<T> other;
    other.load(a, n, t.cb + j);
    f(j, other.get(a.film_kind));
  }
}

// ---- forward ----
// v[] over the channels of a piece -> its sums over runs of q.seg channels (each inside one group), at every q.seg-th place
template <int VE>
__device__ __forceinline__ void add_runs(const Cut& q, float* v) {
  if constexpr (VE >= 2) {
    if (q.seg >= 2) {
#pragma unroll
      for (int e = 0; e < VE; e += 2) v[e] += v[e + 1];
    }
  }
  if constexpr (VE >= 4) {
    if (q.seg >= 4) {
#pragma unroll
      for (int e = 0; e < VE; e += 4) v[e] += v[e + 2];
    }
  }
  if constexpr (VE >= 8) {
    if (q.seg >= 8) v[0] += v[4];
  }
}
// Sums over the tile of M values a channel and thread, per group: gs[m][g] (LDS), the same order for every workgroup.  A run is one word
// in LDS (red[m], NT * VE of them); a team of W lanes adds its group's.
template <int VE, int M>
__device__ __forceinline__ void group_sums(const GnArgs& a, const Tile& t, int slab, float (&v)[M][VE], float* const (&red)[M], float* const (&gs)[M]) {
  const Cut& q = a.cut;
  const int thread = fresh_thread();
#pragma unroll
  for (int k = 0; k < M; ++k) add_runs<VE>(q, v[k]);
  const int RS = q.PP * (VE >> q.logseg);      // runs of a row
  if (thread < q.RPI * q.PP) {
    const int first = (thread * VE) >> q.logseg;      // a thread's runs follow those of the thread in front
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if ((e & (q.seg - 1)) == 0) {
#pragma unroll
        for (int k = 0; k < M; ++k) red[k][first + (e >> q.logseg)] = v[k][e];
      }
  }
  __syncthreads();
  const int g = thread >> q.logW, W = 1 << q.logW, l = thread & (W - 1);
  const int c0 = slab * q.S + g * a.Cg;
  const int lo = (max(c0, t.cb) - t.cb) >> q.logseg, hi = g < groups_of(a, slab) ? (min(c0 + a.Cg, t.ce) - t.cb) >> q.logseg : 0;
  const int w = max(hi - lo, 0), rows = min(q.RPI, t.nrow);
  float sum[M];
#pragma unroll
  for (int k = 0; k < M; ++k) sum[k] = 0.f;
  if (w > 0) {
    const bool whole = w == a.Cg >> q.logseg;
    const int dr = whole ? q.by_runs.of(W) : W / w, dj = W - dr * w;
    int row = whole ? q.by_runs.of(l) : l / w;
    int j = l - row * w;
    while (row < rows) {
#pragma unroll
      for (int k = 0; k < M; ++k) sum[k] += red[k][row * RS + lo + j];
      row += dr;
      j += dj;
      if (j >= w) { j -= w; ++row; }
    }
  }
  for (int o = W >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < M; ++k) sum[k] += __shfl_xor(sum[k], o);
  }
  if (l == 0 && g < q.GS) {
#pragma unroll
    for (int k = 0; k < M; ++k) gs[k][g] = sum[k];
  }
  __syncthreads();
}

// A thread's channel sums s[] -> the means of the tile's groups in gmean[] (LDS) and, of each of the thread's channels, in m[].
template <int VE>
__device__ __forceinline__ void tile_means(const GnArgs& a, const Tile& t, int slab, float (&s)[1][VE], float* m, float* red, float* gmean) {
  const Cut& q = a.cut;
  group_sums<VE, 1>(a, t, slab, s, {red}, {gmean});
  const int g = fresh_thread();
  if (g < groups_of(a, slab)) gmean[g] /= fmaxf((float)t.nrow * (float)columns_of(a, slab, t.kc, g, VE), 1.f);
  __syncthreads();
  const int c = min(t.c, t.ce - 1);
  int ge = q.by_Cg.of(c), r = c - ge * a.Cg;
  ge -= slab * q.GS;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    m[e] = gmean[min(ge, MAX_GS - 1)];
    if (++r == a.Cg) { r = 0; ++ge; }
  }
}

// The sums of a tile that another workgroup holds, by streaming over it (gather() did not find them): the same operations in the
// same order as in the kernel.
template <typename T, int VE>
__device__ __forceinline__ void help_forward(const GnArgs& a, int n, int slab, int k, float* red, float* gmean, float* gsq) {
  const Tile t = tile_of<VE>(a, slab, k, fresh_thread());
  float s[1][VE], m[VE];
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int e = 0; e < VE; ++e) s[0][e] = 0.f;
    Source<T, VE> src(a, n, t);
#pragma unroll 1
    for (int left = t.mine; left > 0; left -= a.cut.RPI) {
      float f[VE];
      unpack<T, VE>(*(const typename Piece<T, VE>::mem*)src.p, f);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (pass == 0) s[0][e] += f[e];
        else { const float d = f[e] - m[e]; s[0][e] = __builtin_fmaf(d, d, s[0][e]); }
      }
      src.p += src.step;
    }
    if (pass == 0) tile_means<VE>(a, t, slab, s, m, red, gmean);
  }
  group_sums<VE, 1>(a, t, slab, s, {red}, {gsq});
}

template <int NT, typename T, int VE, int NV>
__global__ __launch_bounds__(NT, 4) void gn_act_fwd_kernel(GnArgs a, char* __restrict__ out, float* __restrict__ stats,
                                                           unsigned long long* words, const double2* __restrict__ totals) {
  typedef typename Piece<T, VE>::reg reg_t;
  typedef typename Piece<T, VE>::mem mem_t;
  // the threads' sums; afterwards, per channel, the mean and scale
  __shared__ __attribute__((aligned(16))) float red[NT * VE < 2 * MAX_COL ? 2 * MAX_COL : NT * VE];
  __shared__ __attribute__((aligned(16))) float chW[MAX_COL], chB[MAX_COL];      // per channel gamma * (1 + s), beta * (1 + s) + t
  __shared__ float gsq[MAX_GS], gmean[MAX_GS], grstd[MAX_GS];
  __shared__ double2 tot[MAX_GS];
  __shared__ int missing;
  const Cut& q = a.cut;
  const int block = (q.phase >> 2) + blockIdx.x;
  const int rest = q.by_K.of(block), me = block - rest * q.K;      // a cluster's tiles start together
  const int n = q.by_nslab.of(rest), slab = rest - n * q.nslab;
  const Tile t = tile_of<VE>(a, slab, me, threadIdx.x);

  const Affine<T> first = first_affine<T>(a, n, t);
  // ---- the tile into registers ----
  reg_t x[NV];
  {
    Source<T, VE> src(a, n, t);
    int left = t.mine;
    forget(left);
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      x[i] = *(const mem_t*)src.p;
      src.p += left > q.RPI ? src.step : 0;
      left -= q.RPI;
      __builtin_amdgcn_sched_barrier(0);      // else all addresses are computed first and take the registers
    });
  }
  each_channel<NT, T>(a, n, t, first, [&](int j, float2 wb) __attribute__((always_inline)) {
    chW[j] = wb.x;
    chB[j] = wb.y;
  });
  // ---- means and centred squares ----
  float s[1][VE], m[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) s[0][e] = 0.f;
  {
    int left = t.mine;
    forget(left);
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      if (left > 0) {
        float f[VE];
        forget(x[i]);
        unpack<T, VE>(x[i], f);
#pragma unroll
        for (int e = 0; e < VE; ++e) s[0][e] += f[e];
      }
      left -= q.RPI;
    });
    tile_means<VE>(a, t, slab, s, m, red, gmean);
#pragma unroll
    for (int e = 0; e < VE; ++e) s[0][e] = 0.f;
    left = t.mine;
    forget(left);
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      if (left > 0) {
        float f[VE];
        forget(x[i]);
        unpack<T, VE>(x[i], f);
#pragma unroll
        for (int e = 0; e < VE; ++e) { const float d = f[e] - m[e]; s[0][e] = __builtin_fmaf(d, d, s[0][e]); }
      }
      left -= q.RPI;
    });
    group_sums<VE, 1>(a, t, slab, s, {red}, {gsq});
  }
  const int GS = groups_of(a, slab), g = threadIdx.x;
  if (q.K == 1) {
    if (g < GS) grstd[g] = 1.0f / sqrtf(gsq[g] / ((float)a.HW * (float)a.Cg) + a.eps);
  } else {
    if ((q.phase & 3) != PH_RESULT) {
      unsigned long long* const cluster = words + ((size_t)n * q.nslab + slab) * q.K * q.GS * 2;
      for (int k = me;;) {
        if (g < GS) {
          publish(cluster + ((size_t)k * q.GS + g) * 2, gmean[g]);
          publish(cluster + ((size_t)k * q.GS + g) * 2 + 1, gsq[g]);
        }
        if ((q.phase & 3) == PH_SUMS) return;
        k = gather<VE, true>(a, slab, cluster, &missing, tot);
        if (k < 0) break;
        help_forward<T, VE>(a, n, slab, k, red, gmean, gsq);
      }
    }
    if (g < GS) {
      const double2 sum = (q.phase & 3) == PH_RESULT ? totals[((size_t)n * q.nslab + slab) * q.GS + g] : tot[g];
      const double M = (double)a.HW * (double)a.Cg, mean = sum.x / M;
      const double var = fmax(sum.y / M - mean * mean, 0.0);
      gmean[g] = (float)mean;
      // a NaN sum stays one: fmax would drop it
      grstd[g] = sum.y == sum.y ? (float)(1.0 / sqrt(var + (double)a.eps)) : __builtin_nanf("");
    }
  }
  __syncthreads();
  if (me == 0 && g < GS) {
    const size_t i = ((size_t)n * a.G + slab * q.GS + g) * 2;
    stats[i] = gmean[g];
    stats[i + 1] = grstd[g];
  }
  float *const chM = red, *const chS = red + MAX_COL;
  for (int j = g; j < t.ce - t.cb; j += NT) {
    const int gj = q.by_Cg.of(t.cb + j) - slab * q.GS;
    chM[j] = gmean[gj];
    chS[j] = chW[j] * grstd[gj];
  }
  __syncthreads();
  if (t.mine <= 0) return;
  // ---- the result ----
  loads_done();
  float sc[VE], bb[VE];
  read_channels<VE>(chM, t.piece, m);
  read_channels<VE>(chS, t.piece, sc);
  read_channels<VE>(chB, t.piece, bb);
  if (a.drop) drop_resolve(a.rng);
  long long o = ((long long)n * a.HW + t.row0 + t.r0) * a.C + t.c;
  const long long ostep = (long long)q.RPI * a.C;
  int left = t.mine;
  forget(left);
  sweeps<NV>([&](auto i) __attribute__((always_inline)) {
    if (left > 0) {
      float f[VE];
      forget(x[i]);
      unpack<T, VE>(x[i], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = __builtin_fmaf(f[e] - m[e], sc[e], bb[e]);
      if (a.act) {
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = silu_f(f[e]);
      }
      if (a.drop) drop_apply<VE>(a.rng, (unsigned long long)o, f);
      __builtin_nontemporal_store(pack<T, VE>(f), (mem_t*)(out + o * (long long)sizeof(T)));
    }
    o += ostep;
    left -= q.RPI;
  });
}

// ---- backward ----
// d: dy -> gv, f: x -> xc, of one piece; o = its index in dy
template <int VE>
__device__ __forceinline__ void gradient_of(const GnArgs& a, long long o, const float* m, const float* sc, const float* bb, float* f, float* d) {
  if (a.drop) drop_apply<VE>(a.rng, (unsigned long long)o, d);
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] -= m[e];
  if (a.act) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float v = __builtin_fmaf(f[e], sc[e], bb[e]);
      const float sg = __builtin_amdgcn_rcpf(1.0f + __expf(-v));
      d[e] *= sg * __builtin_fmaf(v, 1.0f - sg, 1.0f);
    }
  }
}

struct BwdShared {
  float *redA, *redB, *chM, *chW, *chA, *chB, *gmean, *grstd, *gm1, *gm2;
};
// per channel mean, gamma * (1 + s), offset, scale into LDS
template <int NT, typename T>
__device__ __forceinline__ void bwd_channels(const GnArgs& a, int n, int slab, const Tile& t, const Affine<T>& first, const BwdShared& h) {
  each_channel<NT, T>(a, n, t, first, [&](int j, float2 wb) __attribute__((always_inline)) {
    const int gj = a.cut.by_Cg.of(t.cb + j) - slab * a.cut.GS;
    h.chM[j] = h.gmean[gj];
    h.chW[j] = wb.x;
    h.chA[j] = wb.y;
    h.chB[j] = wb.x * h.grstd[gj];
  });
  __syncthreads();
}
// The threads' channel sums A, B (of gv and gv * xc) -> the sums of g and g * xhat of the tile's groups, gm1 and gm2.
template <int VE>
__device__ __forceinline__ void group_gradients(const GnArgs& a, const Tile& t, int slab, const float* A, const float* B, const BwdShared& h) {
  float gw[VE], sc[VE], v[2][VE];
  read_channels<VE>(h.chW, t.piece, gw);
  read_channels<VE>(h.chB, t.piece, sc);
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    v[0][e] = t.mine > 0 ? A[e] * gw[e] : 0.f;
    v[1][e] = t.mine > 0 ? B[e] * sc[e] : 0.f;
  }
  group_sums<VE, 2>(a, t, slab, v, {h.redA, h.redB}, {h.gm1, h.gm2});
}
// ... -> those of the tile's channels, of gv and gv * xhat: done(j, A, B) for each.
template <int NT, int VE, typename F>
__device__ __forceinline__ void channel_gradients(const GnArgs& a, const Tile& t, int slab, const float* A, const float* B, const BwdShared& h, F done) {
  const Cut& q = a.cut;
  const int thread = fresh_thread();
  const int RS = q.PP * VE + 8, ncol = t.ce - t.cb;      // (padded: several rows are read at once)
  if (t.r0 < q.RPI) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      h.redA[t.r0 * RS + t.piece * VE + e] = A[e];
      h.redB[t.r0 * RS + t.piece * VE + e] = B[e];
    }
  }
  __syncthreads();
  const int rows = min(q.RPI, t.nrow);
  const int parts = ncol < NT ? NT / ncol : 1;
  int nr = rows, rs = RS;
  if (parts > 1) {
    const int p = thread / ncol, j = thread - p * ncol;
    float sa = 0.f, sb = 0.f;
    if (p < parts) {
#pragma unroll 4
      for (int r = p; r < rows; r += parts) { sa += h.redA[r * RS + j]; sb += h.redB[r * RS + j]; }
    }
    __syncthreads();
    if (p < parts) { h.redA[p * ncol + j] = sa; h.redB[p * ncol + j] = sb; }
    __syncthreads();
    nr = min(parts, rows);
    rs = ncol;
  }
  for (int j = thread; j < ncol; j += NT) {
    float sa = 0.f, sb = 0.f;
    for (int r = 0; r < nr; ++r) { sa += h.redA[r * rs + j]; sb += h.redB[r * rs + j]; }
    done(j, sa, sb * h.grstd[q.by_Cg.of(t.cb + j) - slab * q.GS]);
  }
}

template <int NT, typename T, int VE>
__device__ __forceinline__ void help_backward(const GnArgs& a, int n, int slab, int k, const char* dy, const BwdShared& h) {
  typedef typename Piece<T, VE>::mem mem_t;
  const Tile t = tile_of<VE>(a, slab, k, fresh_thread());
  bwd_channels<NT, T>(a, n, slab, t, first_affine<T>(a, n, t), h);
  float m[VE], sc[VE], bb[VE], A[VE], B[VE];
  read_channels<VE>(h.chM, t.piece, m);
  read_channels<VE>(h.chA, t.piece, bb);
  read_channels<VE>(h.chB, t.piece, sc);
#pragma unroll
  for (int e = 0; e < VE; ++e) A[e] = B[e] = 0.f;
  Source<T, VE> src(a, n, t);
  long long o = ((long long)n * a.HW + t.row0 + t.r0) * a.C + t.c;
#pragma unroll 1
  for (int left = t.mine; left > 0; left -= a.cut.RPI) {
    float f[VE], d[VE];
    unpack<T, VE>(*(const mem_t*)src.p, f);
    unpack<T, VE>(*(const mem_t*)(dy + o * (long long)sizeof(T)), d);
    gradient_of<VE>(a, o, m, sc, bb, f, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) { A[e] += d[e]; B[e] = __builtin_fmaf(d[e], f[e], B[e]); }
    src.p += src.step;
    o += (long long)a.cut.RPI * a.C;
  }
  group_gradients<VE>(a, t, slab, A, B, h);
}

template <int NT, typename T, int VE, int NV>
__global__ __launch_bounds__(NT, 2) void gn_act_bwd_kernel(GnArgs a, const float* __restrict__ stats, const char* __restrict__ dy,
                                                           char* __restrict__ d0, char* __restrict__ d1, unsigned long long* words,
                                                           const double2* __restrict__ totals, float2* __restrict__ part) {
  typedef typename Piece<T, VE>::reg reg_t;
  typedef typename Piece<T, VE>::mem mem_t;
  __shared__ __attribute__((aligned(16))) float redA[NT * (VE + 8)], redB[NT * (VE + 8)];
  // per channel: mean, gamma * (1 + s), offset and scale; afterwards the coefficients of the result
  __shared__ __attribute__((aligned(16))) float chM[MAX_COL], chW[MAX_COL], chA[MAX_COL], chB[MAX_COL];
  __shared__ float gmean[MAX_GS], grstd[MAX_GS], gm1[MAX_GS], gm2[MAX_GS];
  __shared__ double2 tot[MAX_GS];
  __shared__ int missing;
  BwdShared h;      // (assigned: an initialiser list would be a constant with LDS addresses)
  h.redA = redA; h.redB = redB; h.chM = chM; h.chW = chW; h.chA = chA; h.chB = chB;
  h.gmean = gmean; h.grstd = grstd; h.gm1 = gm1; h.gm2 = gm2;
  const Cut& q = a.cut;
  const int rest = q.by_K.of(blockIdx.x), me = blockIdx.x - rest * q.K;      // a cluster's tiles start together
  const int n = q.by_nslab.of(rest), slab = rest - n * q.nslab;
  const Tile t = tile_of<VE>(a, slab, me, threadIdx.x);
  const int GS = groups_of(a, slab), g = threadIdx.x;
  const long long o0 = ((long long)n * a.HW + t.row0 + t.r0) * a.C + t.c, ostep = (long long)q.RPI * a.C;

  unsigned long long* const cluster = words + ((size_t)n * q.nslab + slab) * q.K * q.GS * 2;

  reg_t x[NV];
  float gv[NV][VE];
  {
    // ---- the tile into registers ----
    const Affine<T> first = first_affine<T>(a, n, t);
    const float2 stat = ((const float2*)stats)[(size_t)n * a.G + slab * q.GS + min(g, GS - 1)];
    reg_t dd[NV];
    Source<T, VE> src(a, n, t);
    const char* pd = dy + (t.mine > 0 ? o0 : ((long long)n * a.HW + t.row0) * a.C + t.cb) * (long long)sizeof(T);
    int left = t.mine;
    forget(left);
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      x[i] = *(const mem_t*)src.p;
      dd[i] = *(const mem_t*)pd;
      src.p += left > q.RPI ? src.step : 0;
      pd += left > q.RPI ? ostep * (long long)sizeof(T) : 0;
      left -= q.RPI;
      __builtin_amdgcn_sched_barrier(0);      // else all addresses are computed first and take the registers
    });
    if (g < GS) {
      gmean[g] = stat.x;
      grstd[g] = stat.y;
    }
    if (a.drop) drop_resolve(a.rng);
    __syncthreads();
    bwd_channels<NT, T>(a, n, slab, t, first, h);
    // ---- gv and the channels' sums ----
    float m[VE], bb[VE], sc[VE], A[VE], B[VE];
    read_channels<VE>(chM, t.piece, m);
    read_channels<VE>(chA, t.piece, bb);
    read_channels<VE>(chB, t.piece, sc);
#pragma unroll
    for (int e = 0; e < VE; ++e) A[e] = B[e] = 0.f;
    left = t.mine;
    forget(left);
    long long o = o0;
    sweeps<NV>([&](auto i) __attribute__((always_inline)) {
      if (left > 0) {
        float f[VE], d[VE];
        forget(x[i]);
        unpack<T, VE>(x[i], f);
        unpack<T, VE>(dd[i], d);
        gradient_of<VE>(a, o, m, sc, bb, f, d);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          gv[i][e] = d[e];
          A[e] += d[e];
          B[e] = __builtin_fmaf(d[e], f[e], B[e]);
        }
      }
      o += ostep;
      left -= q.RPI;
    });
    // the groups' sums go out first: the others wait for them while the channels' are added
    group_gradients<VE>(a, t, slab, A, B, h);
    if (q.K > 1 && q.phase != PH_RESULT && g < GS) {
      publish(cluster + ((size_t)me * q.GS + g) * 2, gm1[g]);
      publish(cluster + ((size_t)me * q.GS + g) * 2 + 1, gm2[g]);
    }
    channel_gradients<NT, VE>(a, t, slab, A, B, h, [&](int j, float sa, float sb) __attribute__((always_inline)) {
      part[((size_t)n * q.krows + (q.kcols > 1 ? me / q.kcols : me)) * a.C + t.cb + j] = make_float2(sa, sb);
    });
  }
  if (q.phase == PH_SUMS) return;
  const float Mf = (float)a.HW * (float)a.Cg;
  if (q.K > 1) {
    bool helped = false;
    if (q.phase != PH_RESULT) {
      for (;;) {
        const int k = gather<VE, false>(a, slab, cluster, &missing, tot);
        if (k < 0) break;
        help_backward<NT, T, VE>(a, n, slab, k, dy, h);
        helped = true;
        if (g < GS) {
          publish(cluster + ((size_t)k * q.GS + g) * 2, gm1[g]);
          publish(cluster + ((size_t)k * q.GS + g) * 2 + 1, gm2[g]);
        }
      }
    }
    if (g < GS) {
      const double2 sum = q.phase == PH_RESULT ? totals[((size_t)n * q.nslab + slab) * q.GS + g] : tot[g];
      const double M = (double)a.HW * (double)a.Cg;
      gm1[g] = (float)(sum.x / M);
      gm2[g] = (float)(sum.y / M);
    }
    if (helped && q.kcols > 1) {      // another column chunk's channels are in LDS now
      __syncthreads();
      bwd_channels<NT, T>(a, n, slab, t, first_affine<T>(a, n, t), h);
    }
  } else if (g < GS) {
    gm1[g] /= Mf;
    gm2[g] /= Mf;
  }
  __syncthreads();
  // dx = gv * (rstd * gamma * (1 + s)) - rstd * sum(g) / M - xc * (rstd^2 * sum(g * xhat) / M); one value a group has no gradient, which
  // three rounded coefficients would miss by a rounding of terms that are 1 / sqrt(eps) large
  const bool alone = Mf == 1.0f;
  for (int j = threadIdx.x; j < t.ce - t.cb; j += NT) {
    const int gj = q.by_Cg.of(t.cb + j) - slab * q.GS;
    const float rs = alone ? 0.f : grstd[gj];
    chA[j] = gm1[gj] * rs;
    chB[j] = gm2[gj] * rs * rs;
    chW[j] *= rs;
  }
  __syncthreads();
  if (t.mine <= 0) return;
  // ---- the result ----
  loads_done();
  const bool second = t.c >= a.C0;
  const long long ld = second ? a.C - a.C0 : a.C0;
  char* o = (second ? d1 : d0) + (((long long)n * a.HW + t.row0 + t.r0) * ld + (t.c - (second ? a.C0 : 0))) * (long long)sizeof(T);
  const long long ostep2 = ld * (q.RPI * (int)sizeof(T));
  int left = t.mine;
  forget(left);
  float m[VE], k0[VE], k1[VE], k2[VE];
  read_channels<VE>(chM, t.piece, m);
  read_channels<VE>(chW, t.piece, k0);
  read_channels<VE>(chA, t.piece, k1);
  read_channels<VE>(chB, t.piece, k2);
  sweeps<NV>([&](auto i) __attribute__((always_inline)) {
    if (left > 0) {
      float f[VE];
      forget(x[i]);
      unpack<T, VE>(x[i], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = __builtin_fmaf(gv[i][e], k0[e], __builtin_fmaf(m[e] - f[e], k2[e], -k1[e]));
      __builtin_nontemporal_store(pack<T, VE>(f), (mem_t*)o);
    }
    o += ostep2;
    left -= q.RPI;
  });
}

// the words of one cluster added up, between PH_SUMS and PH_RESULT: one workgroup per (sample, slab)
template <int NT, int VE, bool MOMENTS>
__global__ __launch_bounds__(NT) void gn_act_total_kernel(GnArgs a, const unsigned long long* words, double2* __restrict__ totals) {
  __shared__ double2 tot[MAX_GS];
  __shared__ int missing;
  const Cut& q = a.cut;
  const int slab = blockIdx.x % q.nslab;
  gather<VE, MOMENTS>(a, slab, words + (size_t)blockIdx.x * q.K * q.GS * 2, &missing, tot);
  if (threadIdx.x < groups_of(a, slab)) totals[(size_t)blockIdx.x * q.GS + threadIdx.x] = tot[threadIdx.x];
}

// zeroes the clusters' words (a kernel, so that it may be captured)
__global__ __launch_bounds__(NT_AUX) void gn_act_clear_kernel(ulonglong2* words, long long n) {
  const long long i = (long long)blockIdx.x * NT_AUX + threadIdx.x;
  if (i < n) words[i] = make_ulonglong2(0, 0);
}

// Between tiles and between samples the channels are added in 64 bits, as the groups are: the terms are often alike, and thousands of equal
// ones all round the same way (4096 in one fp32 sum were off by up to 800 times 2^-24).
// part [N][krows][C] -> [N][1][C]: 64 channels a workgroup, four threads a channel
__global__ __launch_bounds__(NT_AUX) void gn_act_fold_kernel(const float2* __restrict__ part, int krows, int C, float2* __restrict__ out) {
  __shared__ double2 red[NT_AUX];
  const int cblk = (C + 63) / 64;
  const int n = blockIdx.x / cblk, c = (blockIdx.x - n * cblk) * 64 + (threadIdx.x & 63), h = threadIdx.x >> 6;
  double A = 0.0, B = 0.0;
  if (c < C) {
#pragma unroll 4
    for (int k = h; k < krows; k += NT_AUX / 64) {
      const float2 v = part[((size_t)n * krows + k) * C + c];
      A += v.x;
      B += v.y;
    }
  }
  red[threadIdx.x] = make_double2(A, B);
  __syncthreads();
  if (h == 0 && c < C) {
#pragma unroll
    for (int j = 1; j < NT_AUX / 64; ++j) { A += red[threadIdx.x + 64 * j].x; B += red[threadIdx.x + 64 * j].y; }
    out[(size_t)n * C + c] = make_float2((float)A, (float)B);
  }
}

// part [N][krows][C] (A, B of a tile) -> dscale, dshift of every (n, c), dgamma, dbeta: 16 channels a workgroup, 16 threads a channel.
// Workgroup row blockIdx.y takes samples [y * per, (y + 1) * per) and leaves its sums in dgamma[y][C], dbeta[y][C].
template <typename T>
__global__ __launch_bounds__(NT_AUX) void gn_act_param_kernel(GnArgs a, const float2* __restrict__ part, int krows, int N, int per,
                                                              float* __restrict__ dgamma, float* __restrict__ dbeta, char* __restrict__ dfilm) {
  __shared__ double2 red[(NT_AUX / 64 - 1) * 16];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), h = threadIdx.x >> 4;
  double sa = 0.0, sb = 0.0;
  if (c < a.C) {
    const float gamma = a.gamma[c], beta = a.beta[c];
    const int n1 = min(N, (int)(blockIdx.y + 1) * per);
    for (int n = blockIdx.y * per + h; n < n1; n += 16) {
      double A = 0.0, B = 0.0;
      const float2* p = part + (size_t)n * krows * a.C + c;
#pragma unroll 4
      for (int k = 0; k < krows; ++k) {
        const float2 v = p[(size_t)k * a.C];
        A += v.x;
        B += v.y;
      }
      float gain = 1.0f;
      if (a.film_kind) {
        gain += film_at<T>(a, (long long)n * a.film_ld + c);
        const float ds = (float)__builtin_fma(gamma, B, beta * A), dt = (float)A;
        const long long i = (long long)n * 2 * a.C + c;
        if (a.film_kind == 1) { ((float*)dfilm)[i] = ds; ((float*)dfilm)[i + a.C] = dt; }
        else { ((T*)dfilm)[i] = (T)ds; ((T*)dfilm)[i + a.C] = (T)dt; }
      }
      sa = __builtin_fma(gain, A, sa);
      sb = __builtin_fma(gain, B, sb);
    }
  }
  // a wave's four threads of a channel, then the waves
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    sa += __shfl_xor(sa, o);
    sb += __shfl_xor(sb, o);
  }
  const int wave = threadIdx.x >> 6;
  if (wave > 0 && (threadIdx.x & 63) < 16) red[(wave - 1) * 16 + (threadIdx.x & 15)] = make_double2(sa, sb);
  __syncthreads();
  if (h == 0 && c < a.C) {
#pragma unroll
    for (int j = 0; j < NT_AUX / 64 - 1; ++j) { sa += red[j * 16 + threadIdx.x].x; sb += red[j * 16 + threadIdx.x].y; }
    dgamma[(size_t)blockIdx.y * a.C + c] = (float)sb;
    dbeta[(size_t)blockIdx.y * a.C + c] = (float)sa;
  }
}
// the rows of the kernel above added up
__global__ __launch_bounds__(NT_AUX) void gn_act_rows_kernel(const float* __restrict__ g, const float* __restrict__ b, int rows, int C,
                                                             float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int c = blockIdx.x * NT_AUX + threadIdx.x;
  if (c >= C) return;
  double sa = 0.0, sb = 0.0;
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    sb += g[(size_t)r * C + c];
    sa += b[(size_t)r * C + c];
  }
  dgamma[c] = (float)sb;
  dbeta[c] = (float)sa;
}

Div div_by(int d) {
  int l = 0;
  while ((1ll << l) < d) ++l;
  return Div{(uint32_t)(((1ull << (24 + l)) + d - 1) / d), (uint32_t)(24 + l)};
}
int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Sweeps that a tile may have (instantiations): 16-byte pieces take the smallest count that holds a sample's pixels, else the largest.
// Narrower pieces have two.
constexpr int SWEEPS_FWD[] = {2, 4, 8, 16}, SWEEPS_BWD[] = {2, 4, 8, 12}, SWEEPS_NARROW[] = {4, 16};
int sweeps_for(int ve, int esz, bool backward, long long needed) {
  if (ve * esz < 16) return SWEEPS_NARROW[needed > SWEEPS_NARROW[0]];
  const int* list = backward ? SWEEPS_BWD : SWEEPS_FWD;
  int i = 0;
  while (i < 3 && list[i] < needed) ++i;
  return list[i];
}

// Prices of the choice below, from measurements at 8 x 8 .. 128 x 128 pixels.  The choice by cost against a fixed one: 64 x 16 x 16 x 1792
// fp16 forward 32 -> 27 us, backward 66 -> 56; 64 x 16 x 16 x 768 bf16 backward 37 -> 34; 64 x 8 x 8 x 1024 forward 12.2 -> 9.2;
// 7 x 37 x 23 x 100 fp16 with dropout 20.8 -> 13.6.
constexpr double TILES_COST = 2.2, SETUP_SWEEPS = 3.0;

int cut_up(const ivid_gn_act_desc* d, bool backward, GnArgs* a, int* ve_out) {
  const int NT = backward ? NT_BWD : NT_FWD;
  const int esz = ivid_esz(d->dtype);
  // the widest piece that every row of every tensor is a whole number of
  int ve = 16 / esz;
  auto fits = [&](int v) {
    const long long mask = v - 1;
    return !((d->C0 | d->C1 | d->ld0 | d->sn0 | (d->C1 ? d->ld1 | d->sn1 : 0)) & mask) && !((uintptr_t)d->src0 % (v * esz)) &&
           !((uintptr_t)d->src1 % (v * esz));
  };
  while (ve > 1 && !fits(ve)) ve >>= 1;
  const int wide = NT < MAX_COL / ve ? NT : MAX_COL / ve;      // pieces of a tile's row at most
  const int C = a->C, Cg = a->Cg;
  const long long unit = (long long)Cg / gcd(Cg, ve) * ve;     // whole groups and whole pieces
  Cut& q = a->cut;
  // The slab: whole groups, a few whole 128-byte lines of channels.  Each candidate costs the lines that two slabs share (half of their
  // traffic: the second reader mostly finds them in the last-level cache), the threads that have no piece, a workgroup's setup, worth
  // about three sweeps, and, when a tile does not hold a sample's pixels, the exchange between tiles.
  long long S = unit;
  double best = 1e30;
  for (long long s = unit; s <= C && (s == unit || (s / Cg <= MAX_GS && s / ve <= wide && s * esz <= 512)); s += unit) {
    const long long pp = s / ve < wide ? s / ve : wide, rpi = NT / pp;
    const int g = gcd((int)(s * esz % 128), 128);
    const double lines = s == C ? 1.0 : 1.0 + (128.0 - g) / (double)(s * esz);
    const double idle = (double)NT / (double)(pp * rpi);
    const long long sweeps = (d->HW + rpi - 1) / rpi;
    const double setup = 1.0 + SETUP_SWEEPS / sweeps_for(ve, esz, backward, sweeps);
    const double cost = (0.5 + 0.5 * lines) * idle * setup * (sweeps > sweeps_for(ve, esz, backward, sweeps) ? TILES_COST : 1.0) * (s * esz < 128 && s < C ? 1.5 : 1.0);
    if (cost < best * 0.999) {
      best = cost;
      S = s;
    }
  }
  q.S = (int)S;
  q.nslab = (int)((C + S - 1) / S);
  q.GS = (int)(S / Cg);
  if (q.GS > MAX_GS) return ivid_set_error("gn_act: internal: too many groups in a slab", hipSuccess);
  const int pieces = (int)(S / ve);
  q.kcols = (pieces + wide - 1) / wide;
  q.PP = (pieces + q.kcols - 1) / q.kcols;
  q.RPI = NT / q.PP;
  for (q.seg = 1, q.logseg = 0; q.seg < ve && Cg % (2 * q.seg) == 0;) { q.seg *= 2; ++q.logseg; }
  q.logW = 6;
  while ((q.GS << q.logW) > NT) --q.logW;
  q.nv = sweeps_for(ve, esz, backward, ((long long)d->HW + q.RPI - 1) / q.RPI);
  q.rows = q.RPI * q.nv;
  q.krows = (int)(((long long)d->HW + q.rows - 1) / q.rows);
  if (q.krows > 1 && (long long)q.nslab * q.krows * q.kcols < MIN_TILES && q.nv > 4) {
    // a cluster anyway, and so few tiles that most of the chip would stand idle for a sample or two: four sweeps a tile.  (By the sample
    // alone: its result does not depend on the batch.)
    q.nv = 4;
    q.rows = q.RPI * q.nv;
    q.krows = (int)(((long long)d->HW + q.rows - 1) / q.rows);
  }
  q.polls = d->max_polls > 0 ? d->max_polls : MAX_POLLS;
  *ve_out = ve;
  const double tiles = (double)d->N * q.nslab * q.krows * q.kcols;      // 2^24 - 1 are what Div takes, and 2^32 threads of a backward pass
  q.K = tiles < (1 << 24) ? q.krows * q.kcols : 0;
  if (!q.K || (long long)d->N * ((C + 63) / 64) >= (1 << 24))
    return ivid_set_error("gn_act: too many tiles for one launch", hipSuccess);
  q.by_nslab = div_by(q.nslab);
  q.by_K = div_by(q.K);
  q.by_PP = div_by(q.PP);
  q.by_Cg = div_by(Cg);
  q.by_runs = div_by(Cg >> q.logseg);
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
  if (!((float)d->eps > 0.0f && d->eps <= 3.4e38)) return ivid_set_error("gn_act: eps must be positive and finite in fp32", hipSuccess);
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

// The channels' sums take a launch of their own over the tiles before they are added over the samples when one thread would walk over
// more tiles than this (three microseconds of it cost as much as the launch).
constexpr int FOLD_ABOVE = 48;
// Many samples (tokens, mostly) are added in up to 64 rows of at least 256 of them.
int param_rows(int N) { return N <= 512 ? 1 : (N / 256 < 64 ? N / 256 : 64); }

// scratch: the clusters' words, (K > MAX_K) their totals, then (backward) part [N][krows][C], if folded part [N][C], if in rows [2][rows][C]
struct Scratch { long long words, totals, part, folded, rows, total; };
Scratch layout(const ivid_gn_act_desc* d, const GnArgs& a, bool backward) {
  Scratch s{};
  const Cut& q = a.cut;
  if (q.K > 1) s.words = (long long)d->N * q.nslab * q.K * q.GS * 16;
  if (q.K > MAX_K) s.totals = (long long)d->N * q.nslab * q.GS * 16;
  if (backward) {
    s.part = (long long)d->N * q.krows * a.C * 8;
    if (q.krows > 1 && (long long)q.krows * ((d->N + 15) / 16) > FOLD_ABOVE) s.folded = (long long)d->N * a.C * 8;
  }
  if (backward && param_rows(d->N) > 1) s.rows = (long long)param_rows(d->N) * a.C * 8;
  s.total = s.words + s.totals + s.part + s.folded + s.rows;
  return s;
}

int clear_words(const Scratch& s, void* scratch, hipStream_t stream) {
  if (!s.words || s.totals) return 0;      // two launches: every word is written before any is read
  const long long n = s.words / 16, blocks = (n + NT_AUX - 1) / NT_AUX;
  if (blocks >= (1 << 24)) return ivid_set_error("gn_act: too many tiles for one launch", hipSuccess);
  hipLaunchKernelGGL(gn_act_clear_kernel, dim3((unsigned)blocks), dim3(NT_AUX), 0, stream, (ulonglong2*)scratch, n);
  return 0;
}

// A workgroup that helps reads another one's inputs when that may already have written results: no output may lie over an input.
// p: `bytes` contiguous ones.  (128 bits: strides are the caller's.)
bool meets(const void* p, __int128 bytes, const void* q, __int128 qbytes) {
  const __int128 a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && a < b + qbytes && b < a + bytes;
}
__int128 source_bytes(const ivid_gn_act_desc* d, bool second) {
  const long long ld = second ? d->ld1 : d->ld0, sn = second ? d->sn1 : d->sn0;
  return ((__int128)(d->N - 1) * sn + (__int128)(d->HW - 1) * ld + (second ? d->C1 : d->C0)) * ivid_esz(d->dtype);
}
bool meets_sources(const ivid_gn_act_desc* d, const void* p, __int128 bytes) {
  return meets(p, bytes, d->src0, source_bytes(d, false)) || meets(p, bytes, d->src1, source_bytes(d, true));
}

// `run` launches the kernel once, or as sums - totals - results
template <int NT, bool MOMENTS, typename Run>
void run_phases(GnArgs& a, const ivid_gn_act_desc* d, int ve, const Scratch& s, void* scratch, hipStream_t st, Run run) {
  if (!s.totals) {
    run();
    return;
  }
  a.cut.phase = PH_SUMS;
  run();
  const dim3 grid((unsigned)((long long)d->N * a.cut.nslab));
  double2* totals = (double2*)((char*)scratch + s.words);
#define TOTAL(VE) hipLaunchKernelGGL((gn_act_total_kernel<NT, VE, MOMENTS>), grid, dim3(NT), 0, st, a, (const unsigned long long*)scratch, totals)
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
  if (meets_sources(d, out, (__int128)d->N * d->HW * a.C * ivid_esz(d->dtype))) return ivid_set_error("gn_act_forward: out overlaps a source", hipSuccess);
  const Scratch s = layout(d, a, false);
  if (scratch_bytes < s.total || (s.total && (!scratch || ((uintptr_t)scratch & 15)))) return ivid_set_error("gn_act: scratch too small or misaligned", hipSuccess);
  hipStream_t st = (hipStream_t)stream;
  if (int e = clear_words(s, scratch, st)) return e;
  // A grid of 2^32 threads is dropped without an error: several launches, and no cluster that waits is cut in two.
  const int tiles = d->N * a.cut.nslab * a.cut.K;
  int most = (int)(0xFFFFFFFFu / NT_FWD);
  if (a.cut.K <= MAX_K) most -= most % a.cut.K;
  dim3 grid;
#define LAUNCH(T, VE, NV) \
  hipLaunchKernelGGL((gn_act_fwd_kernel<NT_FWD, T, VE, NV>), grid, dim3(NT_FWD), 0, st, a, (char*)out, stats, (unsigned long long*)scratch, \
                     (const double2*)((char*)scratch + s.words))
#define LAUNCH_NV(T, VE)                                        \
  do {                                                          \
    if (a.cut.nv == SWEEPS_FWD[0]) LAUNCH(T, VE, SWEEPS_FWD[0]);   \
    else if (a.cut.nv == SWEEPS_FWD[1]) LAUNCH(T, VE, SWEEPS_FWD[1]); \
    else if (a.cut.nv == SWEEPS_FWD[2]) LAUNCH(T, VE, SWEEPS_FWD[2]); \
    else LAUNCH(T, VE, SWEEPS_FWD[3]);                            \
  } while (0)
#define LAUNCH_NARROW(T, VE)                                    \
  do {                                                          \
    if (a.cut.nv == SWEEPS_NARROW[0]) LAUNCH(T, VE, SWEEPS_NARROW[0]); \
    else LAUNCH(T, VE, SWEEPS_NARROW[1]);                        \
  } while (0)
#define LAUNCH16(T)                               \
  do {                                            \
    if (ve == 8) LAUNCH_NV(T, 8);                 \
    else if (ve == 4) LAUNCH_NARROW(T, 4);        \
    else if (ve == 2) LAUNCH_NARROW(T, 2);        \
    else LAUNCH_NARROW(T, 1);                     \
  } while (0)
  run_phases<NT_FWD, true>(a, d, ve, s, scratch, st, [&] {
    const int phase = a.cut.phase;
    for (int block0 = 0; block0 < tiles; block0 += most) {
      a.cut.phase = phase | block0 << 2;
      grid = dim3((unsigned)(tiles - block0 < most ? tiles - block0 : most));
      if (d->dtype == IVID_F32) {
        if (ve == 4) LAUNCH_NV(float, 4);
        else if (ve == 2) LAUNCH_NARROW(float, 2);
        else LAUNCH_NARROW(float, 1);
      } else if (d->dtype == IVID_BF16) {
        LAUNCH16(__bf16);
      } else {
        LAUNCH16(_Float16);
      }
    }
  });
#undef LAUNCH_NV
#undef LAUNCH_NARROW
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
      ((uintptr_t)stats & 7) || (((uintptr_t)dgamma | (uintptr_t)dbeta | (uintptr_t)dfilm) & 3))
    return ivid_set_error("gn_act_backward: NULL or misaligned pointer", hipSuccess);
  const __int128 pixels = (__int128)d->N * d->HW * ivid_esz(d->dtype);
  if (meets_sources(d, dsrc0, pixels * d->C0) || meets_sources(d, dsrc1, pixels * d->C1) || meets(dsrc0, pixels * d->C0, dy, pixels * a.C) ||
      meets(dsrc1, pixels * d->C1, dy, pixels * a.C) || meets(dsrc0, pixels * d->C0, dsrc1, pixels * d->C1))
    return ivid_set_error("gn_act_backward: dsrc0 or dsrc1 overlaps another tensor", hipSuccess);
  const Scratch s = layout(d, a, true);
  if (scratch_bytes < s.total || !scratch || ((uintptr_t)scratch & 15)) return ivid_set_error("gn_act_backward: scratch too small or misaligned", hipSuccess);
  hipStream_t st = (hipStream_t)stream;
  if (int e = clear_words(s, scratch, st)) return e;
  float2* part = (float2*)((char*)scratch + s.words + s.totals);
  const dim3 grid((unsigned)((long long)d->N * a.cut.nslab * a.cut.K));
#define LAUNCH(T, VE, NV)                                                                                              \
  hipLaunchKernelGGL((gn_act_bwd_kernel<NT_BWD, T, VE, NV>), grid, dim3(NT_BWD), 0, st, a, stats, (const char*)dy, (char*)dsrc0,   \
                     (char*)dsrc1, (unsigned long long*)scratch, (const double2*)((char*)scratch + s.words), part)
#define LAUNCH_NV(T, VE)                                        \
  do {                                                          \
    if (a.cut.nv == SWEEPS_BWD[0]) LAUNCH(T, VE, SWEEPS_BWD[0]);   \
    else if (a.cut.nv == SWEEPS_BWD[1]) LAUNCH(T, VE, SWEEPS_BWD[1]); \
    else if (a.cut.nv == SWEEPS_BWD[2]) LAUNCH(T, VE, SWEEPS_BWD[2]); \
    else LAUNCH(T, VE, SWEEPS_BWD[3]);                            \
  } while (0)
#define LAUNCH_NARROW(T, VE)                                    \
  do {                                                          \
    if (a.cut.nv == SWEEPS_NARROW[0]) LAUNCH(T, VE, SWEEPS_NARROW[0]); \
    else LAUNCH(T, VE, SWEEPS_NARROW[1]);                        \
  } while (0)
#define LAUNCH16(T)                               \
  do {                                            \
    if (ve == 8) LAUNCH_NV(T, 8);                 \
    else if (ve == 4) LAUNCH_NARROW(T, 4);        \
    else if (ve == 2) LAUNCH_NARROW(T, 2);        \
    else LAUNCH_NARROW(T, 1);                     \
  } while (0)
  run_phases<NT_BWD, false>(a, d, ve, s, scratch, st, [&] {
    if (d->dtype == IVID_F32) {
      if (ve == 4) LAUNCH_NV(float, 4);
      else if (ve == 2) LAUNCH_NARROW(float, 2);
      else LAUNCH_NARROW(float, 1);
    } else if (d->dtype == IVID_BF16) {
      LAUNCH16(__bf16);
    } else {
      LAUNCH16(_Float16);
    }
  });
#undef LAUNCH_NV
#undef LAUNCH_NARROW
#undef LAUNCH16
#undef LAUNCH
  int krows = a.cut.krows;
  if (s.folded) {
    float2* folded = (float2*)((char*)part + s.part);
    hipLaunchKernelGGL(gn_act_fold_kernel, dim3((unsigned)((long long)d->N * ((a.C + 63) / 64))), dim3(NT_AUX), 0, st, (const float2*)part, krows, a.C, folded);
    part = folded;
    krows = 1;
  }
  const int rows = param_rows(d->N), per = (d->N + rows - 1) / rows;
  float* g = s.rows ? (float*)((char*)scratch + s.total - s.rows) : dgamma;
  float* b = s.rows ? g + (size_t)rows * a.C : dbeta;
#define PARAM(T)                                                                                                                  \
  hipLaunchKernelGGL(gn_act_param_kernel<T>, dim3((unsigned)((a.C + 15) / 16), (unsigned)rows), dim3(NT_AUX), 0, st, a,           \
                     (const float2*)part, krows, d->N, per, g, b, (char*)dfilm)
  if (d->dtype == IVID_F32) PARAM(float); else if (d->dtype == IVID_BF16) PARAM(__bf16); else PARAM(_Float16);
#undef PARAM
  if (s.rows)
    hipLaunchKernelGGL(gn_act_rows_kernel, dim3((unsigned)((a.C + NT_AUX - 1) / NT_AUX)), dim3(NT_AUX), 0, st, (const float*)g, (const float*)b, rows, a.C,
                       dgamma, dbeta);
  return ivid_check_launch("gn_act_backward");
}
