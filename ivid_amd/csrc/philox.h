// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC'11): four 32-bit words, a pure
// function of (counter, key).  Shared by the Gaussian noise (elementwise.hip) and the dropout draws (dropout.hip, gn_act.hip).
#pragma once
#include <stdint.h>

// One 64-bit product per multiplier (v_mad_u64_u32) gives the high and the low word at once; the two exclusive ors of a word are one
// three-input operation.
__device__ __forceinline__ void philox4x32_10(uint32_t c[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c[1], k0, 0x96);
    const uint32_t n2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c[3], k1, 0x96);
    c[0] = n0; c[1] = (uint32_t)p1; c[2] = n2; c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
}

// Dropout draws: element i of a tensor (row-major) takes 16 bits, half i % 2 (low first) of word (i % 8) / 2 of the block with
// counter (i / 8, stream) -- eight elements a block, because ten rounds cost as much as streaming two.  The key's high word is
// tagged, so that the draws are independent of Gaussian noise with the same (seed, stream).  Kept: draw >= thr.
constexpr uint32_t DROP_KEY_TAG = 0x44524F50u;

struct DropRng {
  unsigned long long seed, stream;
  const unsigned long long* dev;  // device {seed, stream}, read by the kernel instead of the two above; or NULL
  uint32_t thr;                   // floor(p * 65536 + 1/2)
  float scale;                    // 65536 / (65536 - thr), 0 for thr = 65536
};

__device__ __forceinline__ void drop_resolve(DropRng& r) {
  if (r.dev) { r.seed = r.dev[0]; r.stream = r.dev[1]; }
}

__device__ __forceinline__ void drop_block(const DropRng& r, unsigned long long block, uint32_t w[4]) {
  w[0] = (uint32_t)block;
  w[1] = (uint32_t)(block >> 32);
  w[2] = (uint32_t)r.stream;
  w[3] = (uint32_t)(r.stream >> 32);
  philox4x32_10(w, (uint32_t)r.seed, (uint32_t)(r.seed >> 32) ^ DROP_KEY_TAG);
}

// f[e] = kept ? f[e] * scale : 0 for the VE elements from `idx` on (idx % VE == 0, VE = 1, 2, 4 or 8: all in one block)
template <int VE>
__device__ __forceinline__ void drop_apply(const DropRng& r, unsigned long long idx, float* f) {
  uint32_t w[4];
  drop_block(r, idx >> 3, w);
  if constexpr (VE == 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t d = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu;
      f[e] = d >= r.thr ? f[e] * r.scale : 0.f;
    }
  } else if constexpr (VE == 4) {
    const bool hi = (idx & 4) != 0;
    const uint32_t a = hi ? w[2] : w[0], b = hi ? w[3] : w[1];
    const uint32_t d[4] = {a & 0xFFFFu, a >> 16, b & 0xFFFFu, b >> 16};
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = d[e] >= r.thr ? f[e] * r.scale : 0.f;
  } else {
    const uint32_t a = (idx & 2) ? w[1] : w[0], b = (idx & 2) ? w[3] : w[2];
    const uint32_t v = (idx & 4) ? b : a;
    if constexpr (VE == 2) {
      f[0] = (v & 0xFFFFu) >= r.thr ? f[0] * r.scale : 0.f;
      f[1] = (v >> 16) >= r.thr ? f[1] * r.scale : 0.f;
    } else {
      const uint32_t d = (idx & 1) ? v >> 16 : v & 0xFFFFu;
      f[0] = d >= r.thr ? f[0] * r.scale : 0.f;
    }
  }
}
