// philox.cuh -- the counter-based random bits behind dropout.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011): a bijection of a 128-bit counter under a 64-bit
// key, ten rounds of two 32 x 32 -> 64 bit products.  The bits of an element
// are a pure function of (seed, offset, site, element index), so a mask is
// never stored: the backward pass draws the forward's bits again.
//
//   key     = seed (low word, high word)
//   counter = (element index / 8, site, offset low word, offset high word)
//   element 8 g + e has the 16 bits  (word[e / 2] >> 16 (e % 2)) & 0xffff  of
//   group g, and is kept where they are below the threshold
//   t = floor((1 - p) * 65536 + 1/2).
// Sixteen bits an element make one generator call serve a 16-byte vector of
// bf16.  The probability is rounded to a multiple of 2^-16, and a kept element
// is multiplied by 65536 / t, not 1 / (1 - p): the expectation is exact for
// the probability that is drawn.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace tfb {

struct DropoutParams {
  const unsigned long long* rng;  // device: seed, offset (null: nothing is dropped)
  unsigned site;
  unsigned limit;  // t << 16, t = 0 .. 65535 (t = 65536 drops nothing: no rng)
  float scale;     // 65536 / t (0 when t == 0: everything is dropped)
};

struct PhiloxState {
  uint32_t k0, k1, c1, c2, c3;
};

__device__ __forceinline__ PhiloxState philox_state(const DropoutParams& d) {
  const unsigned long long seed = __ldg(d.rng), offset = __ldg(d.rng + 1);
  // The same value in every lane; the warp reduction tells the compiler so, and
  // the ten rounds' keys then cost no instruction of a lane's.
  auto uniform = [](uint32_t v) { return __reduce_or_sync(0xffffffffu, v); };
  PhiloxState s;
  s.k0 = uniform((uint32_t)seed);
  s.k1 = uniform((uint32_t)(seed >> 32));
  s.c1 = d.site;
  s.c2 = uniform((uint32_t)offset);
  s.c3 = uniform((uint32_t)(offset >> 32));
  return s;
}

__device__ __forceinline__ uint4 philox4x32_10(const PhiloxState& s, uint32_t group) {
  uint32_t c0 = group, c1 = s.c1, c2 = s.c2, c3 = s.c3, k0 = s.k0, k1 = s.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Which of the eight elements of group g stay: the others become 0 whatever
// they held (a select, so an infinity or NaN that is dropped leaves no NaN
// behind).  The caller multiplies by d.scale.  A half is compared with t in
// the upper 16 bits of a word: below a high half nothing can tip the compare.
__device__ __forceinline__ void dropout_select8(const DropoutParams& d, const PhiloxState& s,
                                                uint32_t group, float (&v)[8]) {
  const uint4 r = philox4x32_10(s, group);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = (w[i] << 16) < d.limit ? v[2 * i] : 0.0f;
    v[2 * i + 1] = w[i] < d.limit ? v[2 * i + 1] : 0.0f;
  }
}

// ... and with the scale.
__device__ __forceinline__ void dropout8(const DropoutParams& d, const PhiloxState& s,
                                         uint32_t group, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= d.scale;
  dropout_select8(d, s, group, v);
}

}  // namespace tfb
