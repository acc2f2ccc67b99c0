// Random bits from a counter: Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011).  The counter is an element's index / 8, the key the seed; element i takes 16 bits, half (i % 2) of word
// (i % 8) / 2.  It is dropped where these are below T = round(65536 p), else multiplied by 65536 / (65536 - T), so that the expectation is
// exact for the probability T / 65536.  The backward pass forms the same bits again: no mask is stored.
//
// A round is two 32 x 32 -> 64-bit products (v_mad_u64_u32, quarter rate): 10 rounds for 8 elements are about 70 cycles of
// a SIMD per 64 elements, half of what the memory traffic of a float32 dropout leaves; 32 bits an element would be twice that.
#pragma once
#include "common.h"

namespace s2cnn {

struct Dropout {
  unsigned long long seed;
  const long long* seed_at;        // device memory that holds the seed, or NULL
  unsigned threshold;
  float factor;
  bool on;                         // false: nothing is dropped, and no bits are formed
};

inline Dropout make_dropout(double p, unsigned long long seed, const long long* seed_at) {
  Dropout d;
  d.seed = seed;
  d.seed_at = seed_at;
  const double t = p * 65536.0;
  const unsigned n = (unsigned)__builtin_rint(t);          // ties to even, as round() of the definition
  d.threshold = n > 65535u ? 65535u : n;
  d.factor = (float)(65536.0 / (65536.0 - d.threshold));
  d.on = d.threshold != 0;
  return d;
}

__device__ __forceinline__ unsigned long long dropout_seed(const Dropout& d) { return d.seed_at ? (unsigned long long)*d.seed_at : d.seed; }

__device__ __forceinline__ uint4 philox(unsigned long long counter, unsigned long long key, unsigned long long upper = 0) {      // upper half of the counter
  unsigned c0 = (unsigned)counter, c1 = (unsigned)(counter >> 32), c2 = (unsigned)upper, c3 = (unsigned)(upper >> 32), k0 = (unsigned)key, k1 = (unsigned)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// dropout of the N elements from index on, N = 4 or 8; what is dropped is zero whatever it was
template <int N> __device__ __forceinline__ void drop(const Dropout& d, unsigned long long key, long index, float (&v)[N]) {
  const int shift = (int)(index & 7);
  const uint4 r = philox((unsigned long long)index >> 3, key);
  unsigned w[8] = {r.x, r.y, r.z, r.w, 0, 0, 0, 0};
  if (shift + N > 8) {
    const uint4 s = philox(((unsigned long long)index >> 3) + 1, key);
    w[4] = s.x, w[5] = s.y, w[6] = s.z, w[7] = s.w;
  }
  if (shift & 4) w[0] = w[2], w[1] = w[3], w[2] = w[4], w[3] = w[5], w[4] = w[6], w[5] = w[7];
  if (shift & 2) w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = w[4], w[4] = w[5];
  if (shift & 1) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], 16);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ((w[i / 2] >> (16 * (i % 2))) & 0xffffu) >= d.threshold ? v[i] * d.factor : 0.f;
}

}  // namespace s2cnn
