// 16 bytes of a type in registers, loaded and stored at any entry, and sums over a few lanes: what kernels that are bound by memory share.
#pragma once
#include "common.h"

namespace s2cnn {

typedef _Float16 half_t;
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// 16 bytes of a type
template <class T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <class T, class T2> struct Chunk16 {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&v)[8]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f2 x = __builtin_convertvector(__builtin_bit_cast(T2, w[i]), f2);
      v[2 * i] = x[0], v[2 * i + 1] = x[1];
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&v)[8]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f2{v[2 * i], v[2 * i + 1]}, T2));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Chunk<__bf16> : Chunk16<__bf16, bf2> {};
template <> struct Chunk<half_t> : Chunk16<half_t, h2> {};

typedef unsigned loose4 __attribute__((ext_vector_type(4), aligned(2)));    // 16 bytes at any entry
// The n first entries of a chunk at p (any alignment of the type's: rows of odd length), the others zero.
template <class T> __device__ __forceinline__ uint4 load_chunk(const T* p, int n, bool stream = false) {
  constexpr int N = Chunk<T>::N;
  uint4 u = make_uint4(0, 0, 0, 0);
  if (n >= N) {
    if (stream) {
      const loose4 x = __builtin_nontemporal_load(reinterpret_cast<const loose4*>(p));
      return make_uint4(x[0], x[1], x[2], x[3]);
    }
    __builtin_memcpy(&u, p, 16);
    return u;
  }
  unsigned w[4] = {0, 0, 0, 0};
  for (int i = 0; i < n; ++i) {
    if constexpr (N == 4) {
      unsigned e;
      __builtin_memcpy(&e, p + i, 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = i == j ? e : w[j];
    } else {
      unsigned short e;
      __builtin_memcpy(&e, p + i, 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] |= i / 2 == j ? (unsigned)e << (16 * (i & 1)) : 0u;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T> __device__ __forceinline__ void store_chunk(T* p, int n, const float (&v)[Chunk<T>::N], bool stream = false) {
  if (n >= Chunk<T>::N) {
    const uint4 u = Chunk<T>::put(v);
    if (stream) __builtin_nontemporal_store(loose4{u.x, u.y, u.z, u.w}, reinterpret_cast<loose4*>(p));
    else __builtin_memcpy(p, &u, 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < Chunk<T>::N; ++i)
    if (i < n) p[i] = (T)v[i];
}

// Sum over a group of L lanes, in all of them
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int L> __device__ __forceinline__ float sum_lanes(float v) {
  v = add_dpp<0xB1>(v);                       // the neighbour
  v = add_dpp<0x4E>(v);                       // two further
  if (L >= 8) v = add_dpp<0x141>(v);          // 8 lanes mirrored: the other four
  if (L >= 16) v = add_dpp<0x140>(v);         // 16 lanes mirrored: the other eight
  if (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

}  // namespace s2cnn
