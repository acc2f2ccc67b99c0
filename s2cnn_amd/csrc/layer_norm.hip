// Layer normalisation over the last axis, dropout, and the step between two sublayers that joins residual, dropout and
// normalisation; forward and backward.  All are bound by memory: every tensor is read once and written once, in 16 bytes a
// lane, and what is formed on the way stays in registers.
//
// A row belongs to a group of L lanes, each with up to K chunks of 16 bytes of it: L = 8 up to 16 chunks, so that short rows
// leave few lanes idle and are summed in three lane exchanges, then 16, 32, 64, and a workgroup of 256; rows of more than
// 1024 chunks are read again per pass.  Mean and variance are formed one after the other from the registers (the variance from the centred
// values, not as a difference of large sums).
//
//   forward    y = (h - mean) rstd w + b, h = x, or residual + dropout(x)
//   backward   u = g w, dh = rstd (u - mean(u) - xh mean(u xh)) (+ the gradient of h), dx = dropout(dh); dw = sum g xh, db = sum g
//
// The two sums over the rows are kept in registers by the groups, which run over many rows each, joined per workgroup in LDS,
// and a second kernel adds the workgroups' sums in a fixed order.  The backward pass reads h, which is rounded to the tensors' type; in the
// step with a residual what the rounding left goes along in 8 bits an entry (16-bit types).  Without it the weights' gradient had that rounding
// beside its own, 1.41 times the error; x and the residual once more instead of h would be twice the traffic.  The error of a normalised entry in
// the backward pass is then 2^-16 (float16: 2^-19) of |h| over the row's deviation: below the rounding of the results up to offsets of 100 deviations.
//
// Measured, with a copy of 1 GiB at 5.1 TB/s: 65536 rows of 1024 in bfloat16: forward 58 us, 4.6 TB/s, backward 82 us, 4.9 TB/s; the step
// with a residual and dropout, 16384 rows of 512: 20 us, 3.8 TB/s, and 25 us, 3.7 TB/s (tensors of 17 MB: a third of the time is launch and
// first loads); 12800 rows of 100 in float32: 5 and 9 us; the sums of the workgroups 3 to 6 us on top.  Dropout of 67 million float32:
// 88 us, 6.1 TB/s, its accesses past the caches.
#include "counter_random.h"

namespace s2cnn {
namespace norm {

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

// What the rounding of v to a 16-bit type leaves, in units of 2^-7 of half a spacing (of numbers of that exponent): 8 bits with a sign.
template <class T> __device__ __forceinline__ float low_unit(float rounded) {      // 2^exponent, times 2^-15 or 2^-18
  return __uint_as_float(__float_as_uint(rounded) & 0x7f800000u) * (__is_same(T, __bf16) ? 0x1p-15f : 0x1p-18f);
}
template <class T> __device__ __forceinline__ uint2 low_parts(const float (&v)[Chunk<T>::N]) {
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < Chunk<T>::N; ++i) {
    const float r = (float)(T)v[i], inverse = __uint_as_float(0x7f000000u - (__float_as_uint(r) & 0x7f800000u)) * (__is_same(T, __bf16) ? 0x1p15f : 0x1p18f);
    const float q = __builtin_amdgcn_fmed3f(rintf((v[i] - r) * inverse), -127.f, 127.f);
    w[i / 4] |= ((unsigned)(int)q & 255u) << (8 * (i % 4));
  }
  return make_uint2(w[0], w[1]);
}
template <class T> __device__ __forceinline__ void add_low(const uint2& low, float (&v)[Chunk<T>::N]) {
  const unsigned w[2] = {low.x, low.y};
#pragma unroll
  for (int i = 0; i < Chunk<T>::N; ++i) v[i] = fmaf((float)((int)(w[i / 4] << (24 - 8 * (i % 4))) >> 24), low_unit<T>(v[i]), v[i]);
}
__device__ __forceinline__ uint2 load_low(const signed char* p, int n) {
  uint2 u = make_uint2(0, 0);
  if (n >= 8) __builtin_memcpy(&u, p, 8);
  else
    for (int i = 0; i < n; ++i) (i < 4 ? u.x : u.y) |= (unsigned)(unsigned char)p[i] << (8 * (i % 4));
  return u;
}
__device__ __forceinline__ void store_low(signed char* p, int n, const uint2& u) {
  if (n >= 8) __builtin_memcpy(p, &u, 8);
  else
    for (int i = 0; i < n; ++i) p[i] = (signed char)((i < 4 ? u.x : u.y) >> (8 * (i % 4)));
}

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

// ---- sums over a group of L lanes, in all of them -------------------------------------------------------------------
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
// `slot`: LDS of four floats that no other sum before the next barrier uses
template <int L> __device__ __forceinline__ float sum_group(float v, float* slot) {
  if constexpr (L <= 64) return sum_lanes<L>(v);
  v = sum_lanes<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
  __syncthreads();
  return (slot[0] + slot[1]) + (slot[2] + slot[3]);
}

struct Forward {
  const void *x, *residual, *weight, *bias;
  void *h, *y;
  float* stats;                  // [rows, 2] mean, rstd, then the low parts of h; may be NULL
  long rows;
  int features;
  float eps;
  Dropout drop;
};
struct Backward {
  const void *h, *g, *g_h, *weight;
  const float* stats;
  void *gx, *gresidual;
  float* partial;                // [workgroups, 2, features], or NULL
  long rows;
  int features;
  Dropout drop;
};

constexpr int THREADS = 256;

// LONG: more than K L chunks a row; h is formed again in every pass
template <class T, int L, int K, bool STEP, bool LONG> __global__ __launch_bounds__(THREADS) void forward_kernel(Forward p) {
  typedef Chunk<T> C;
  __shared__ float slots[2][4];
  const int lane = threadIdx.x % L, chunks = (p.features + C::N - 1) / C::N;
  const int passes = LONG ? (chunks + K * L - 1) / (K * L) : 1;
  const unsigned long long key = STEP && p.drop.on ? dropout_seed(p.drop) : 0;
  const T* const w = static_cast<const T*>(p.weight);
  const T* const b = static_cast<const T*>(p.bias);
  const float inv_n = 1.f / (float)p.features;

  const auto load_h = [&](long row, int c, float (&v)[C::N]) {       // chunk c of a row: x, or residual + dropout(x)
    const int n = p.features - c * C::N;
    const long at = row * p.features + (long)c * C::N;
    C::get(load_chunk<T>(static_cast<const T*>(p.x) + at, n), v);
    if constexpr (STEP) {
      float r[C::N];
      C::get(load_chunk<T>(static_cast<const T*>(p.residual) + at, n), r);
      if (p.drop.on) drop<C::N>(p.drop, key, at, v);
#pragma unroll
      for (int i = 0; i < C::N; ++i) v[i] += r[i];
    }
  };

  uint4 wraw[K], braw[K];                                           // loads in the loop would wait for those of the rows
  const auto fetch_weights = [&](int pass) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (pass * K + k) * L + lane, n = p.features - c * C::N;
      wraw[k] = braw[k] = make_uint4(0, 0, 0, 0);
      if (w && c < chunks) wraw[k] = load_chunk<T>(w + c * C::N, n);
      if (b && c < chunks) braw[k] = load_chunk<T>(b + c * C::N, n);
    }
  };
  if (!LONG) fetch_weights(0);

  for (long row0 = (long)blockIdx.x * (THREADS / L); row0 < p.rows; row0 += (long)gridDim.x * (THREADS / L)) {
    const long row = row0 + threadIdx.x / L;
    const bool ok = row < p.rows;
    const long r = ok ? row : p.rows - 1;
    float v[K][C::N], sum = 0.f;
    for (int pass = 0; pass < passes; ++pass) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (pass * K + k) * L + lane;
        if (c < chunks) load_h(r, c, v[k]);
        else
#pragma unroll
          for (int i = 0; i < C::N; ++i) v[k][i] = 0.f;
#pragma unroll
        for (int i = 0; i < C::N; ++i) sum += v[k][i];                // entries past the row's end are zero
      }
    }
    const float mean = sum_group<L>(sum, slots[0]) * inv_n;
    float square = 0.f;
    for (int pass = 0; pass < passes; ++pass) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (pass * K + k) * L + lane, n = p.features - c * C::N;
        if (LONG && c < chunks) load_h(r, c, v[k]);
#pragma unroll
        for (int i = 0; i < C::N; ++i)
          if (i < n) square = fmaf(v[k][i] - mean, v[k][i] - mean, square);
      }
    }
    const float rstd = 1.f / sqrtf(fmaf(sum_group<L>(square, slots[1]), inv_n, p.eps));
    for (int pass = 0; pass < passes; ++pass) {
      if (LONG) fetch_weights(pass);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (pass * K + k) * L + lane, n = p.features - c * C::N;
        if (c >= chunks || !ok) continue;
        if (LONG) load_h(r, c, v[k]);
        const long at = r * p.features + (long)c * C::N;
        if constexpr (STEP) {
          store_chunk<T>(static_cast<T*>(p.h) + at, n, v[k]);
          if constexpr (C::N == 8)
            if (p.stats) store_low(reinterpret_cast<signed char*>(p.stats + 2 * p.rows) + at, n, low_parts<T>(v[k]));
        }
        float ws[C::N], bs[C::N], y[C::N];
        C::get(wraw[k], ws);
        C::get(braw[k], bs);
#pragma unroll
        for (int i = 0; i < C::N; ++i) {
          y[i] = (v[k][i] - mean) * rstd;
          y[i] = w ? (b ? fmaf(y[i], ws[i], bs[i]) : y[i] * ws[i]) : (b ? y[i] + bs[i] : y[i]);
        }
        store_chunk<T>(static_cast<T*>(p.y) + at, n, y);
      }
    }
    if (p.stats && lane == 0 && ok) reinterpret_cast<float2*>(p.stats)[r] = make_float2(mean, rstd);
  }
}

template <class T, int L, int K, bool STEP, bool LONG> __global__ __launch_bounds__(THREADS) void backward_kernel(Backward p) {
  typedef Chunk<T> C;
  __shared__ float slots[2][4];
  extern __shared__ float joined[];                                 // the sums of THREADS / L groups, where L < THREADS
  const int lane = threadIdx.x % L, chunks = (p.features + C::N - 1) / C::N;
  const int passes = LONG ? (chunks + K * L - 1) / (K * L) : 1;
  const unsigned long long key = STEP && p.drop.on ? dropout_seed(p.drop) : 0;
  const T* const w = static_cast<const T*>(p.weight);
  const T* const hs = static_cast<const T*>(p.h);
  const T* const gs = static_cast<const T*>(p.g);
  const float inv_n = 1.f / (float)p.features;
  float gw[K][C::N] = {}, gb[K][C::N] = {};
  constexpr bool LOW = STEP && C::N == 8;
  const signed char* const lows = reinterpret_cast<const signed char*>(p.stats + 2 * p.rows);
  uint2 lnext[K], lraw[K];
  uint4 hnext[K], gnext[K], wraw[K];                                // the group's next row; the weights, whose loads in the loop would wait for it
  float2 stnext = make_float2(0.f, 0.f);
  const auto fetch_weights = [&](int pass) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (pass * K + k) * L + lane;
      wraw[k] = w && c < chunks ? load_chunk<T>(w + c * C::N, p.features - c * C::N) : make_uint4(0, 0, 0, 0);
    }
  };
  const auto fetch = [&](long row, int pass, uint4 (&h)[K], uint4 (&g)[K], uint2 (&low)[K]) {
    const long r = row < p.rows ? row : p.rows - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (pass * K + k) * L + lane, n = p.features - c * C::N;
      h[k] = g[k] = make_uint4(0, 0, 0, 0);
      low[k] = make_uint2(0, 0);
      if (c >= chunks) continue;
      if constexpr (LOW) low[k] = load_low(lows + r * p.features + (long)c * C::N, n);
      h[k] = load_chunk<T>(hs + r * p.features + (long)c * C::N, n);
      g[k] = load_chunk<T>(gs + r * p.features + (long)c * C::N, n);
    }
  };
  if (!LONG) {
    fetch_weights(0);
    fetch((long)blockIdx.x * (THREADS / L) + threadIdx.x / L, 0, hnext, gnext, lnext);
    stnext = reinterpret_cast<const float2*>(p.stats)[min((long)blockIdx.x * (THREADS / L) + threadIdx.x / L, p.rows - 1)];
  }

  for (long row0 = (long)blockIdx.x * (THREADS / L); row0 < p.rows; row0 += (long)gridDim.x * (THREADS / L)) {
    const long row = row0 + threadIdx.x / L;
    const bool ok = row < p.rows;
    const long r = ok ? row : p.rows - 1;
    const float2 st = LONG ? reinterpret_cast<const float2*>(p.stats)[r] : stnext;
    uint4 hraw[K], graw[K];
    float a = 0.f, c2 = 0.f;
    const auto form = [&](int k, float (&xh)[C::N], float (&g)[C::N], float (&u)[C::N]) {
      C::get(hraw[k], xh);
      if constexpr (LOW) add_low<T>(lraw[k], xh);
      C::get(graw[k], g);
      float ws[C::N];
      C::get(wraw[k], ws);
#pragma unroll
      for (int i = 0; i < C::N; ++i) {
        xh[i] = (xh[i] - st.x) * st.y;
        u[i] = w ? g[i] * ws[i] : g[i];
      }
    };
    for (int pass = 0; pass < passes; ++pass) {
      if (LONG) fetch(r, pass, hraw, graw, lraw);
      else {
#pragma unroll
        for (int k = 0; k < K; ++k) hraw[k] = hnext[k], graw[k] = gnext[k], lraw[k] = lnext[k];
        const long next = row + (long)gridDim.x * (THREADS / L);
        fetch(next, 0, hnext, gnext, lnext);
        stnext = reinterpret_cast<const float2*>(p.stats)[next < p.rows ? next : p.rows - 1];
      }
      if (LONG) fetch_weights(pass);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (pass * K + k) * L + lane;
        if (c >= chunks) continue;
        float xh[C::N], g[C::N], u[C::N];
        form(k, xh, g, u);                        // entries past the row's end: g = u = 0
#pragma unroll
        for (int i = 0; i < C::N; ++i) {
          a += u[i];
          c2 = fmaf(u[i], xh[i], c2);
          if (!LONG && ok) gw[k][i] = fmaf(g[i], xh[i], gw[k][i]), gb[k][i] += g[i];
        }
      }
    }
    a = sum_group<L>(a, slots[0]) * inv_n;
    c2 = sum_group<L>(c2, slots[1]) * inv_n;
    for (int pass = 0; pass < passes; ++pass) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (pass * K + k) * L + lane, n = p.features - c * C::N;
        if (c >= chunks || !ok) continue;
        const long at = r * p.features + (long)c * C::N;
        if (LONG) hraw[k] = load_chunk<T>(hs + at, n), graw[k] = load_chunk<T>(gs + at, n), wraw[k] = w ? load_chunk<T>(w + c * C::N, n) : make_uint4(0, 0, 0, 0);
        if constexpr (LONG && LOW) lraw[k] = load_low(lows + at, n);
        float xh[C::N], g[C::N], u[C::N];
        form(k, xh, g, u);
#pragma unroll
        for (int i = 0; i < C::N; ++i) u[i] = st.y * (u[i] - a - xh[i] * c2);
        if constexpr (STEP) {
          if (p.g_h) {
            float e[C::N];
            C::get(load_chunk<T>(static_cast<const T*>(p.g_h) + at, n), e);
#pragma unroll
            for (int i = 0; i < C::N; ++i) u[i] += e[i];
          }
          if (p.gresidual) store_chunk<T>(static_cast<T*>(p.gresidual) + at, n, u);
          if (p.gx) {
            if (p.drop.on) drop<C::N>(p.drop, key, at, u);
            store_chunk<T>(static_cast<T*>(p.gx) + at, n, u);
          }
        } else {
          store_chunk<T>(static_cast<T*>(p.gx) + at, n, u);
        }
      }
    }
  }
  if (LONG || !p.partial) return;
  float* const out = p.partial + (long)blockIdx.x * 2 * p.features;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = k * L + lane, n = p.features - c * C::N;
      const float (&v)[C::N] = which ? gb[k] : gw[k];
      if constexpr (L < THREADS) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < C::N; ++i) joined[(i * (THREADS / L) + threadIdx.x / L) * L + lane] = v[i];
        __syncthreads();
        if (threadIdx.x < L)
#pragma unroll
          for (int i = 0; i < C::N; ++i) {
            float t = 0.f;
            for (int s = 0; s < THREADS / L; ++s) t += joined[(i * (THREADS / L) + s) * L + lane];
            if (i < n) out[which * p.features + c * C::N + i] = t;
          }
      } else {
#pragma unroll
        for (int i = 0; i < C::N; ++i)
          if (i < n) out[which * p.features + c * C::N + i] = v[i];
      }
    }
  }
}

// dw, db of rows longer than the registers hold: a workgroup takes 64 features and a part of the rows
template <class T> __global__ __launch_bounds__(THREADS) void long_weights_kernel(Backward p, int parts, bool low) {
  __shared__ float sums[2][4][64];
  const int f = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  float gw = 0.f, gb = 0.f;
  if (f < p.features)
    for (long r = (long)blockIdx.y * 4 + wave; r < p.rows; r += 4L * parts) {
      const float2 st = reinterpret_cast<const float2*>(p.stats)[r];
      const float g = (float)static_cast<const T*>(p.g)[r * p.features + f];
      float h = (float)static_cast<const T*>(p.h)[r * p.features + f];
      if constexpr (Chunk<T>::N == 8)
        if (low) h = fmaf((float)reinterpret_cast<const signed char*>(p.stats + 2 * p.rows)[r * p.features + f], low_unit<T>(h), h);
      gw = fmaf(g, (h - st.x) * st.y, gw);
      gb += g;
    }
  sums[0][wave][threadIdx.x & 63] = gw;
  sums[1][wave][threadIdx.x & 63] = gb;
  __syncthreads();
  if (wave < 2 && f < p.features) {
    const float (&s)[4][64] = sums[wave];
    const int i = threadIdx.x & 63;
    p.partial[((long)blockIdx.y * 2 + wave) * p.features + f] = (s[0][i] + s[1][i]) + (s[2][i] + s[3][i]);
  }
}

// Sums over the rows of a tensor (the gradient of a bias), in parts like these: torch's own sum clears a counter in memory first, and a
// captured graph that holds such a node gives other sums when it is replayed.
template <class T> __global__ __launch_bounds__(THREADS) void column_parts_kernel(const T* x, float* partial, long rows, int features, int parts) {
  __shared__ float sums[4][64];
  const int i = threadIdx.x & 63, f = blockIdx.x * 64 + i, wave = threadIdx.x >> 6;
  const long step = 4L * parts;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (f < features)
    for (long r = (long)blockIdx.y * 4 + wave; r < rows; r += 4 * step)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r + j * step < rows) t[j] += (float)x[(r + j * step) * features + f];
  sums[wave][i] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  if (wave == 0 && f < features) partial[(long)blockIdx.y * features + f] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// the sums of the workgroups, of `tensors` tensors: 32 features a workgroup, 32 groups of lanes over the parts
template <class T> __global__ __launch_bounds__(1024) void sum_kernel(const float* partial, int parts, int features, int tensors, T* gw, T* gb) {
  __shared__ float sums[32][33];
  const int i = threadIdx.x & 31, s = threadIdx.x >> 5;
  const long col = (long)blockIdx.x * 32 + i, width = (long)tensors * features;
  float t = 0.f;
  if (col < width)
    for (int k = s; k < parts; k += 32) t += partial[k * width + col];
  sums[s][i] = t;
  __syncthreads();
  t = sum_lanes<32>(sums[i][s]);                    // lanes over the groups: feature s
  const long out = (long)blockIdx.x * 32 + s;
  if (i == 0 && out < width) {
    if (out < features) {
      if (gw) gw[out] = (T)t;
    } else if (gb) {
      gb[out - features] = (T)t;
    }
  }
}

// Dropout of a tensor.  16-bit types: a lane's 16 bytes are the eight elements of a counter.  float32: they are four, and two
// neighbouring lanes have the halves of one; a lane takes two chunks, 64 lanes apart, the even one forms the counter of the first and the
// odd one that of the second, and they exchange halves, so that accesses stay contiguous and no counter is formed twice.
template <class T> __global__ __launch_bounds__(THREADS) void dropout_kernel(const T* x, T* y, long n, Dropout d, bool stream) {
  typedef Chunk<T> C;
  constexpr int PER = 8 / C::N;                                     // chunks a lane, 64 lanes apart
  const unsigned long long key = dropout_seed(d);
  const int lane = threadIdx.x & 63;
  for (long first = ((long)blockIdx.x * THREADS + (threadIdx.x & ~63)) * 8; first < n; first += (long)gridDim.x * THREADS * 8) {     // the wave's
    uint4 raw[PER];
    long left[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const long at = first + (k * 64 + lane) * C::N;
      left[k] = n - at;
      raw[k] = left[k] > 0 ? load_chunk<T>(x + at, (int)min(left[k], 8L), stream) : make_uint4(0, 0, 0, 0);
    }
    unsigned w[PER][C::N / 2];                                      // 16 bits an element
    if (d.on) {
      if constexpr (PER == 1) {
        const uint4 r = philox((unsigned long long)(first + lane * 8) >> 3, key);
        w[0][0] = r.x, w[0][1] = r.y, w[0][2] = r.z, w[0][3] = r.w;
      } else {
        const bool odd = lane & 1;
        const uint4 r = philox((unsigned long long)(first + ((odd ? 64 : 0) + (lane & ~1)) * 4) >> 3, key);
        const unsigned s0 = __builtin_amdgcn_update_dpp(0, odd ? r.x : r.z, 0xB1, 0xf, 0xf, true), s1 = __builtin_amdgcn_update_dpp(0, odd ? r.y : r.w, 0xB1, 0xf, 0xf, true);
        w[0][0] = odd ? s0 : r.x, w[0][1] = odd ? s1 : r.y;
        w[1][0] = odd ? r.z : s0, w[1][1] = odd ? r.w : s1;
      }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      float v[C::N];
      C::get(raw[k], v);
      if (d.on) {
#pragma unroll
        for (int i = 0; i < C::N; ++i) v[i] = ((w[k][i / 2] >> (16 * (i % 2))) & 0xffffu) >= d.threshold ? v[i] * d.factor : 0.f;
      }
      if (left[k] > 0) store_chunk<T>(y + first + (k * 64 + lane) * C::N, (int)min(left[k], 8L), v, stream);
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;

int group_of(int dtype, int features) {              // lanes of a row
  const int chunks = (features + (dtype == S2CNN_F32 ? 3 : 7)) / (dtype == S2CNN_F32 ? 4 : 8);
  return chunks <= 16 ? 8 : chunks <= 32 ? 16 : chunks <= 64 ? 32 : chunks <= 256 ? 64 : 256;
}
bool is_long(int dtype, int features) { return features > (dtype == S2CNN_F32 ? 4096 : 8192); }
// Workgroups that run over all rows.  Backward: their number is that of the partial sums, two a CU; forward: eight a CU.
int workgroups(int dtype, long rows, int features, bool backward) {
  const long per = THREADS / group_of(dtype, features), need = (rows + per - 1) / per, most = CUS * (backward ? 2 : 8);
  return (int)(need < most ? need : most);
}
int parts_of(int dtype, long rows, int features) {
  if (!is_long(dtype, features)) return workgroups(dtype, rows, features, true);
  return (int)((rows + 63) / 64 < 64 ? (rows + 63) / 64 : 64);
}

template <class T, int L, int K, bool STEP, bool LONG = false> void launch(const Forward& p, int wgs, hipStream_t s) {
  hipLaunchKernelGGL((forward_kernel<T, L, K, STEP, LONG>), dim3((unsigned)wgs), dim3(THREADS), 0, s, p);
}
template <class T, int L, int K, bool STEP, bool LONG = false> void launch(const Backward& p, int wgs, hipStream_t s) {
  const size_t lds = !LONG && L < THREADS ? THREADS * Chunk<T>::N * sizeof(float) : 0;
  hipLaunchKernelGGL((backward_kernel<T, L, K, STEP, LONG>), dim3((unsigned)wgs), dim3(THREADS), lds, s, p);
}
template <class T, bool STEP, class P> void dispatch(const P& p, int wgs, hipStream_t s) {
  const int chunks = (p.features + Chunk<T>::N - 1) / Chunk<T>::N;
  if (chunks <= 8) launch<T, 8, 1, STEP>(p, wgs, s);
  else if (chunks <= 16) launch<T, 8, 2, STEP>(p, wgs, s);
  else if (chunks <= 32) launch<T, 16, 2, STEP>(p, wgs, s);
  else if (chunks <= 64) launch<T, 32, 2, STEP>(p, wgs, s);
  else if (chunks <= 128) launch<T, 64, 2, STEP>(p, wgs, s);
  else if (chunks <= 256) launch<T, 64, 4, STEP>(p, wgs, s);
  else if (chunks <= 1024) launch<T, 256, 4, STEP>(p, wgs, s);
  else launch<T, 256, 4, STEP, true>(p, wgs, s);
}
template <class T> void forward(const Forward& p, bool step, int wgs, hipStream_t s) {
  if (step) dispatch<T, true>(p, wgs, s);
  else dispatch<T, false>(p, wgs, s);
}
template <class T> void backward(const Backward& p, bool step, int dtype, void* gw, void* gb, hipStream_t s) {
  const int wgs = workgroups(dtype, p.rows, p.features, true), parts = parts_of(dtype, p.rows, p.features);
  if (step) dispatch<T, true>(p, wgs, s);
  else dispatch<T, false>(p, wgs, s);
  if (!p.partial) return;
  if (is_long(dtype, p.features))
    hipLaunchKernelGGL(long_weights_kernel<T>, dim3((unsigned)((p.features + 63) / 64), (unsigned)parts), dim3(THREADS), 0, s, p, parts, step);
  hipLaunchKernelGGL(sum_kernel<T>, dim3((unsigned)((2L * p.features + 31) / 32)), dim3(1024), 0, s, p.partial, parts, p.features, 2, static_cast<T*>(gw),
                     static_cast<T*>(gb));
}
template <class T> void dropout(const void* x, void* y, long n, const Dropout& d, hipStream_t s) {
  const long need = (n + 8 * THREADS - 1) / (8 * THREADS), most = CUS * 16;
  hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)(need < most ? need : most)), dim3(THREADS), 0, s, static_cast<const T*>(x), static_cast<T*>(y), n, d,
                     (size_t)n * sizeof(T) >= STREAM_BYTES);
}

// At least 64 rows a part, and up to 1024 workgroups.
int column_parts(long rows, long features) {
  const long most = 1024 / ((features + 63) / 64), need = (rows + 63) / 64, parts = need < most ? need : most;
  return parts < 1 ? 1 : (int)parts;
}
template <class T> void column_sums(const void* x, float* out, float* partial, long rows, int features, hipStream_t s) {
  const int parts = column_parts(rows, features);
  hipLaunchKernelGGL(column_parts_kernel<T>, dim3((unsigned)((features + 63) / 64), (unsigned)parts), dim3(THREADS), 0, s, static_cast<const T*>(x), partial, rows, features, parts);
  hipLaunchKernelGGL(sum_kernel<float>, dim3((unsigned)((features + 31) / 32)), dim3(1024), 0, s, partial, parts, features, 1, out, nullptr);
}

bool sizes_ok(long rows, long features, int dtype) {
  return rows >= 1 && rows < (1L << 31) && features >= 1 && features < (1L << 24) && (dtype == S2CNN_F32 || dtype == S2CNN_BF16 || dtype == S2CNN_F16);
}
template <class... P> bool aligned(int dtype, P... p) {
  const uintptr_t mask = dtype == S2CNN_F32 ? 3 : 1;
  return !((reinterpret_cast<uintptr_t>(p) | ...) & mask);
}

}  // namespace norm
}  // namespace s2cnn

using namespace s2cnn;
using namespace s2cnn::norm;

extern "C" int s2cnn_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias, void* h, void* y, float* stats, long rows,
                              long features, float eps, double p, unsigned long long seed, const long long* seed_at, int dtype, void* stream) {
  clear_stale_error();
  if (!sizes_ok(rows, features, dtype) || !x || !y || !residual != !h || !(p >= 0.0 && p < 1.0) || (!residual && p != 0.0)) return S2CNN_EINVAL;
  if (!aligned(dtype, x, residual, weight, bias, h, y) || !aligned8(stats) || !aligned8(seed_at)) return S2CNN_EALIGN;
  const Forward f{x, residual, weight, bias, h, y, stats, rows, (int)features, eps, make_dropout(p, seed, seed_at)};
  const int wgs = workgroups(dtype, rows, (int)features, false);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == S2CNN_F32) norm::forward<float>(f, residual != nullptr, wgs, s);
  else if (dtype == S2CNN_BF16) norm::forward<__bf16>(f, residual != nullptr, wgs, s);
  else norm::forward<half_t>(f, residual != nullptr, wgs, s);
  return launch_status();
}

extern "C" size_t s2cnn_layer_norm_stats_floats(long rows, long features, int dtype, int step) {
  if (!sizes_ok(rows, features, dtype)) return 0;
  return 2 * (size_t)rows + (step && dtype != S2CNN_F32 ? ((size_t)rows * features + 3) / 4 : 0);
}

extern "C" size_t s2cnn_layer_norm_bwd_workspace(long rows, long features, int dtype) {
  if (!sizes_ok(rows, features, dtype)) return 0;
  return (size_t)parts_of(dtype, rows, (int)features) * 2 * features * sizeof(float);
}

extern "C" int s2cnn_layer_norm_bwd(const void* h, const void* g, const void* g_h, const void* weight, const float* stats, void* gx, void* gresidual, void* gweight,
                              void* gbias, void* workspace, size_t workspace_bytes, long rows, long features, double p, unsigned long long seed,
                              const long long* seed_at, int step, int dtype, void* stream) {
  clear_stale_error();
  if (!sizes_ok(rows, features, dtype) || !h || !g || !stats || !(p >= 0.0 && p < 1.0)) return S2CNN_EINVAL;
  if (step ? (!gx && !gresidual) : (!gx || gresidual || g_h || p != 0.0)) return S2CNN_EINVAL;
  if (!aligned(dtype, h, g, g_h, weight, gx, gresidual, gweight, gbias) || !aligned8(stats) || !aligned8(seed_at)) return S2CNN_EALIGN;
  const bool sums = gweight || gbias;
  if (sums && (!workspace || workspace_bytes < s2cnn_layer_norm_bwd_workspace(rows, features, dtype) || !aligned16(workspace))) return S2CNN_EWORKSPACE;
  const norm::Backward b{h, g, g_h, weight, stats, gx, gresidual, sums ? static_cast<float*>(workspace) : nullptr, rows, (int)features, make_dropout(p, seed, seed_at)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == S2CNN_F32) norm::backward<float>(b, step != 0, dtype, gweight, gbias, s);
  else if (dtype == S2CNN_BF16) norm::backward<__bf16>(b, step != 0, dtype, gweight, gbias, s);
  else norm::backward<half_t>(b, step != 0, dtype, gweight, gbias, s);
  return launch_status();
}

extern "C" size_t s2cnn_column_sums_workspace(long rows, long features, int dtype) {
  return sizes_ok(rows, features, dtype) ? (size_t)column_parts(rows, features) * features * sizeof(float) : 0;
}

extern "C" int s2cnn_column_sums(const void* x, float* out, void* workspace, size_t workspace_bytes, long rows, long features, int dtype, void* stream) {
  clear_stale_error();
  if (!sizes_ok(rows, features, dtype) || !x || !out) return S2CNN_EINVAL;
  if (!aligned(dtype, x) || !aligned(S2CNN_F32, out)) return S2CNN_EALIGN;
  if (!workspace || workspace_bytes < s2cnn_column_sums_workspace(rows, features, dtype) || !aligned16(workspace)) return S2CNN_EWORKSPACE;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float* const partial = static_cast<float*>(workspace);
  if (dtype == S2CNN_F32) norm::column_sums<float>(x, out, partial, rows, (int)features, s);
  else if (dtype == S2CNN_BF16) norm::column_sums<__bf16>(x, out, partial, rows, (int)features, s);
  else norm::column_sums<half_t>(x, out, partial, rows, (int)features, s);
  return launch_status();
}

extern "C" int s2cnn_dropout(const void* x, void* y, long n, double p, unsigned long long seed, const long long* seed_at, int dtype, void* stream) {
  clear_stale_error();
  if (!x || !y || n < 1 || n >= (1L << 40) || !(p >= 0.0 && p < 1.0) || (dtype != S2CNN_F32 && dtype != S2CNN_BF16 && dtype != S2CNN_F16)) return S2CNN_EINVAL;
  if (!aligned(dtype, x, y) || !aligned8(seed_at)) return S2CNN_EALIGN;
  const Dropout d = make_dropout(p, seed, seed_at);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == S2CNN_F32) norm::dropout<float>(x, y, n, d, s);
  else if (dtype == S2CNN_BF16) norm::dropout<__bf16>(x, y, n, d, s);
  else norm::dropout<half_t>(x, y, n, d, s);
  return launch_status();
}
