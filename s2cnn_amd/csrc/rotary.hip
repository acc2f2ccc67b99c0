// Rotation of queries and keys by position, alone or after a normalisation of every head's vectors, forward and backward, and the table of
// the rotations.
//
//   forward    y = R (w x r),  r = 1 / sqrt(mean(x^2) + eps)     (without the normalisation: y = R x)
//   backward   g = R^T gy, u = g w, gx = r (u - xh mean(u xh)) with xh = x r, gw = sum of g xh over all vectors
//
// R turns pair j of a vector's entries by the angle of row n of the table: (a, b) -> (a cos - b sin, a sin + b cos).  Pairs are neighbours (2j,
// 2j + 1), or halves apart (j, pairs + j); entries from 2 pairs on stay.  R^T is the same with -sin.
//
// All of it is bound by memory: x (and gy) read once, y (or gx) written once, the rest in registers; r is formed again in the backward pass from x, which
// it reads anyway.  A vector belongs to a group of L lanes (a power of two).  A lane holds two chunks of 16 bytes, so that both entries of a pair
// are its own: no exchange between lanes but the sums over a vector.  Where a chunk would run past the end of its part, it begins earlier and
// overlaps the one before (both lanes form the same numbers; sums count them once), so that all accesses are 16 bytes wide, at any alignment; only
// parts shorter than a chunk are loaded entry by entry, in kernels of their own (not FULL: rotations of 4 x 16 heads x 4096 places x 64 in float32
// take 27 us each way; with the tests for tails a quarter more).
//
// Measured, with a copy of 1 GiB at 5.1 TB/s: 4 x (32 + 8) heads x 8192 places x 128 in bfloat16: forward 122 us, 5.5 TB/s, backward 185 to 195 us, 5.2 to
// 5.4 TB/s, and 4 us for the sums of its weights' gradients; tensors of 256 MB or more go past the caches (in them: 127 and 205 to 215 us).  A
// batch of 32 x 10 heads x 400 places of 20 in float32: 9 and 12 us, a launch, two trips to memory and their instructions; single places 3 to 5 us.
//
// Arithmetic is float32: squares and the gradients of weights are summed in it, r is one instruction's root of a product with 1 / d.  In float32 y is off by a
// tenth more than by a root and a quotient of their own; 16-bit results hide it.
#include "chunk.h"

namespace s2cnn {
namespace rotary {

constexpr int THREADS = 256;
constexpr int MAX_D = 256;

// x / divisor for 0 <= x < 2^31 by a product: (mulhi(x, magic) + x) >> shift
struct Divider {
  unsigned magic, shift, divisor;
};
inline Divider divider(long n) {
  unsigned s = 0;
  while ((1L << s) < n) ++s;
  return {(unsigned)((((1UL << s) - (unsigned long)n) << 32) / (unsigned long)n + 1), s, (unsigned)n};
}
__device__ __forceinline__ unsigned divide(unsigned x, const Divider& d, unsigned& rest) {
  const unsigned q = (__umulhi(x, d.magic) + x) >> d.shift;
  rest = x - q * d.divisor;
  return q;
}

struct Tensor {                  // vectors of a tensor: entries from head to head, place to place, signal to signal
  const void* at;
  long head, place, batch;
};
struct Side {                    // queries, or keys
  Tensor x, g, y;
  const void* weight;
  float* partial;                // [workgroups, d]
  Divider inner, middle;         // of an item's number: runs of heads and places, or the other way round
  unsigned items;                // runs of `run` heads at a place
  int heads, run;
  int heads_inside;
};
struct Args {
  Side side[2];
  unsigned blocks0;              // workgroups of side 0
  const float2* table;
  const int* index;
  long table_stride, index_stride;      // of the batch
  int rows, d, pairs, units, lanes, log_lanes;
  float inv_d, eps, sign;
  bool stream;
};

// The part of a vector that a lane holds.
struct Part {
  int a, b, na, nb;              // first entries and numbers of entries of its two chunks
  int skip_a, skip_b;            // leading entries that belong to another lane as well
  int pair;                      // the pair of the first entry
  bool own;                      // not: another lane's part once more, so that all lanes do the same
};
template <int V, bool NEIGHBOURS> __device__ __forceinline__ Part part_of(int u, int units, int d, int pairs) {
  Part p = {0, 0, 0, 0, 0, 0, pairs, u < units};
  u = min(u, units - 1);
  int first, length;                                               // a run of entries that is cut into two chunks a lane
  if (!NEIGHBOURS && u < (pairs + V - 1) / V) {
    p.pair = pairs >= V ? min(u * V, pairs - V) : 0;
    p.a = p.pair, p.b = pairs + p.pair;
    p.na = p.nb = min(pairs, V);
    p.skip_a = p.skip_b = u * V - p.pair;
    return p;
  }
  if (NEIGHBOURS) {
    first = 0, length = d & ~1;
    if (u >= (length + 2 * V - 1) / (2 * V)) first = length, length = 1, u = 0;
  } else {
    first = 2 * pairs, length = d - first, u -= (pairs + V - 1) / V;
  }
  const int at = length >= 2 * V ? min(u * 2 * V, length - 2 * V) : 0, skip = u * 2 * V - at;
  p.a = first + at, p.b = p.a + V;
  p.na = min(length, V), p.nb = min(length - p.na, V);
  p.skip_a = min(skip, V), p.skip_b = skip - p.skip_a;
  if (NEIGHBOURS) p.pair = p.a / 2;
  return p;
}
// A copy that the compiler takes for new: what is compared with it in a loop is compared there, and not kept as dozens of lane masks across it,
// for which there are not enough scalar registers.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
inline int units_of(int V, int d, int pairs, bool neighbours) {
  if (neighbours) return ((d & ~1) + 2 * V - 1) / (2 * V) + (d & 1);
  return (pairs + V - 1) / V + (d - 2 * pairs + 2 * V - 1) / (2 * V);
}

// The first n entries at p, the others zero, in 16 bytes: one load, or entry by entry.
template <class T, bool FULL> __device__ __forceinline__ uint4 load(const T* p, int n, bool stream = false) {
  constexpr int N = Chunk<T>::N;
  if (FULL || n == N) return load_chunk<T>(p, N, FULL && stream);
  n = fresh(n);
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  return Chunk<T>::put(v);
}
template <class T, bool FULL> __device__ __forceinline__ void store(T* p, int n, const float (&v)[Chunk<T>::N], bool stream) {
  constexpr int N = Chunk<T>::N;
  if (FULL || n == N) return store_chunk<T>(p, N, v, FULL && stream);
  n = fresh(n);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = (T)v[i];
}

// cos and sin of the first `turned` of V pairs from `pair` on of a row; of a row that is not there NaN.  FULL: all or none of them.
template <int V, bool FULL> __device__ __forceinline__ void load_turns(const float2* row, bool there, int pair, int turned, float sign, float (&c)[V], float (&s)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
  if (there && turned == V) {
    typedef float loose __attribute__((ext_vector_type(4), aligned(8)));
    const loose* const at = reinterpret_cast<const loose*>(row + pair);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const loose t = at[i];
      c[2 * i] = t[0], s[2 * i] = t[1] * sign, c[2 * i + 1] = t[2], s[2 * i + 1] = t[3] * sign;
    }
  } else if (!FULL && there) {
    turned = fresh(turned);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < turned) c[i] = row[pair + i].x, s[i] = row[pair + i].y * sign;
  }
}

// The first `turned` pairs of a lane.  Others are left alone rather than turned by nothing: 0 times an infinity is none.
// Sums of products are written as fused operations, here and below, and the compiler makes no others: a vector's result is the same bits in every kernel.
template <int V, bool NEIGHBOURS, bool FULL> __device__ __forceinline__ void turn(int turned, const float (&c)[V], const float (&s)[V], float (&a)[V], float (&b)[V]) {
#pragma clang fp contract(off)
  if (!FULL) turned = fresh(turned);
  const bool whole = turned == V;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float& u = NEIGHBOURS ? (i < V / 2 ? a[(2 * i) % V] : b[(2 * i) % V]) : a[i];
    float& v = NEIGHBOURS ? (i < V / 2 ? a[(2 * i + 1) % V] : b[(2 * i + 1) % V]) : b[i];
    const float x = u, y = v;
    const bool mine = FULL ? whole : i < turned;
    u = mine ? fmaf(x, c[i], -(y * s[i])) : x;
    v = mine ? fmaf(x, s[i], y * c[i]) : y;
  }
}

__device__ __forceinline__ float sum_of(float v, int lanes) {           // over a group, `lanes` the same in all of the launch
  asm volatile("" : "+s"(lanes));                                       // compared here each time, as above
  if (lanes > 1) v = add_dpp<0xB1>(v);
  if (lanes > 2) v = add_dpp<0x4E>(v);
  if (lanes > 4) v = add_dpp<0x141>(v);
  if (lanes > 8) v = add_dpp<0x140>(v);
  if (lanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lanes > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sum over the entries of a lane that are its own of x y
template <int V> __device__ __forceinline__ float dot(const Part& p, const float (&xa)[V], const float (&xb)[V], const float (&ya)[V], const float (&yb)[V]) {
  float t = 0.f;
  if (p.skip_a == 0 && p.skip_b == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) t = fmaf(xa[i], ya[i], fmaf(xb[i], yb[i], t));
  } else {
    const int skip_a = fresh(p.skip_a), skip_b = fresh(p.skip_b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i >= skip_a) t = fmaf(xa[i], ya[i], t);
      if (i >= skip_b) t = fmaf(xb[i], yb[i], t);
    }
  }
  return p.own ? t : 0.f;
}

enum Pass { TURN, NORM, NORM_BACK };           // TURN: both directions of the rotation alone

// FULL: no lane's chunks are shorter than 16 bytes, and each is turned whole or not at all.  HEADS: the most heads of a run, whose loads are under way together and which share the cosines and sines of their place.
template <class T, Pass PASS, bool NEIGHBOURS, int HEADS, bool FULL> __global__ __launch_bounds__(THREADS, PASS == NORM_BACK ? 3 : 4) void rotary_kernel(Args p) {
#pragma clang fp contract(off)
  constexpr int V = Chunk<T>::N;
  const bool second = blockIdx.x >= p.blocks0;
  const Side& s = p.side[__builtin_amdgcn_readfirstlane((int)second)];        // a number, so that the fields are loaded together
  const unsigned block = second ? blockIdx.x - p.blocks0 : blockIdx.x, blocks = second ? gridDim.x - p.blocks0 : p.blocks0;
  const int lane = threadIdx.x & (p.lanes - 1);
  const unsigned groups = (unsigned)(THREADS >> p.log_lanes);
  const Part part = part_of<V, NEIGHBOURS>(lane, p.units, p.d, p.pairs);
  uint4 wraw_a, wraw_b;                                            // weights
  float ga[V] = {}, gb[V] = {};                                    // sums of their gradients
  if (PASS != TURN && s.weight) {
    wraw_a = load<T, FULL>(static_cast<const T*>(s.weight) + part.a, part.na);
    wraw_b = load<T, FULL>(static_cast<const T*>(s.weight) + part.b, part.nb);
  }
  const auto weigh = [&](float (&a)[V], float (&b)[V]) {
    if (!s.weight) return;
    float w[V];
    Chunk<T>::get(wraw_a, w);
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] *= w[i];
    Chunk<T>::get(wraw_b, w);
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] *= w[i];
  };
  // every group of the launch takes as many turns, so that no lane is missing from a sum
  for (unsigned first = block * groups; first < s.items; first += blocks * groups) {
    const unsigned mine = first + (threadIdx.x >> p.log_lanes), item = min(mine, s.items - 1);
    unsigned inner, middle;
    const unsigned outer = divide(divide(item, s.inner, inner), s.middle, middle);
    const unsigned place = s.heads_inside ? middle : inner;
    const int head = (int)(s.heads_inside ? inner : middle) * s.run, heads = mine < s.items ? min(s.run, s.heads - head) : 0;
    const auto at = [&](const Tensor& t) { return (T*)t.at + ((long)outer * t.batch + (long)place * t.place + (long)head * t.head); };
    uint4 raw[HEADS][2] = {}, graw[HEADS][2] = {};
    const T* const x = at(s.x);
    const T* const g = PASS == NORM_BACK ? at(s.g) : nullptr;
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
      if (h < heads) {
        raw[h][0] = load<T, FULL>(x + h * s.x.head + part.a, part.na, p.stream), raw[h][1] = load<T, FULL>(x + h * s.x.head + part.b, part.nb, p.stream);
        if (PASS == NORM_BACK) graw[h][0] = load<T, FULL>(g + h * s.g.head + part.a, part.na, p.stream), graw[h][1] = load<T, FULL>(g + h * s.g.head + part.b, part.nb, p.stream);
      }
    int row = (int)place;
    if (p.index) row = p.index[outer * p.index_stride + place];
    float c[V], sn[V];
    const int turned = row < 0 ? 0 : max(min(p.pairs - part.pair, V), 0);     // a row below zero: the vector is not turned
    load_turns<V, FULL>(p.table + outer * p.table_stride + (long)row * p.pairs, row < p.rows, part.pair, turned, p.sign, c, sn);
    T* const y = at(s.y);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      if (h >= s.run) break;
      float a[V], b[V];
      Chunk<T>::get(raw[h][0], a);
      Chunk<T>::get(raw[h][1], b);
      if constexpr (PASS == TURN) {
        turn<V, NEIGHBOURS, FULL>(turned, c, sn, a, b);
      } else {
        const float r = rsqrtf(fmaf(sum_of(dot<V>(part, a, b, a, b), p.lanes), p.inv_d, p.eps));
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] *= r, b[i] *= r;
        if constexpr (PASS == NORM) {
          weigh(a, b);
          turn<V, NEIGHBOURS, FULL>(turned, c, sn, a, b);
        } else {
          float u[V], v[V];
          Chunk<T>::get(graw[h][0], u);
          Chunk<T>::get(graw[h][1], v);
          turn<V, NEIGHBOURS, FULL>(turned, c, sn, u, v);
          if (h < heads)
#pragma unroll
            for (int i = 0; i < V; ++i) ga[i] = fmaf(u[i], a[i], ga[i]), gb[i] = fmaf(v[i], b[i], gb[i]);
          weigh(u, v);
          const float m = sum_of(dot<V>(part, u, v, a, b), p.lanes) * p.inv_d;
#pragma unroll
          for (int i = 0; i < V; ++i) a[i] = r * fmaf(-a[i], m, u[i]), b[i] = r * fmaf(-b[i], m, v[i]);
        }
      }
      if (h < heads && part.own) {
        store<T, FULL>(y + h * s.y.head + part.a, part.na, a, p.stream);
        store<T, FULL>(y + h * s.y.head + part.b, part.nb, b, p.stream);
      }
    }
  }
  if constexpr (PASS == NORM_BACK) {
    if (!s.partial) return;
    __shared__ float joined[THREADS / 64][64][2 * V + 1];
    for (int m = p.lanes; m < 64; m <<= 1)                         // groups of a wave
#pragma unroll
      for (int i = 0; i < V; ++i) ga[i] += __shfl_xor(ga[i], m), gb[i] += __shfl_xor(gb[i], m);
    if ((threadIdx.x & 63) < (unsigned)p.lanes)
#pragma unroll
      for (int i = 0; i < V; ++i) joined[threadIdx.x >> 6][lane][i] = ga[i], joined[threadIdx.x >> 6][lane][V + i] = gb[i];
    __syncthreads();
    if (threadIdx.x < (unsigned)p.lanes) {
      float* const out = s.partial + (long)block * p.d;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const auto sum = [&](int k) { return (joined[0][lane][k] + joined[1][lane][k]) + (joined[2][lane][k] + joined[3][lane][k]); };
        if (i >= part.skip_a && i < part.na) out[part.a + i] = sum(i);
        if (i >= part.skip_b && i < part.nb) out[part.b + i] = sum(V + i);
      }
    }
  }
}

// The workgroups' sums of the weights' gradients, in a fixed order: 32 entries a workgroup, 32 groups of lanes over the workgroups.
template <class T> __global__ __launch_bounds__(1024) void weights_kernel(const float* partial0, const float* partial1, unsigned blocks0, unsigned blocks1, int d, T* out0,
                                                                       T* out1) {
  __shared__ float sums[32][33];
  const float* const partial = blockIdx.y ? partial1 : partial0;
  T* const out = blockIdx.y ? out1 : out0;
  const unsigned blocks = blockIdx.y ? blocks1 : blocks0;
  if (!out) return;
  const int i = threadIdx.x & 31, s = threadIdx.x >> 5, col = blockIdx.x * 32 + i;
  float t = 0.f;
  if (col < d) {
#pragma unroll 8
    for (unsigned k = s; k < blocks; k += 32) t += partial[(long)k * d + col];
  }
  sums[s][i] = t;
  __syncthreads();
  t = sum_lanes<32>(sums[i][s]);
  if (i == 0 && (int)blockIdx.x * 32 + s < d) out[blockIdx.x * 32 + s] = (T)t;
}

// ---- the table ------------------------------------------------------------------------------------------------------
// An angle is formed in quarters of a turn and in 64 bits; adding 1.5 2^52 leaves the nearest whole number, whose lowest bits say which sine or cosine to
// take of what is left, -1/2 .. 1/2, in 32 bits: positions of a million lose nothing.  Sine and cosine of that are polynomials of its square that interpolate
// them at Chebyshev's points, in float32 with all roundings off by at most 0.95 2^-24 and 1.24 2^-24 (in the mean of squares 1.3 and 1.1 times what a rounding
// of the exact value leaves).  pi/2, the sine's first coefficient, has its low part with it: without, 1.72 2^-24 and twice.  A scale other than one
// is one more rounding.  A thread keeps its PER neighbouring pairs and takes one row after the other, so that a position is
// converted once for 16 bytes of the table.  262144 rows of 64 pairs, 134 MB: 26 to 28 us, 4.8 to 5.1 TB/s (one pair a thread and the library's sincospi: 43).
__device__ __forceinline__ float2 turn_of(double quarters, float scale) {
  double whole = (quarters + 0x1.8p52) - 0x1.8p52;
  unsigned q = (unsigned)__double_as_longlong(quarters + 0x1.8p52);
  if (!(fabs(quarters) < 0x1p50)) {                                       // beyond: what 64 bits have of it
    whole = rint(quarters);
    q = (unsigned)(int)(whole - 4.0 * floor(0.25 * whole));
  }
  const float x = (float)(quarters - whole), z = x * x;
  const float sin = fmaf(x, 0x1.921fb6p+0f, x * fmaf(z, fmaf(z, fmaf(z, -0x1.2d9b40p-8f, 0x1.465ec4p-4f), -0x1.4abbbap-1f), -0x1.777a5cp-25f));
  const float cos = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0x1.d9c2e8p-11f, -0x1.55c57ap-6f), 0x1.03c1dcp-2f), -0x1.3bd3ccp+0f), 1.f);
  const float c = q & 1 ? sin : cos, s = q & 1 ? cos : sin;
  return make_float2(__uint_as_float(__float_as_uint(c) ^ (((q + 1) & 2) << 30)) * scale, __uint_as_float(__float_as_uint(s) ^ ((q & 2) << 30)) * scale);
}

template <int PER, class P> __global__ __launch_bounds__(THREADS) void table_kernel(const P* positions, const double* frequencies, float2* table, long n, int axes, int pairs,
                                                                                float scale) {
  constexpr double QUARTERS = 0.63661977236758134308;                    // of a turn in a radian
  const int threads = pairs / PER, side = THREADS / threads, r = threadIdx.x / threads, j = (threadIdx.x - r * threads) * PER;
  if (r >= side) return;
  double f[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) f[i] = frequencies[j + i] * QUARTERS;
#pragma unroll 4
  for (long row = (long)blockIdx.x * side + r; row < n; row += (long)gridDim.x * side) {
    const double p = (double)positions[row * axes];
    double quarters[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) quarters[i] = p * f[i];
    for (int a = 1; a < axes; ++a) {
      const double q = (double)positions[row * axes + a] * QUARTERS;
#pragma unroll
      for (int i = 0; i < PER; ++i) quarters[i] = fma(q, frequencies[a * pairs + j + i], quarters[i]);
    }
    float2* const out = table + row * pairs + j;
    if constexpr (PER == 2) {
      typedef float loose __attribute__((ext_vector_type(4), aligned(8)));
      const float2 u = turn_of(quarters[0], scale), v = turn_of(quarters[1], scale);
      *reinterpret_cast<loose*>(out) = loose{u.x, u.y, v.x, v.y};
    } else {
      *out = turn_of(quarters[0], scale);
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;

struct Plan {
  int units, lanes, log_lanes, most;      // most: heads of a run that the kernel is made for
  bool full;
  int run[2];
  unsigned items[2], blocks[2];
};

bool sizes_ok(const s2cnn_rotary_t* a) {
  if (!a || (a->dtype != S2CNN_F32 && a->dtype != S2CNN_BF16 && a->dtype != S2CNN_F16)) return false;
  if (a->batch < 1 || a->n < 1 || a->d < 1 || a->d > MAX_D || a->pairs < 0 || 2 * a->pairs > a->d) return false;
  if (a->pairs && (!a->table || a->rows < 1 || (!a->index && a->rows < a->n))) return false;
  if (!a->pairs && (a->table || a->index)) return false;
  if (a->heads[0] < 1 || a->heads[1] < 0 || (a->norm && !(a->eps >= 0x1p-126f))) return false;
  const long limit = 1L << 31;
  for (int heads : a->heads)
    if ((long)a->batch * a->n >= limit || (heads && (long)a->batch * a->n >= limit / heads)) return false;
  return true;
}

// Runs of four heads (two where x and g are read) where that leaves every group two runs or more, else of one: 4 x 40 heads x 8192 places of 128 in bfloat16,
// in the caches, forward and backward, 128 and 205 us, of one head each 160 and 224; 32 x 10 heads x 400 places of 20 in float32 the other way round, 10.7 and
// 14.5 us, of one 9.4 and 12.5.  Four workgroups a CU (three; runs of one head: eight, four), or fewer that take as many turns.  In 16 bits that is what the
// registers let run at once, but for the normalisation of one head, which gets seven of its eight; in float32, with half the registers, up to eight
// would fit in all of them.
Plan plan_of(const s2cnn_rotary_t& a, bool two) {
  Plan p;
  p.units = units_of(a.dtype == S2CNN_F32 ? 4 : 8, a.d, a.pairs, a.interleaved != 0);
  for (p.lanes = 1, p.log_lanes = 0; p.lanes < p.units; ++p.log_lanes) p.lanes *= 2;
  const int V = a.dtype == S2CNN_F32 ? 4 : 8, rest = a.d - 2 * a.pairs;
  p.full = a.interleaved ? a.d % 2 == 0 && a.d >= 2 * V && (rest == 0 || a.pairs == 0 || (a.d % (2 * V) == 0 && a.pairs % V == 0))
                         : (a.pairs == 0 || a.pairs >= V) && (rest == 0 || rest >= 2 * V);
  const long groups = THREADS / p.lanes, places = (long)a.batch * a.n, vectors = places * ((long)a.heads[0] + a.heads[1]);
  p.most = two ? 2 : 4;
  long most = CUS * (two ? 3 : 4);
  if (!p.full || vectors < 2 * most * groups * p.most) p.most = 1, most = CUS * (two ? 4 : 8);
  long runs[2], total = 0;
  for (int i = 0; i < 2; ++i) {
    runs[i] = (a.heads[i] + p.most - 1) / p.most;
    p.run[i] = runs[i] ? (int)((a.heads[i] + runs[i] - 1) / runs[i]) : 1;
    runs[i] = (a.heads[i] + p.run[i] - 1) / p.run[i];
    p.items[i] = (unsigned)(places * runs[i]);
    total += p.items[i];
  }
  for (int i = 0; i < 2; ++i) {
    const long need = (p.items[i] + groups - 1) / groups;
    long share = (long)((double)most * p.items[i] / total);
    if (share < 1) share = 1;
    const long turns = (need + share - 1) / share;
    p.blocks[i] = (unsigned)(total <= most * groups ? need : need ? (need + turns - 1) / turns : 0);
  }
  return p;
}

Args args_of(const s2cnn_rotary_t& a, const Plan& p, bool backward, float* partial) {
  Args k = {};
  for (int i = 0; i < 2; ++i) {
    Side& s = k.side[i];
    s.items = p.items[i];
    if (!a.heads[i]) continue;
    const bool only_g = backward && !a.norm;
    const long* const read = only_g ? a.g_stride[i] : a.x_stride[i];
    s.heads = a.heads[i], s.run = p.run[i];
    const int runs = (s.heads + s.run - 1) / s.run;
    s.heads_inside = a.n == 1 || (s.heads > 1 && read[1] <= read[2]);      // neighbouring groups take vectors that lie next to each other
    s.inner = divider(s.heads_inside ? runs : a.n);
    s.middle = divider(s.heads_inside ? a.n : runs);
    const auto tensor = [](const void* at, const long* stride) { return Tensor{at, stride[1], stride[2], stride[0]}; };
    s.x = only_g ? tensor(a.g[i], a.g_stride[i]) : tensor(a.x[i], a.x_stride[i]);
    s.g = tensor(a.g[i], a.g_stride[i]);
    s.y = tensor(a.y[i], a.y_stride[i]);
    s.weight = a.norm ? a.weight[i] : nullptr;
    if (backward && a.gweight[i]) s.partial = partial + (i ? (long)p.blocks[0] * a.d : 0);
  }
  k.blocks0 = p.blocks[0];
  k.table = reinterpret_cast<const float2*>(a.table);
  k.index = a.index;
  k.table_stride = a.table_stride / 2;
  k.index_stride = a.index_stride;
  k.rows = a.rows, k.d = a.d, k.pairs = a.pairs, k.units = p.units, k.lanes = p.lanes, k.log_lanes = p.log_lanes;
  k.inv_d = 1.f / (float)a.d;
  k.eps = a.eps;
  k.stream = (size_t)(p.items[0] + p.items[1]) * p.most * a.d * (a.dtype == S2CNN_F32 ? 4 : 2) >= STREAM_BYTES;
  k.sign = backward ? -1.f : 1.f;
  return k;
}

template <class T, bool NEIGHBOURS, int HEADS, bool FULL> void launch(const Args& k, const Plan& p, bool norm, bool backward, hipStream_t s) {
  const dim3 grid(p.blocks[0] + p.blocks[1]);
  if (!norm) hipLaunchKernelGGL((rotary_kernel<T, TURN, NEIGHBOURS, HEADS, FULL>), grid, dim3(THREADS), 0, s, k);
  else if (!backward) hipLaunchKernelGGL((rotary_kernel<T, NORM, NEIGHBOURS, HEADS, FULL>), grid, dim3(THREADS), 0, s, k);
  else hipLaunchKernelGGL((rotary_kernel<T, NORM_BACK, NEIGHBOURS, (HEADS < 2 ? HEADS : 2), FULL>), grid, dim3(THREADS), 0, s, k);
}
template <class T, bool NEIGHBOURS> void launch(const Args& k, const Plan& p, bool norm, bool backward, hipStream_t s) {
  if (!p.full) launch<T, NEIGHBOURS, 1, false>(k, p, norm, backward, s);
  else if (p.most == 1) launch<T, NEIGHBOURS, 1, true>(k, p, norm, backward, s);
  else launch<T, NEIGHBOURS, 4, true>(k, p, norm, backward, s);
}
template <class T> void run(const s2cnn_rotary_t& a, bool backward, float* partial, hipStream_t s) {
  const Plan p = plan_of(a, backward && a.norm);
  const Args k = args_of(a, p, backward, partial);
  if (a.interleaved) launch<T, true>(k, p, a.norm != 0, backward, s);
  else launch<T, false>(k, p, a.norm != 0, backward, s);
  if (partial)
    hipLaunchKernelGGL(weights_kernel<T>, dim3((unsigned)((a.d + 31) / 32), 2), dim3(1024), 0, s, k.side[0].partial, k.side[1].partial, p.blocks[0], p.blocks[1], a.d,
                       static_cast<T*>(a.heads[0] ? a.gweight[0] : nullptr), static_cast<T*>(a.heads[1] ? a.gweight[1] : nullptr));
}
void run(const s2cnn_rotary_t& a, bool backward, float* partial, hipStream_t s) {
  if (a.dtype == S2CNN_F32) run<float>(a, backward, partial, s);
  else if (a.dtype == S2CNN_BF16) run<__bf16>(a, backward, partial, s);
  else run<half_t>(a, backward, partial, s);
}

// S2CNN_OK, or why a call is refused
int check(const s2cnn_rotary_t* a, bool backward) {
  if (!sizes_ok(a)) return S2CNN_EINVAL;
  const uintptr_t mask = a->dtype == S2CNN_F32 ? 3 : 1;
  for (int i = 0; i < 2; ++i) {
    if (!a->heads[i]) continue;
    const bool needs_x = !backward || a->norm;
    if ((needs_x && !a->x[i]) || (backward && !a->g[i]) || !a->y[i] || (a->weight[i] && !a->norm)) return S2CNN_EINVAL;
    if (a->gweight[i] && !(backward && a->norm)) return S2CNN_EINVAL;
    uintptr_t all = reinterpret_cast<uintptr_t>(a->y[i]) | reinterpret_cast<uintptr_t>(a->weight[i]) | reinterpret_cast<uintptr_t>(a->gweight[i]);
    if (needs_x) all |= reinterpret_cast<uintptr_t>(a->x[i]);
    if (backward) all |= reinterpret_cast<uintptr_t>(a->g[i]);
    if (all & mask) return S2CNN_EALIGN;
  }
  if (!aligned8(a->table) || (a->table_stride & 1) || (reinterpret_cast<uintptr_t>(a->index) & 3)) return S2CNN_EALIGN;
  return S2CNN_OK;
}
bool wants_sums(const s2cnn_rotary_t& a) { return a.norm && ((a.heads[0] && a.gweight[0]) || (a.heads[1] && a.gweight[1])); }

}  // namespace rotary
}  // namespace s2cnn

using namespace s2cnn;

extern "C" int s2cnn_rotary_fwd(const s2cnn_rotary_t* a, void* stream) {
  clear_stale_error();
  const int rc = rotary::check(a, false);
  if (rc) return rc;
  rotary::run(*a, false, nullptr, static_cast<hipStream_t>(stream));
  return launch_status();
}

extern "C" size_t s2cnn_rotary_workspace(const s2cnn_rotary_t* a) {
  if (!rotary::sizes_ok(a) || !a->norm) return 0;
  const rotary::Plan p = rotary::plan_of(*a, true);
  return ((size_t)p.blocks[0] + p.blocks[1]) * a->d * sizeof(float);
}

extern "C" int s2cnn_rotary_bwd(const s2cnn_rotary_t* a, void* workspace, size_t workspace_bytes, void* stream) {
  clear_stale_error();
  const int rc = rotary::check(a, true);
  if (rc) return rc;
  const bool sums = rotary::wants_sums(*a);
  if (sums && (!workspace || workspace_bytes < s2cnn_rotary_workspace(a) || !aligned16(workspace))) return S2CNN_EWORKSPACE;
  rotary::run(*a, true, sums ? static_cast<float*>(workspace) : nullptr, static_cast<hipStream_t>(stream));
  return launch_status();
}

extern "C" int s2cnn_rotary_table(const void* positions, int positions_type, const double* frequencies, float* table, long n, int axes, int pairs, float scale, void* stream) {
  clear_stale_error();
  if (!positions || !frequencies || !table || n < 1 || axes < 1 || axes > 1024 || pairs < 1 || pairs > rotary::MAX_D / 2 || n >= (1L << 40)) return S2CNN_EINVAL;
  if (positions_type < S2CNN_POSITIONS_F32 || positions_type > S2CNN_POSITIONS_I64) return S2CNN_EINVAL;
  const bool wide = positions_type == S2CNN_POSITIONS_F64 || positions_type == S2CNN_POSITIONS_I64;
  if ((reinterpret_cast<uintptr_t>(positions) & (wide ? 7 : 3)) || !aligned8(frequencies) || !aligned8(table)) return S2CNN_EALIGN;
  const bool two = pairs % 2 == 0;
  const long side = rotary::THREADS / (two ? pairs / 2 : pairs), need = (n + side - 1) / side, most = rotary::CUS * 16;
  const dim3 grid((unsigned)(need < most ? need : most)), block(rotary::THREADS);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float2* const out = reinterpret_cast<float2*>(table);
  const auto run = [&](auto* at) {
    if (two) hipLaunchKernelGGL(rotary::table_kernel<2>, grid, block, 0, s, at, frequencies, out, n, axes, pairs, scale);
    else hipLaunchKernelGGL(rotary::table_kernel<1>, grid, block, 0, s, at, frequencies, out, n, axes, pairs, scale);
  };
  switch (positions_type) {
    case S2CNN_POSITIONS_F32: run(static_cast<const float*>(positions)); break;
    case S2CNN_POSITIONS_F64: run(static_cast<const double*>(positions)); break;
    case S2CNN_POSITIONS_I32: run(static_cast<const int*>(positions)); break;
    default: run(static_cast<const long long*>(positions));
  }
  return launch_status();
}
