// What the attention kernels share: operand fragments of the matrix cores, the tiles of rows in LDS, the loads.
//
// All three kernels have one form.  A wave keeps 32 COLUMNS for good (queries, or keys in the kernel of the key and value
// gradients), their vectors as B operands in registers, and runs over tiles of 32 ROWS of the other side, which the workgroup
// stages in LDS.  A product of rows and columns (v_mfma_f32_32x32x16: 32 rows x 32 columns) leaves lane (h, c), h = lane / 32,
// c = lane % 32, with column c and the rows 8 g + 4 h + i in register 4 g + i: the softmax of a column and all that is known
// per column stays in one lane and the one 32 further on.  The second product contracts over the rows: register 8 t + j of
// a lane is taken as slot j of its B operand of step t, which makes slot j the row 16 t + 8 (j / 4) + 4 h + j % 4, and the A
// operand (the staged rows, transposed) is laid out in that order.  So the probabilities never leave their registers.
//
// float32 is computed on the bf16 matrix cores, each value the sum of three bf16 parts, six of the nine products of parts
// (split_bf16.h: the error is that of a float32 product; here without its power of two: parts of values below 2^-107 are
// lost).  bfloat16 and float16 take one product.  Everything between the products is float32.
#pragma once
#include "split_bf16.h"

namespace s2cnn {
namespace attn {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int ROWS = 32;             // rows of a staged tile, columns of a wave
constexpr int MAX_BUCKETS = 64;
constexpr int MAX_GROUP = 128;       // heads that share a key head where there are buckets: the table's rows of all of them are 33 KB of LDS

struct F32 { typedef float type; static constexpr int PARTS = 3; static constexpr bool HALF = false; };
struct BF16 { typedef __bf16 type; static constexpr int PARTS = 1; static constexpr bool HALF = false; };
// HALF: probabilities and their gradients are held times powers of two, as float16 has few exponents (see ScoreScale)
struct F16 { typedef _Float16 type; static constexpr int PARTS = 1; static constexpr bool HALF = true; };

__device__ __forceinline__ float ninf() { return -__builtin_inff(); }
__device__ __forceinline__ float pinf() { return __builtin_inff(); }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// the maximum / sum of a lane and the one 32 away, in both
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// LDS accesses of 16 and 8 bytes, free of the types that the bytes are written and read as: where a workgroup is one wave, its
// barriers order nothing for the compiler, and accesses of different types may then be exchanged.
__device__ __forceinline__ uint4 read16(const unsigned char* p) {
  uint4 v;
  __builtin_memcpy(&v, __builtin_assume_aligned(p, 16), 16);
  return v;
}
__device__ __forceinline__ void read16(const float* p, float (&x)[4]) { __builtin_memcpy(x, __builtin_assume_aligned(p, 16), 16); }
__device__ __forceinline__ void write8(unsigned char* p, unsigned a, unsigned b) {
  const uint2 v = make_uint2(a, b);
  __builtin_memcpy(__builtin_assume_aligned(p, 8), &v, 8);
}

__device__ __forceinline__ void write4(unsigned char* p, unsigned a) { __builtin_memcpy(__builtin_assume_aligned(p, 4), &a, 4); }

// ---- operands -------------------------------------------------------------------------------------------------------
template <class T> struct Frag { uint4 part[T::PARTS]; };

template <class T> __device__ __forceinline__ v16f mfma(uint4 a, uint4 b, v16f c) {
  if constexpr (T::HALF) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// c += a b, small products first.  TURNED: in the order of the product of b and a, so that the sums are the same
template <class T, bool TURNED = false> __device__ __forceinline__ void mma_small(const Frag<T>& a, const Frag<T>& b, v16f& c) {
  constexpr int I = TURNED ? 0 : 2, J = TURNED ? 0 : 1;
  c = mfma<T>(a.part[I], b.part[2 - I], c);
  c = mfma<T>(a.part[2 - I], b.part[I], c);
  c = mfma<T>(a.part[1], b.part[1], c);
  c = mfma<T>(a.part[J], b.part[1 - J], c);
  c = mfma<T>(a.part[1 - J], b.part[J], c);
}
template <class T, bool TURNED = false> __device__ __forceinline__ void mma(const Frag<T>& a, const Frag<T>& b, v16f& c) {
  if constexpr (T::PARTS == 3) mma_small<T, TURNED>(a, b, c);
  c = mfma<T>(a.part[0], b.part[0], c);
}

// two values as packed parts
template <class T> __device__ __forceinline__ void cut(float x, float y, unsigned (&w)[T::PARTS]) {
  if constexpr (T::PARTS == 3) split_pair<true>(x, y, w[0], w[1], w[2]);
  else if constexpr (T::HALF) w[0] = __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{x, y}, v2h));
  else w[0] = pack_bf16(x, y);
}
// two values times a factor as packed parts, float32; what is left of a first part is that of the product before its rounding.  Written
// out, so that it is so in every kernel: left to the compiler's contraction, one had other scores than another.
template <class T> __device__ __forceinline__ void cut_scaled(float x, float y, float factor, unsigned (&w)[3]) {
  w[0] = pack_bf16(x * factor, y * factor);
  const v2f h = {__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u)};
  const float xr = fmaf(x, factor, -h[0]), yr = fmaf(y, factor, -h[1]);
  w[1] = pack_bf16(xr, yr);
  w[2] = pack_bf16(xr - __uint_as_float(w[1] << 16), yr - __uint_as_float(w[1] & 0xffff0000u));
}
// what a packed pair of 16-bit values holds
template <class T> __device__ __forceinline__ v2f uncut(unsigned w) {
  if constexpr (T::HALF) return __builtin_convertvector(__builtin_bit_cast(v2h, w), v2f);
  else return v2f{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}
// sum + the two values of a packed pair
template <class T> __device__ __forceinline__ float add_pair(unsigned w, float sum) {
  if constexpr (T::HALF) return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), __builtin_bit_cast(v2h, 0x3c003c00u), sum, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w), __builtin_bit_cast(v2bf, 0x3f803f80u), sum, false);
}
template <class T, bool SCALE = false> __device__ __forceinline__ Frag<T> cut8(const float* x, float factor = 1.f) {
  unsigned w[4][T::PARTS];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if constexpr (SCALE) cut_scaled<T>(x[2 * i], x[2 * i + 1], factor, w[i]);
    else cut<T>(x[2 * i], x[2 * i + 1], w[i]);
  Frag<T> f;
#pragma unroll
  for (int p = 0; p < T::PARTS; ++p) f.part[p] = make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
  return f;
}
// registers 8 t .. 8 t + 7 of a product of rows and columns as the operand of step t of the product over the rows
template <class T> __device__ __forceinline__ Frag<T> cut_rows(const v16f& s, int t) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = s[8 * t + j];
  return cut8<T>(x);
}

// The 16-bit types' probabilities and their gradients go into their products as two parts, 16 bits in bfloat16 and 22 in float16.  Rounded to
// one they are off by as much as the result's own rounding: out and its gradients were 1.35 times as far from exact ones as rounded exact
// ones are, the table's gradient up to 1.5 times; with two parts the ratio is 1.00.  The price is a half more matrix instructions in the
// forward pass (73 -> 82 us at 16 signals, 8 heads, 1024 points of 64 entries); the backward pass, which had to round its
// probabilities as the forward pass did, gains as much.
template <class T> struct TwoParts {
  static constexpr int N = T::PARTS == 1 ? 2 : 1;
  Frag<T> part[N];
};
template <class T> __device__ __forceinline__ TwoParts<T> cut_rows_in_two(const v16f& s, int t) {
  TwoParts<T> f;
  f.part[0] = cut_rows<T>(s, t);
  if constexpr (T::PARTS == 1) {
    const unsigned w[4] = {f.part[0].part[0].x, f.part[0].part[0].y, f.part[0].part[0].z, f.part[0].part[0].w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v2f r = uncut<T>(w[i]);
      x[2 * i] = s[8 * t + 2 * i] - r[0], x[2 * i + 1] = s[8 * t + 2 * i + 1] - r[1];
    }
    f.part[1] = cut8<T>(x);
  }
  return f;
}
template <class T> __device__ __forceinline__ void mma(const Frag<T>& a, const TwoParts<T>& b, v16f& c) {
  if constexpr (T::PARTS == 1) mma<T>(a, b.part[1], c);
  mma<T>(a, b.part[0], c);
}

// ---- vectors in memory ----------------------------------------------------------------------------------------------
// The vectors of one (batch, head): vector i starts at base + i stride, at any entry, and has d entries.
template <class T> struct Vectors {
  const typename T::type* base;
  long stride;
  int n, d;
};

struct Quad { uint4 w; };            // four entries as they are in memory: floats, or 16-bit values in x and y

// A vector of d >= 4 entries is read, multiplied and written in quads: quad q holds entries 4 q .. 4 q + 3, the last one of a d
// that is no multiple of four the entries d - 4 .. d - 1, so that every access is one of four entries inside the vector.  Quads
// from d on hold any entries of it.  Columns have zeros for what is there twice or not at all (load_quad), so that it adds nothing to
// the products over the entries; in the products over the rows it makes entries that are written twice, or not.
// Vectors need no alignment: the memory pipeline takes any.
__device__ __forceinline__ int quad_at(int q, int d) { return 4 * q < d ? min(4 * q, d - 4) : 0; }
__device__ __forceinline__ int slot_of(int entry, int d) { return entry < (d & ~3) ? entry : entry + 4 - (d & 3); }    // where the quads hold it
template <class T> __device__ __forceinline__ Quad load_four(const typename T::type* p) {
  Quad v;
  if constexpr (T::PARTS == 3) __builtin_memcpy(&v.w, p, 16);
  else {
    uint2 u;
    __builtin_memcpy(&u, p, 8);
    v.w = make_uint4(u.x, u.y, 0, 0);
  }
  return v;
}
// the same from a uniform pointer and an offset in bytes: a scalar address and one register a lane, which the compiler would otherwise
// make 64-bit sums in every lane
template <class T> __device__ __forceinline__ Quad load_four_at(const typename T::type* uniform, unsigned bytes) {
  typedef unsigned words4 __attribute__((ext_vector_type(4), aligned(4), may_alias));
  typedef unsigned words2 __attribute__((ext_vector_type(2), aligned(2), may_alias));
  typedef const __attribute__((address_space(1))) char global_bytes;
  unsigned long long address = reinterpret_cast<unsigned long long>(uniform);
  asm("" : "+s"(address), "+v"(bytes));
  global_bytes* const p = reinterpret_cast<global_bytes*>(address) + bytes;
  Quad v;
  if constexpr (T::PARTS == 3) {
    const words4 u = *reinterpret_cast<const __attribute__((address_space(1))) words4*>(p);
    v.w = make_uint4(u.x, u.y, u.z, u.w);
  } else {
    const words2 u = *reinterpret_cast<const __attribute__((address_space(1))) words2*>(p);
    v.w = make_uint4(u.x, u.y, 0, 0);
  }
  return v;
}
// likewise a word of any alignment
__device__ __forceinline__ unsigned load_word_at(const signed char* uniform, unsigned bytes) {
  typedef unsigned word __attribute__((aligned(1), may_alias));
  typedef const __attribute__((address_space(1))) char global_bytes;
  unsigned long long address = reinterpret_cast<unsigned long long>(uniform);
  asm("" : "+s"(address), "+v"(bytes));
  return *reinterpret_cast<const __attribute__((address_space(1))) word*>(reinterpret_cast<global_bytes*>(address) + bytes);
}
template <class T> __device__ __forceinline__ Quad load_quad(const typename T::type* p, int q, int d) {
  Quad v = load_four<T>(p + quad_at(q, d));
  // So many of its first entries count as zero.  A column's quads each have their own number and four conditions on it, which the
  // compiler must not share between the vectors of a column (hundreds of scalar registers, and spills of them that went with wrong
  // results; the build refuses those): the empty statement hides that the numbers are equal.
  int twice = 4 * q < d ? 4 * q - quad_at(q, d) : 4;
  asm volatile("" : "+v"(twice));
  if constexpr (T::PARTS == 3) {
    if (twice > 0) v.w.x = 0;
    if (twice > 1) v.w.y = 0;
    if (twice > 2) v.w.z = 0;
    if (twice > 3) v.w.w = 0;
  } else {
    v.w.x &= twice > 1 ? 0 : twice > 0 ? 0xffff0000u : ~0u;
    v.w.y &= twice > 3 ? 0 : twice > 2 ? 0xffff0000u : ~0u;
  }
  return v;
}
template <class T, bool SCALE = false> __device__ __forceinline__ void quad_parts(const Quad& v, unsigned (&lo)[T::PARTS], unsigned (&hi)[T::PARTS], float factor = 1.f) {
  if constexpr (SCALE) {
    cut_scaled<T>(__uint_as_float(v.w.x), __uint_as_float(v.w.y), factor, lo);
    cut_scaled<T>(__uint_as_float(v.w.z), __uint_as_float(v.w.w), factor, hi);
  } else if constexpr (T::PARTS == 3) {
    cut<T>(__uint_as_float(v.w.x), __uint_as_float(v.w.y), lo);
    cut<T>(__uint_as_float(v.w.z), __uint_as_float(v.w.w), hi);
  } else {
    lo[0] = v.w.x;
    hi[0] = v.w.y;
  }
}
template <class T> __device__ __forceinline__ void quad_values(const Quad& v, float (&x)[4]) {
  if constexpr (T::PARTS == 3) {
    x[0] = __uint_as_float(v.w.x), x[1] = __uint_as_float(v.w.y), x[2] = __uint_as_float(v.w.z), x[3] = __uint_as_float(v.w.w);
  } else {
    const v2f a = uncut<T>(v.w.x), b = uncut<T>(v.w.y);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  }
}
template <class T> __device__ __forceinline__ void store_quad(typename T::type* p, int q, int d, float a, float b, float c, float e) {
  if (4 * q >= d) return;
  if constexpr (T::PARTS == 3) {
    const float4 x = make_float4(a, b, c, e);
    __builtin_memcpy(p + quad_at(q, d), &x, 16);
  } else {
    unsigned u[1], v[1];
    cut<T>(a, b, u), cut<T>(c, e, v);
    const uint2 x = make_uint2(u[0], v[0]);
    __builtin_memcpy(p + quad_at(q, d), &x, 8);
  }
}

// The B operands of one column: the vector at `p` (float32: times `factor`, 16-bit types: with its sign), in steps of 16 entries, 8 of them in either half of
// the wave.
template <class T, int D>
__device__ __forceinline__ void load_column(const typename T::type* p, int d, bool ok, int half, float factor, Frag<T> (&f)[D / 16]) {
  const unsigned flip = factor < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    Quad a = load_quad<T>(p, 4 * s + 2 * half, d), b = load_quad<T>(p, 4 * s + 2 * half + 1, d);
    if (!ok) a.w = b.w = make_uint4(0, 0, 0, 0);
    if constexpr (T::PARTS == 3) {
      float x[8];
      quad_values<T>(a, reinterpret_cast<float (&)[4]>(x[0]));
      quad_values<T>(b, reinterpret_cast<float (&)[4]>(x[4]));
      f[s] = cut8<T, true>(x, factor);
    } else {
      f[s].part[0] = make_uint4(a.w.x ^ flip, a.w.y ^ flip, b.w.x ^ flip, b.w.y ^ flip);
    }
  }
}

// acc[b][4 g + i] is entry 32 b + 8 g + 4 half + i of the lane's column
template <class T, int D> __device__ __forceinline__ void store_column(typename T::type* p, int d, int half, const v16f (&acc)[D / 32], float factor) {
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      store_quad<T>(p, 8 * b + 2 * g + half, d, acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor, acc[b][4 * g + 2] * factor,
                    acc[b][4 * g + 3] * factor);
}
// the same into an array of partial sums, D floats a column
template <int D> __device__ __forceinline__ void store_partial(float* p, int half, const v16f (&acc)[D / 32]) {
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(p + 32 * b + 8 * g + 4 * half) = make_float4(acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]);
}

// ---- a tile of 32 rows in LDS ---------------------------------------------------------------------------------------
// Two layouts, both as the A operands are read: 1 KB per part and step, 16 bytes a lane.
//   by rows: step s of the product over the entries; lane (h, r) reads entries 16 s + 8 h .. + 7 of row r
//   by entries: block b of 32 entries, step t of the product over the rows; lane (h, m) reads entry 32 b + m of the rows above
// A thread of the staging holds a block of 4 rows x 4 entries, and writes 8 bytes per row or entry.  The 16-byte slots are
// permuted (by s and h, or by m / 8) so that these writes go to all banks; readers permute within 128 bytes and lose nothing.
enum Layouts { BY_ROWS = 1, BY_ENTRIES = 2, BOTH = 3 };
template <class T, int D> struct Tile {
  static constexpr int STEPS = D / 16;                             // as many KB per part in either layout
  static constexpr int BYTES = T::PARTS * STEPS * 1024;
  static constexpr int BLOCKS = (ROWS / 4) * (D / 4);

  static __device__ __forceinline__ int row_slot(int s, int h, int r) { return (h * 32 + r) ^ ((2 * s + h) & 7); }
  static __device__ __forceinline__ int entry_slot(int h, int m) { return h * 32 + (m ^ ((m >> 3) & 3)); }

  static __device__ __forceinline__ Frag<T> by_rows(const unsigned char* lds, int s, int lane) {
    Frag<T> f;
    const int at = row_slot(s, lane >> 5, lane & 31);
#pragma unroll
    for (int p = 0; p < T::PARTS; ++p) f.part[p] = read16(lds + ((p * STEPS + s) * 64 + at) * 16);
    return f;
  }
  static __device__ __forceinline__ uint4 first_by_rows(const unsigned char* lds, int s, int lane) {      // the first part alone
    return read16(lds + (s * 64 + row_slot(s, lane >> 5, lane & 31)) * 16);
  }
  static __device__ __forceinline__ Frag<T> by_entries(const unsigned char* lds, int b, int t, int lane) {
    Frag<T> f;
    const int at = entry_slot(lane >> 5, lane & 31);
#pragma unroll
    for (int p = 0; p < T::PARTS; ++p) f.part[p] = read16(lds + ((p * STEPS + 2 * b + t) * 64 + at) * 16);
    return f;
  }

  // where a block of the tile is written that begins with row `row` (a multiple of two) and entry 4 q: its first row, its first entry.  The
  // others are as many slots on, exclusive or: they differ in the two lowest bits of the slot alone
  static __device__ __forceinline__ unsigned rows_at(int row, int q) {
    const int s = q >> 2, h = (q >> 1) & 1;
    return (unsigned)((s * 64 + row_slot(s, h, row)) * 16 + (q & 1) * 8);
  }
  static __device__ __forceinline__ unsigned entries_at(int row, int q) {
    const int b = q >> 3, t = row >> 4, half = (row >> 3) & 1, h = (row >> 2) & 1;
    return (unsigned)(((2 * b + t) * 64 + entry_slot(h, (4 * q) & 31)) * 16 + half * 8 + (row & 3) * 2);
  }
  // a block of N rows (2 or 4) into the layouts, at the places `at_rows` and `at_entries`; LAYOUTS: which of the two
  template <int LAYOUTS, int N, bool SCALE = false>
  static __device__ __forceinline__ void write(unsigned char* rows, unsigned char* entries, unsigned at_rows, unsigned at_entries, const Quad (&v)[N], float factor = 1.f) {
    unsigned w[N][2][T::PARTS];                                    // [row][pair of entries][part]
#pragma unroll
    for (int i = 0; i < N; ++i) quad_parts<T, SCALE>(v[i], w[i][0], w[i][1], factor);
    if constexpr ((LAYOUTS & BY_ROWS) != 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int p = 0; p < T::PARTS; ++p) write8(rows + (at_rows ^ (16 * i)) + p * STEPS * 1024, w[i][0][p], w[i][1][p]);
    }
    if constexpr ((LAYOUTS & BY_ENTRIES) != 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned sel = (j & 1) ? 0x07060302u : 0x05040100u;  // the entry's 16 bits of two rows
#pragma unroll
        for (int p = 0; p < T::PARTS; ++p) {
          unsigned char* const to = entries + (at_entries ^ (16 * j)) + p * STEPS * 1024;
          const unsigned two = __builtin_amdgcn_perm(w[1][j >> 1][p], w[0][j >> 1][p], sel);
          if constexpr (N == 4) write8(to, two, __builtin_amdgcn_perm(w[3][j >> 1][p], w[2][j >> 1][p], sel));
          else write4(to, two);
        }
      }
    }
  }
};

// LDS of a kernel that stages `layouts` layouts of a tile: two tiles where they fit beside a second workgroup, so that a tile is
// written while the one before is used, with one barrier per tile; else one.  One, too, where the workgroup is a wave: it fetches
// a tile and writes it at once (a thread has up to eight blocks then, too many registers to hold beside the operands), and the
// other waves of the CU are what hides the wait.
template <class T, int D, int W> constexpr int buffers(int layouts) { return W > 1 && 2 * layouts * Tile<T, D>::BYTES <= 64 * 1024 ? 2 : 1; }

// Two tensors staged by the same tiles of rows, in the layouts LA and LB (those of the first, then those of the second): THREADS threads
// fetch the blocks of a tile into registers, and write them later.
// The address of a block's rows is a uniform pointer, moved on by the tile, and an offset of the thread that stays (below
// 2^32 bytes: the entry checks 32 strides).
// SCALE: the first tensor is staged times `factor` (float32).
template <class T, int D, int THREADS, int LA, int LB, bool SCALE = false> struct Stage {
  typedef Tile<T, D> Tl;
  typedef typename T::type E;
  static constexpr int A = LA == BOTH ? 2 * Tl::BYTES : Tl::BYTES;      // where the second tensor's layouts begin
  static constexpr int N = 2 * Tl::BLOCKS < THREADS ? 2 : 4;           // rows of a block: two where four leave threads without one
  static constexpr int BLOCKS = Tl::BLOCKS * 4 / N;
  static constexpr int PER = (2 * BLOCKS + THREADS - 1) / THREADS;
  static constexpr bool IDLE = 2 * BLOCKS % THREADS != 0;      // some threads have no block
  Quad v[PER][N];
  unsigned offset[PER], at_rows[PER], at_entries[PER];
  float factor = 1.f;

  // of the thread's block u: which tensor (uniform in a wave), and which block of it
  static __device__ __forceinline__ bool second(int u, int tid) {
    if constexpr (BLOCKS % THREADS == 0) return u >= PER / 2;
    else return __builtin_amdgcn_readfirstlane(u * THREADS + tid) >= BLOCKS;
  }
  static __device__ __forceinline__ bool idle(int u, int tid) { return IDLE && __builtin_amdgcn_readfirstlane(u * THREADS + tid) >= 2 * BLOCKS; }
  static __device__ __forceinline__ int block(int u, int tid) { return (u * THREADS + tid) % BLOCKS; }

  // bytes from the tile's first row to row i of block u, or to row `last` if that comes before it
  static __device__ __forceinline__ unsigned place(const Vectors<T>& x, int u, int tid, int i, int last) {
    const int kk = block(u, tid);
    return (unsigned)sizeof(E) * (unsigned)(min(N * (kk / (D / 4)) + i, last) * (int)x.stride + quad_at(kk % (D / 4), x.d));
  }
  static __device__ __forceinline__ unsigned in_rows(int u, int tid) { return Tl::rows_at(N * (block(u, tid) / (D / 4)), block(u, tid) % (D / 4)); }
  static __device__ __forceinline__ unsigned in_entries(int u, int tid) { return Tl::entries_at(N * (block(u, tid) / (D / 4)), block(u, tid) % (D / 4)); }
  // before the first fetch; the strides and sizes are those of all
  __device__ __forceinline__ void prepare(const Vectors<T>& a, const Vectors<T>& b, int tid) {
    if constexpr (THREADS == 64) return;                   // a wave has too many blocks to keep their offsets
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      offset[u] = place(second(u, tid) ? b : a, u, tid, 0, ROWS);
      at_rows[u] = in_rows(u, tid), at_entries[u] = in_entries(u, tid);
    }
  }

  // blocks [U0, U1) of the thread
  template <int U0 = 0, int U1 = PER> __device__ __forceinline__ void fetch(const Vectors<T>& a, const Vectors<T>& b, int row0, int tid) {
#pragma unroll
    for (int u = U0; u < U1; ++u) {
      if (idle(u, tid)) break;
      const Vectors<T>& x = second(u, tid) ? b : a;
      const unsigned stride = (unsigned)x.stride;          // below 2^25, so that products with it are of 32 bits
      const E* const base = x.base + (unsigned long long)(unsigned)row0 * stride;
      const int left = x.n - 1 - row0;                     // last row of the tile that exists
      if (left >= ROWS - 1) {
        const unsigned at = THREADS == 64 ? place(x, u, tid, 0, ROWS) : offset[u];
#pragma unroll
        for (int i = 0; i < N; ++i) v[u][i] = load_four_at<T>(base + i * stride, at);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[u][i] = load_four_at<T>(base, place(x, u, tid, i, left));
        asm volatile("");                                  // keeps the last load of both branches from becoming one, of a 64-bit address
      }
    }
  }
  // keep(row of the tile): false for rows that count as zero, whatever their memory holds
  template <int U0 = 0, int U1 = PER, class Keep>
  __device__ __forceinline__ void write(unsigned char* to, int tid, Keep keep) {
#pragma unroll
    for (int u = U0; u < U1; ++u) {
      if (idle(u, tid)) break;
      const int row = N * (block(u, tid) / (D / 4));
      bool k[N], all = true;
#pragma unroll
      for (int i = 0; i < N; ++i) k[i] = keep(row + i), all = all && k[i];
      if (!__all(all)) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (!k[i]) v[u][i].w = make_uint4(0, 0, 0, 0);
      }
      unsigned r = THREADS == 64 ? in_rows(u, tid) : at_rows[u], e = THREADS == 64 ? in_entries(u, tid) : at_entries[u];
      asm volatile("" : "+v"(r), "+v"(e));                 // four places each, formed here: kept from tile to tile they were registers spilled
      if (second(u, tid)) Tl::template write<LB, N>(to + A, to + A + (LB == BOTH ? Tl::BYTES : 0), r, e, v[u]);
      else Tl::template write<LA, N, SCALE>(to, to + (LA == BOTH ? Tl::BYTES : 0), r, e, v[u], factor);
    }
  }
  // a wave's own way: fetch and write, one tensor after the other, so that half the registers do
  template <class Keep>
  __device__ __forceinline__ void fetch_and_write(const Vectors<T>& a, const Vectors<T>& b, int row0, unsigned char* to, int tid, Keep keep) {
    static_assert(THREADS == 64, "one wave");
    fetch<0, PER / 2>(a, b, row0, tid);
    write<0, PER / 2>(to, tid, keep);
    __builtin_amdgcn_sched_barrier(0);
    fetch<PER / 2, PER>(a, b, row0, tid);
    write<PER / 2, PER>(to, tid, keep);
  }
  // the largest |entry| of the second tensor's blocks, as they were written
  __device__ __forceinline__ float largest_second(int tid) const {
    float t = 0.f;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if (idle(u, tid)) break;
      if (!second(u, tid)) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float x[4];
        quad_values<T>(v[u][i], x);
#pragma unroll
        for (int e = 0; e < 4; ++e) t = fmaxf(t, fabsf(x[e]));
      }
    }
    return t;
  }
};

// ---- scores -----------------------------------------------------------------------------------------------------------
// Scores are kept in base 2: x = log2(e) (scale q.k + table + key bias), the factor in the scale, the table and the key biases.
// The reference that a query's probabilities are taken to, 2^(x - reference), is an integer, its largest score rounded up: a change of
// it is an exact factor, and a query seldom has one after its first tiles, so that the output is multiplied only in those.  The
// sum of a query is that of the parts that enter its product, so that a query with one key has its value exactly.
//
// The product starts from the biases instead of zero: x = c (q.k + bias / c), c = log2(e) |scale|; float32 takes c into the queries as
// they are loaded, and needs no factor; the other types take the sign.  All kernels form a score from the same numbers in the same order: the
// references are of scores as the forward pass had them, and a score of 10^4 that is rounded otherwise makes another probability.  Biases of
// keys and entries of the table are held within +-1.5e38 of a score, so that the type's lowest value stays finite, and the sum of two: keys
// that all have it share a row evenly.
// In two steps, the load and what is made of it: the tiles' loads are under way in between, and a wait for this one, issued before them,
// is no wait for them.
__device__ __forceinline__ float load_key_bias(const float* key_bias, int key, int end) { return key_bias ? key_bias[max(min(key, end - 1), 0)] : 0.f; }
// most: the largest magnitude of a bias, in units of c
__device__ __forceinline__ float key_value(float bias, int key, int end, float inv_c, float most) {
  const float x = bias * LOG2E * inv_c;
  const float y = fabsf(bias) < pinf() ? __builtin_amdgcn_fmed3f(x, -most, most) : x;
  return key < end ? y : ninf();                           // takes no part
}

// Scores of the 16-bit types are multiplied by c and taken off their reference in one operation, whose product is not rounded; the reference is
// a rounded product, off by up to 2^-25 of it.  That is nothing for any score of use, but at 2^27 (float16) a probability of 2^9, at 2^32 none or
// infinity: rows whose keys all have biases of -10^9, or the type's lowest value.  Where a query's largest score has passed 2^24, its scores and
// the reference are taken times the power of two that brings it below: a factor of the query in place of c, exact, the same in all kernels, and no
// operation more.  Such scores keep a resolution of 2^-24 of the largest in place of one unit, which is what their sums are rounded to.
__device__ __forceinline__ float shrink(float top) {
  const int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;
  return __uint_as_float((unsigned)(127 - max(0, e - 23)) << 23);
}
// What a query's probabilities are taken to, from its largest score rounded up, and the factor of its scores.  float16: 2^10 of the probabilities,
// as its smallest normal number is 2^-14.
struct Reference { float at, c; };
template <class T> __device__ __forceinline__ Reference reference(float top, float c) {
  if constexpr (T::PARTS == 3) return {top, c};
  const float by = shrink(top);
  return {fmaf(top, by, T::HALF ? -10.f : 0.f), c * by};
}
template <class T> __device__ __forceinline__ float off_reference(float s, const Reference& r) { return T::PARTS == 3 ? s - r.at : fmaf(s, r.c, -r.at); }
// 2^(a - b) of two largest scores, a <= b, as the probabilities that are taken to them have it
template <class T> __device__ __forceinline__ float fade_to(float b, float a) { return exp2_(T::PARTS == 3 ? a - b : (a - b) * shrink(b)); }

// A tile's values of its rows (keys' biases; the queries' statistics) in LDS, in a ring: tile t's are read in step t, and in step
// t - 1, in which its rows are written; they are put there at the start of step t - 2, and loaded in step t - 3: put at that step's end
// they would wait for its tile's loads too, which are issued after them.
constexpr int RING = 4;

// the table's rows of heads head0 .. head0 + heads - 1 in LDS, n_buckets + 1 entries a head, the last one for excluded pairs; most: the largest
// magnitude of a finite one
template <class T> __device__ __forceinline__ void stage_table(float* lds, const void* table, int n_buckets, int head0, int heads, float most, int tid, int threads) {
  const typename T::type* t = static_cast<const typename T::type*>(table);
  for (int k = tid; k < heads * (n_buckets + 1); k += threads) {
    const int h = k / (n_buckets + 1), n = k % (n_buckets + 1);
    const float x = n == n_buckets ? ninf() : (float)t[(long)(head0 + h) * n_buckets + n];
    lds[k] = fabsf(x) < pinf() ? __builtin_amdgcn_fmed3f(x * LOG2E, -most, most) : x;
  }
}

// Buckets of the lane's column and keys key0 + 8 g + 4 half + i, a byte each; 255 past the end.  A lane loads 16 bytes, the first or the second
// half of its row's 32, in place of four words of four: a quarter of the requests, each of which is to 32 rows.  The two lanes of a row
// then exchange words: those of groups 0 and 2 are the first two of either, those of 1 and 3 the others.  The exchange is left to
// place_buckets, so that the load can be under way.
__device__ __forceinline__ void load_buckets(const signed char* row, int key0, int end, int half, unsigned (&w)[4]) {
  if (key0 + ROWS <= end) {
#pragma unroll
    for (int g = 0; g < 4; ++g) __builtin_memcpy(&w[g], row + key0 + 16 * half + 4 * g, 4);
  } else {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      w[g] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * half + 4 * g + i;
        w[g] |= (key < end ? (unsigned)(unsigned char)row[key] : 255u) << (8 * i);
      }
    }
  }
}
__device__ __forceinline__ void place_buckets(const unsigned (&w)[4], unsigned (&now)[4]) {
  const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false), b = __builtin_amdgcn_permlane32_swap(w[2], w[3], false, false);
  now[0] = a[0], now[1] = b[0], now[2] = a[1], now[3] = b[1];
}
__device__ __forceinline__ int bucket_of(unsigned w, int i, int n_buckets) { return min((int)((w >> (8 * i)) & 255u), n_buckets); }

// Whether a wave's words of a tile exclude every pair of it: with a bias over near points only, most tiles of far ones.  The wave leaves
// them out: they would add zeros.  (Excluded by negative numbers; by positive ones beyond the table they are formed as any other.)
__device__ __forceinline__ bool none_takes_part(const unsigned (&w)[4]) { return __all((w[0] & w[1] & w[2] & w[3] & 0x80808080u) == 0x80808080u); }

// What the scores of a tile start from: the keys' biases, and the table's entries of the pairs where there are buckets.  In the
// accumulators before the product begins, they need no registers beside them.
template <class T> __device__ __forceinline__ void start_scores(v16f& s, const float* kb, int half, bool buckets, const unsigned (&words)[4], const float* table,
                                                                int n_buckets, float inv_c) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float start[4];
    read16(kb + 8 * g + 4 * half, start);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * g + i] = start[i];
  }
  if (buckets) {
    float t[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r] = table[bucket_of(words[r / 4], r % 4, n_buckets)];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = T::PARTS == 3 ? s[r] + t[r] : fmaf(t[r], inv_c, s[r]);
  }
}

// ---- arguments ------------------------------------------------------------------------------------------------------
// The header's struct and what the entry has made of it.
struct Args {
  s2cnn_attention_t a;
  float c, inv_c;          // log2(e) |scale| and its inverse; 1 for float32
  float most;              // see key_value
  int forward_splits;
  int splits;              // parts of the long axis (keys; queries in the kernel of dk and dv)
  int tiles;               // workgroups along the columns
  int workgroups;
  float* partial;          // results of the parts
  double* gtable_partial;  // of every workgroup
  int gtable_parts;        // workgroups of a signal and head
  float* delta;            // [batch, heads, n_q] dout . out; float16: then the exponents of their ds
};

// Consecutive workgroups go to the eight XCDs in turn: the ones that read the same rows are given numbers of one XCD.  Not where signals
// have lengths of their own: an XCD would have the longest ones alone, so each gets tiles of all.
__device__ __forceinline__ int work_of_block(const Args& p) {
  if (p.a.lengths) return (int)blockIdx.x;
  const int per = (p.workgroups + 7) / 8;
  return (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
}
// Signal and head of group i of `per` heads a signal; of signals with lengths of their own, the heads follow those of the other signals.
struct Group { int b, head; };
__device__ __forceinline__ Group group_of(const s2cnn_attention_t& a, int i, int per) { return a.lengths ? Group{i % a.batch, i / a.batch} : Group{i / per, i % per}; }
// Tiles of one number see as many pairs in every group (near the poles of a grid with a bias over near points: few), and a CU's workgroups
// are 32 apart: each group's tiles are turned by three eighths.
__device__ __forceinline__ int tile_of(const Args& p, int work, int group) { return (work + group % 8 * (p.tiles * 3 / 8)) % p.tiles; }
__host__ __device__ inline int blocks_for(int workgroups) { return (workgroups + 7) / 8 * 8; }


// ---- launches -------------------------------------------------------------------------------------------------------
// Whether there are workgroups of one wave.  Not for float32 heads of more than 64 entries: a wave's operands and a thread's share of a tile
// are more than its registers then.
template <class T, int D> constexpr bool few_waves = T::PARTS * D <= 256;

// How a kernel's work is laid out: waves per workgroup, workgroups along the columns, parts of the long axis.
struct Plan { int waves, tiles, splits; long workgroups; };
struct Plans { int D; Plan fwd, grad_q, grad_kv; };

template <class K> void launch(K kernel, const Args& p, int waves, size_t lds, hipStream_t stream, int beyond = 0) {
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks_for(p.workgroups) + beyond)), dim3(64 * waves), lds, stream, p);
}

// one translation unit per type
template <class T> void forward(const Args& p, const Plans& plans, hipStream_t stream);
template <class T> void backward(Args p, const Plans& plans, float* partial_q, float* partial_kv, hipStream_t stream);

}  // namespace attn
}  // namespace s2cnn
