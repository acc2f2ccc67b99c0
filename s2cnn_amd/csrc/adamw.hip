// The step of an optimizer over a list of tensors (AdamW), with moments in 32 or in 8 bits, and the norm of a list of gradients.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p - lr decay p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// with g multiplied by min(1, max_norm / norm) first where a norm is given.  Bound by memory: every tensor is read once and written once, in one
// launch for some fifty tensors, whose addresses travel in the kernel's arguments: nothing is copied to the device, and a captured graph keeps them.
// A workgroup takes 2048 entries of one tensor, four or eight a lane at a time, all loads of a wave under way together.
//
// Measured, with a copy of 1 GiB at 5.1 TB/s: 134 million parameters in float32, 28 bytes each: 704 to 713 us, 5.3 TB/s (past the caches: the same); 25 million in bfloat16
// with masters and moments in 8 bits, 18 bytes each: 97 us in three launches, 4.7 TB/s, where vector instructions take 0.55 of the SIMDs' time, a third of them for
// the random numbers (each load waited for by itself: 115; four entries a lane, both ways of rounding formed for every entry: 122); the
// decoded moments of these, 10 bytes each: 44 us, 5.7 TB/s.  28 tensors of 0.15 million together: 5 us.
//
// Moments in 8 bits.  A block of 256 entries (32 lanes') has a factor s of each moment; an entry is s f(c), f(c) = c for c < 8, (8 + c % 8) 2^(c / 8 - 1)
// beyond: three bits after the leading one, so that a step is 1/8 to 1/16 of the value.  First moments: a sign and c <= 126, in units of 2^-9
// the type float8_e4m3fn.  Second moments: c <= 255, 2^34 from the smallest to the largest, because their roots go through the same range as
// first moments do, and never 0 where the moment is not: the quotient stays bounded.  A step changes a second moment by a thousandth
// (b2 = 0.999), far below the spacing, and would be rounded away; so both are rounded up or down at random, with the probability that leaves the
// mean right.  The random bits are a function of the seed, the step and the entry's number: 16 for each moment.
// m, v, s and the codes are formed by single float32 operations in the order written, without fused ones: a program that does the same gets the same codes.
#include <float.h>
#include <stdlib.h>
#include "chunk.h"
#include "counter_random.h"

namespace s2cnn {
namespace adamw {

constexpr int THREADS = 256;
constexpr int BLOCK = 256;                     // entries of a factor
constexpr int PART = 2048;                     // entries of a workgroup
constexpr int MOST = 56;                       // tensors of a launch: 4 KB of arguments
constexpr int MOST_SUMS = 184;
constexpr float TOP_FIRST = 229376.f, TOP_SECOND = 15.f * 1073741824.f;      // f(126), f(255)

struct Tensors {
  void* p[MOST];
  const void* g[MOST];
  void* first[MOST];
  void* second[MOST];
  float2* scales[MOST];
  float* master[MOST];
  long n[MOST];
  unsigned long long counter[MOST];            // random numbers before this tensor's, in fours
  unsigned part[MOST + 1];                     // workgroups before this tensor's
  int count;
};
struct Step {
  const float *lr_at, *norm;
  const long long* step_at;
  long long step;
  unsigned long long seed;
  float log_b1, log_b2, lr, b1, rest1, b2, rest2, eps, decay, max_norm;
};
static_assert(sizeof(Tensors) + sizeof(Step) <= 4096, "kernel arguments");

// The tensor of workgroup `part`: the last whose first workgroup is not behind it.
template <int N> __device__ __forceinline__ int tensor_of(const unsigned (&first)[N], int count, unsigned part) {
  int low = 0, high = count;
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (first[mid] <= part) low = mid;
    else high = mid;
  }
  return low;
}

// N entries at any address of the type; not FULL: the first n of them, the others zero
template <bool FULL, class T, int N> __device__ __forceinline__ void load(const T* p, long n, float (&v)[N]) {
  if (FULL || n >= N) {
    typedef T loose __attribute__((ext_vector_type(sizeof(T) == 4 ? 4 : N), aligned(sizeof(T))));
    constexpr int M = sizeof(T) == 4 ? 4 : N;
#pragma unroll
    for (int k = 0; k < N / M; ++k) {
      const loose x = *reinterpret_cast<const loose*>(p + k * M);
#pragma unroll
      for (int i = 0; i < M; ++i) v[k * M + i] = (float)x[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
}
template <bool FULL, class T, int N> __device__ __forceinline__ void store(T* p, long n, const float (&v)[N]) {
  if (FULL || n >= N) {
    constexpr int M = sizeof(T) == 4 ? 4 : N;
    typedef T loose __attribute__((ext_vector_type(M), aligned(sizeof(T))));
#pragma unroll
    for (int k = 0; k < N / M; ++k) {
      loose x;
#pragma unroll
      for (int i = 0; i < M; ++i) x[i] = (T)v[k * M + i];
      *reinterpret_cast<loose*>(p + k * M) = x;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = (T)v[i];
}
// eight bytes in the same way
typedef unsigned loose2 __attribute__((ext_vector_type(2), aligned(1)));
template <bool FULL> __device__ __forceinline__ uint2 load8(const unsigned char* p, long n) {
  if (FULL || n >= 8) {
    const loose2 x = *reinterpret_cast<const loose2*>(p);
    return make_uint2(x[0], x[1]);
  }
  unsigned c[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) c[i / 4] |= (unsigned)p[i] << (8 * (i % 4));
  return make_uint2(c[0], c[1]);
}
template <bool FULL> __device__ __forceinline__ void store8(unsigned char* p, long n, uint2 c) {
  if (FULL || n >= 8) {
    *reinterpret_cast<loose2*>(p) = loose2{c.x, c.y};
    return;
  }
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) p[i] = (unsigned char)((i < 4 ? c.x : c.y) >> (8 * (i % 4)));
}

// ---- codes ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void first_of(uint2 codes, float s, float (&m)[8]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned c = k ? codes.y : codes.x;
    const f2 low = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    m[4 * k] = low[0] * 512.f * s, m[4 * k + 1] = low[1] * 512.f * s, m[4 * k + 2] = high[0] * 512.f * s, m[4 * k + 3] = high[1] * 512.f * s;
  }
}
// f(c) 2^-129 is the float32 of bits c 2^20: the codes below eight are its subnormal numbers, and the product with 2^127 is exact.
__device__ __forceinline__ void second_of(uint2 codes, float s, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float((((i < 4 ? codes.x : codes.y) >> (8 * (i % 4))) & 255u) << 20) * 0x1p127f * (4.f * s);
}
// A block's factor from its largest entry (the bits of a float32 without sign, so that what is no number is the largest); below 2^-126 none.
__device__ __forceinline__ float factor_of(unsigned largest, float inverse_top) {
#pragma clang fp contract(off)
  const float s = __uint_as_float(largest) * inverse_top;
  return s < 0x1p-126f ? 0.f : s;
}
__device__ __forceinline__ unsigned max_block(unsigned v) {           // over 32 lanes, in all of them
  const auto with = [&](unsigned o) { v = max(v, o); };
  with(__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(a[0], a[1]);
}
// The code of y >= 0, rounded by 16 random bits, in the upper byte.  From 8 on it is in the bits of the float32 with those added behind the three that
// stay.  No code is above that of the largest entry, which is off by less than 2^-21 of itself from its code's value: 2^-17 of a spacing, less than what
// the largest random number leaves.
__device__ __forceinline__ unsigned upper_code(float y, unsigned random) { return (__float_as_uint(y) + ((random << 4) - (129u << 23))) << 4; }
__device__ __forceinline__ unsigned any_code(float y, unsigned random) {
  return y >= 8.f ? upper_code(y, random) >> 24 : (unsigned)(y + (float)random * 0x1p-16f);
}
// the upper bytes of four words
__device__ __forceinline__ unsigned upper_bytes(const unsigned (&x)[4]) {
  const unsigned low = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0703u), high = __builtin_amdgcn_perm(x[3], x[2], 0x07030c0cu);
  return low | high;
}

// Eight entries of a block of 256, whose factors' inverses are i1 and i2: codes of m and v.
__device__ __forceinline__ void codes_of(const float (&m)[8], const float (&v)[8], float i1, float i2, const uint4 (&random)[2], uint2& c1, uint2& c2) {
#pragma clang fp contract(off)
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = fabsf(m[i]) * i1, b[i] = v[i] * i2;
  const unsigned r[8] = {random[0].x, random[0].y, random[0].z, random[0].w, random[1].x, random[1].y, random[1].z, random[1].w};
  unsigned x[2][4], y[2][4];
  bool high = true;                                                // all from 8 on; what is no number is not
#pragma unroll
  for (int i = 0; i < 8; ++i) high &= a[i] >= 8.f && b[i] >= 8.f;
  if (__all(high)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i / 4][i % 4] = (upper_code(a[i], r[i] & 0xffffu) & 0x7fffffffu) | (__float_as_uint(m[i]) & 0x80000000u);
      y[i / 4][i % 4] = upper_code(b[i], r[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i / 4][i % 4] = (any_code(a[i], r[i] & 0xffffu) | (m[i] < 0.f ? 128u : 0u)) << 24;
      y[i / 4][i % 4] = max(any_code(b[i], r[i] >> 16), v[i] > 0.f && i2 > 0.f ? 1u : 0u) << 24;
    }
  }
  c1 = make_uint2(upper_bytes(x[0]), upper_bytes(x[1]));
  c2 = make_uint2(upper_bytes(y[0]), upper_bytes(y[1]));
}

struct Factors {
  long long step;
  float clip, size, inverse2, decay;
};

// The entries of a lane from `at` on, N of them; not FULL: the first `left`.
template <class T, int BITS, bool MASTER, bool FULL> __device__ __forceinline__ void step_entries(const Tensors& t, int k, const Step& h, const Factors& f, long at, long left) {
  constexpr int N = BITS == 8 ? 8 : 4;
  float g[N], p[N], m[N], v[N], master[N];
  load<FULL, T>(static_cast<const T*>(t.g[k]) + at, left, g);
  load<FULL, T>(static_cast<T*>(t.p[k]) + at, left, p);
  if constexpr (MASTER) load<FULL, float>(t.master[k] + at, left, master);
  const long block = at / BLOCK;                                    // 8 bits: of 32 lanes
  if constexpr (BITS == 32) {
    load<FULL, float>(static_cast<float*>(t.first[k]) + at, left, m);
    load<FULL, float>(static_cast<float*>(t.second[k]) + at, left, v);
  } else {
    const float2 s = FULL || left > 0 ? t.scales[k][block] : make_float2(0.f, 0.f);
    const uint2 c1 = load8<FULL>(static_cast<unsigned char*>(t.first[k]) + at, left), c2 = load8<FULL>(static_cast<unsigned char*>(t.second[k]) + at, left);
    first_of(c1, s.x, m);
    second_of(c2, s.y, v);
  }
  {
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      g[i] *= f.clip;
      m[i] = m[i] * h.b1 + g[i] * h.rest1;
      v[i] = v[i] * h.b2 + (g[i] * g[i]) * h.rest2;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (MASTER) p[i] = (float)(T)master[i] == p[i] ? master[i] : p[i];     // where it is not its master's rounding, the program has set it since
    // the instruction takes a subnormal number's root for zero: small ones are taken times 2^32
    const bool small = v[i] < 0x1p-96f;
    const float denominator = fmaf(__builtin_amdgcn_sqrtf(v[i] * (small ? f.inverse2 * 0x1p32f : f.inverse2)), small ? 0x1p-16f : 1.f, h.eps);
    // what decays of an infinite parameter (a mask) is finite: it stays
    const float kept = fmaf(-f.decay, __builtin_amdgcn_fmed3f(p[i], -FLT_MAX, FLT_MAX), p[i]);
    p[i] = fmaf(-f.size, m[i] * __builtin_amdgcn_rcpf(denominator), kept);
    // The parameter is the rounding of the float32 that is stored: without this the compiler makes one operation of the last product, sum and conversion
    // to float16, which rounds once and may differ.
    if constexpr (MASTER) asm volatile("" : "+v"(p[i]));
  }
  store<FULL, T>(static_cast<T*>(t.p[k]) + at, left, p);
  if constexpr (MASTER) store<FULL, float>(t.master[k] + at, left, p);
  if constexpr (BITS == 32) {
    store<FULL, float>(static_cast<float*>(t.first[k]) + at, left, m);
    store<FULL, float>(static_cast<float*>(t.second[k]) + at, left, v);
  } else {
    unsigned top1 = 0, top2 = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top1 = max(top1, __float_as_uint(m[i]) & 0x7fffffffu), top2 = max(top2, __float_as_uint(v[i]) & 0x7fffffffu);
    const float s1 = factor_of(max_block(top1), (float)(1.0 / TOP_FIRST)), s2 = factor_of(max_block(top2), (float)(1.0 / TOP_SECOND));
    const float i1 = s1 == 0.f ? 0.f : 1.f / s1, i2 = s2 == 0.f ? 0.f : 1.f / s2;
    const unsigned long long counter = t.counter[k] + (unsigned long long)(at >> 2);
    const uint4 random[2] = {philox(counter, h.seed, (unsigned long long)f.step), philox(counter + 1, h.seed, (unsigned long long)f.step)};
    uint2 c1, c2;
    codes_of(m, v, i1, i2, random, c1, c2);
    store8<FULL>(static_cast<unsigned char*>(t.first[k]) + at, left, c1);
    store8<FULL>(static_cast<unsigned char*>(t.second[k]) + at, left, c2);
    if ((threadIdx.x & 31) == 0 && (FULL || left > 0)) t.scales[k][block] = make_float2(s1, s2);
  }
}

template <class T, int BITS, bool MASTER> __global__ __launch_bounds__(THREADS) void step_kernel(Tensors t, Step h) {
  constexpr int N = BITS == 8 ? 8 : 4, WAVE = 64 * N;
  const int k = tensor_of(t.part, t.count, blockIdx.x);
  Factors f;
  f.clip = 1.f;
  if (h.norm) {
    const float norm = *h.norm;
    if (!(norm < __builtin_inff())) return;                         // infinite, or no number: the step is left out
    f.clip = fminf(h.max_norm / norm, 1.f);
  }
  f.step = h.step_at ? *h.step_at : h.step;
  const float lr = h.lr_at ? *h.lr_at : h.lr;
  // 1 - b^t = -expm1(t log b): the product's rounding is one of t log b e^(t log b) relative to 1 - b^t, at most its own
  f.size = lr / -expm1f((float)f.step * h.log_b1), f.inverse2 = 1.f / -expm1f((float)f.step * h.log_b2), f.decay = lr * h.decay;
  const long n = t.n[k];
  const long start = (long)(blockIdx.x - t.part[k]) * PART + (threadIdx.x >> 6) * WAVE;
  for (int turn = 0; turn < PART / (THREADS * N); ++turn) {
    const long first = start + (long)turn * THREADS * N, at = first + (threadIdx.x & 63) * N;
    if (first + WAVE <= n) step_entries<T, BITS, MASTER, true>(t, k, h, f, at, N);          // all loads under way together
    else if (first < n) step_entries<T, BITS, MASTER, false>(t, k, h, f, at, n - at);
  }
}

// The moments that 8-bit codes stand for: p and master hold where they are written.
__global__ __launch_bounds__(THREADS) void states_kernel(Tensors t) {
  const int k = tensor_of(t.part, t.count, blockIdx.x);
  const long n = t.n[k];
  const long start = (long)(blockIdx.x - t.part[k]) * PART + threadIdx.x * 8;
#pragma unroll
  for (int turn = 0; turn < PART / (8 * THREADS); ++turn) {
    const long at = start + turn * 8 * THREADS, left = n - at;
    if (left <= 0) break;
    const float2 s = t.scales[k][at / BLOCK];
    float m[8], v[8];
    first_of(load8<false>(static_cast<unsigned char*>(t.first[k]) + at, left), s.x, m);
    second_of(load8<false>(static_cast<unsigned char*>(t.second[k]) + at, left), s.y, v);
    store<false, float>(static_cast<float*>(t.p[k]) + at, left, m);
    store<false, float>(t.master[k] + at, left, v);
  }
}

// ---- the norm of a list ---------------------------------------------------------------------------------------------
// Squares are summed in 64 bits: the factor that gradients are clipped by does not depend on the order, but for ties of its one rounding, and no square
// overflows or vanishes.  A workgroup sums 32 KB of a tensor, eight loads of 16 bytes a lane under way, and a single one joins their sums.  Lists of more than the caches hold
// are streamed past them (210 MB: 41 us instead of 44); shorter ones are left there for the step, which reads them again (50 MB of gradients in bfloat16: streamed
// 14 us instead of 21, and the step 108 instead of 98).
struct Lists {
  const void* g[MOST_SUMS];
  long n[MOST_SUMS];
  unsigned part[MOST_SUMS + 1];
  unsigned char dtype[MOST_SUMS];
  int count;
};
static_assert(sizeof(Lists) + 16 <= 4096, "kernel arguments");
constexpr int LOADS = 8;
inline long sums_part(int dtype) { return (long)LOADS * THREADS * (dtype == S2CNN_F32 ? 4 : 8); }

template <class T> __device__ __forceinline__ double squares(const T* g, long n, bool stream) {
  typedef Chunk<T> C;
  uint4 raw[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const long at = ((long)i * THREADS + threadIdx.x) * C::N;
    raw[i] = at < n ? load_chunk<T>(g + at, (int)min(n - at, (long)C::N), stream) : make_uint4(0, 0, 0, 0);
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    float v[C::N];
    C::get(raw[i], v);
#pragma unroll
    for (int j = 0; j < C::N; ++j) sum = fma((double)v[j], (double)v[j], sum);
  }
  return sum;
}
// over a workgroup, in thread 0
template <int WAVES> __device__ __forceinline__ double sum_workgroup(double v) {
  __shared__ double waves[WAVES];
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < WAVES; ++i) v += waves[i];
  return v;
}
__global__ __launch_bounds__(THREADS) void squares_kernel(Lists t, double* partial, bool stream) {
  const int k = tensor_of(t.part, t.count, blockIdx.x), dtype = t.dtype[k];
  const long per = (long)LOADS * THREADS * (dtype == S2CNN_F32 ? 4 : 8), at = (long)(blockIdx.x - t.part[k]) * per, n = t.n[k] - at;
  double sum;
  if (dtype == S2CNN_F32) sum = squares(static_cast<const float*>(t.g[k]) + at, n, stream);
  else if (dtype == S2CNN_BF16) sum = squares(static_cast<const __bf16*>(t.g[k]) + at, n, stream);
  else sum = squares(static_cast<const half_t*>(t.g[k]) + at, n, stream);
  sum = sum_workgroup<THREADS / 64>(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}
__global__ __launch_bounds__(1024) void norm_kernel(const double* partial, long parts, float* out) {
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  for (long i = threadIdx.x; i < parts; i += 4 * 1024)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * 1024 < parts) sum[j] += partial[i + j * 1024];
  const double all = sum_workgroup<16>((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (threadIdx.x == 0) *out = (float)sqrt(all);
}

// ---- launches -------------------------------------------------------------------------------------------------------
constexpr unsigned long MOST_PARTS = (1UL << 24) - 1;      // workgroups of a launch: fewer than 2^32 threads
constexpr long MOST_ENTRIES = (long)MOST_PARTS * PART;     // of a tensor, which no launch cuts

template <class T, int BITS> void launch(const Tensors& t, const Step& h, bool master, hipStream_t s) {
  const dim3 grid(t.part[t.count]), block(THREADS);
  if constexpr (sizeof(T) == 2)
    if (master) {
      hipLaunchKernelGGL((step_kernel<T, BITS, true>), grid, block, 0, s, t, h);
      return;
    }
  hipLaunchKernelGGL((step_kernel<T, BITS, false>), grid, block, 0, s, t, h);
}
void launch(const Tensors& t, const Step& h, int dtype, int bits, bool master, hipStream_t s) {
  if (dtype == S2CNN_F32) bits == 8 ? launch<float, 8>(t, h, false, s) : launch<float, 32>(t, h, false, s);
  else if (dtype == S2CNN_BF16) bits == 8 ? launch<__bf16, 8>(t, h, master, s) : launch<__bf16, 32>(t, h, master, s);
  else bits == 8 ? launch<half_t, 8>(t, h, master, s) : launch<half_t, 32>(t, h, master, s);
}

bool misaligned(const void* p, unsigned size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }
bool known(int dtype) { return dtype == S2CNN_F32 || dtype == S2CNN_BF16 || dtype == S2CNN_F16; }

// Whether an address that is written stands in the lists (NULL: none) twice; those of tensors without entries are left out.  -1: no memory to tell.
// On the host, 4 us for five lists of 158 tensors.
int twice(void* const* const (&lists)[5], const long* n, int count) {
  unsigned log = 4;
  while ((1UL << log) < 10UL * (unsigned long)count) ++log;
  void** const seen = static_cast<void**>(calloc(1UL << log, sizeof(void*)));
  if (!seen) return -1;
  int found = 0;
  for (void* const* list : lists)
    for (int i = 0; list && i < count && !found; ++i) {
      if (!n[i]) continue;
      unsigned long at = (reinterpret_cast<uintptr_t>(list[i]) * 0x9E3779B97F4A7C15UL) >> (64 - log);
      while (seen[at] && seen[at] != list[i]) at = (at + 1) & ((1UL << log) - 1);
      found = seen[at] != nullptr;
      seen[at] = list[i];
    }
  free(seen);
  return found;
}

// Lists of tensors, MOST of them and MOST_PARTS workgroups at a time, to `run`; those without entries are left out.
template <class F> void for_parts(int count, const long* n, const F& add, void (*launch_part)(const Tensors&, const void*), const void* with) {
  Tensors t = {};
  unsigned long long counter = 0;
  for (int i = 0; i < count; ++i) {
    if (!n[i]) continue;
    const unsigned long need = (unsigned long)(n[i] + PART - 1) / PART;
    if (t.count == MOST || (t.count && t.part[t.count] + need > MOST_PARTS)) {
      launch_part(t, with);
      t.count = 0;
    }
    const int k = t.count++;
    add(t, k, i);
    t.n[k] = n[i];
    t.counter[k] = counter;
    t.part[k + 1] = (k ? t.part[k] : 0) + (unsigned)need;
    t.part[0] = 0;
    counter += (unsigned long long)((n[i] + BLOCK - 1) / BLOCK) * (BLOCK / 4);
  }
  if (t.count) launch_part(t, with);
}

}  // namespace adamw
}  // namespace s2cnn

using namespace s2cnn;
using namespace s2cnn::adamw;

extern "C" int s2cnn_adamw_step(const s2cnn_adamw_t* a, void* stream) {
  clear_stale_error();
  if (!a || a->count < 0 || !known(a->dtype) || (a->bits != 8 && a->bits != 32) || (a->masters && a->dtype == S2CNN_F32)) return S2CNN_EINVAL;
  if (a->count && (!a->p || !a->g || !a->first || !a->second || !a->n || (a->bits == 8) != (a->scales != nullptr))) return S2CNN_EINVAL;
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 && a->eps >= 1e-30 && a->eps < 1e30)) return S2CNN_EINVAL;
  if (!(a->lr >= 0.0 && a->lr < 1e30 && a->weight_decay >= 0.0 && a->weight_decay < 1e30) || (!a->step_at && a->step < 1)) return S2CNN_EINVAL;
  if (a->norm && !(a->max_norm > 0.0 && a->max_norm < 1e38)) return S2CNN_EINVAL;
  if (misaligned(a->lr_at, 4) || misaligned(a->norm, 4) || misaligned(a->step_at, 8)) return S2CNN_EALIGN;
  if (!a->count) return S2CNN_OK;
  const unsigned size = a->dtype == S2CNN_F32 ? 4 : 2, state = a->bits == 8 ? 1 : 4;
  for (int i = 0; i < a->count; ++i) {
    if (a->n[i] < 0 || a->n[i] > MOST_ENTRIES) return S2CNN_EINVAL;
    if (!a->n[i]) continue;
    if (!a->p[i] || !a->g[i] || !a->first[i] || !a->second[i] || (a->scales && !a->scales[i]) || (a->masters && !a->masters[i])) return S2CNN_EINVAL;
    if (misaligned(a->p[i], size) || misaligned(a->g[i], size) || misaligned(a->first[i], state) || misaligned(a->second[i], state)) return S2CNN_EALIGN;
    if ((a->scales && misaligned(a->scales[i], 8)) || (a->masters && misaligned(a->masters[i], 4))) return S2CNN_EALIGN;
  }
  const int repeated = twice({a->p, a->first, a->second, a->scales, a->masters}, a->n, a->count);
  if (repeated) return repeated < 0 ? static_cast<int>(hipErrorOutOfMemory) : S2CNN_EINVAL;
  struct With {
    const s2cnn_adamw_t* a;
    Step h;
    hipStream_t s;
  } with = {a,
            {a->lr_at, a->norm, a->step_at, a->step, a->seed, (float)__builtin_log(a->beta1), (float)__builtin_log(a->beta2), (float)a->lr, (float)a->beta1, (float)(1.0 - a->beta1),
             (float)a->beta2, (float)(1.0 - a->beta2), (float)a->eps, (float)a->weight_decay, (float)a->max_norm},
            static_cast<hipStream_t>(stream)};
  for_parts(
      a->count, a->n,
      [&](Tensors& t, int k, int i) {
        t.p[k] = a->p[i], t.g[k] = a->g[i], t.first[k] = a->first[i], t.second[k] = a->second[i];
        t.scales[k] = a->scales ? static_cast<float2*>(a->scales[i]) : nullptr;
        t.master[k] = a->masters ? static_cast<float*>(a->masters[i]) : nullptr;
      },
      [](const Tensors& t, const void* w) {
        const With& of = *static_cast<const With*>(w);
        launch(t, of.h, of.a->dtype, of.a->bits, of.a->masters != nullptr, of.s);
      },
      &with);
  return launch_status();
}

extern "C" int s2cnn_adamw_states(const void* const* first, const void* const* second, const void* const* scales, void* const* first_out, void* const* second_out,
                                  const long* n, int count, void* stream) {
  clear_stale_error();
  if (count < 0 || (count && (!first || !second || !scales || !first_out || !second_out || !n))) return S2CNN_EINVAL;
  if (!count) return S2CNN_OK;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || n[i] > MOST_ENTRIES) return S2CNN_EINVAL;
    if (!n[i]) continue;
    if (!first[i] || !second[i] || !scales[i] || !first_out[i] || !second_out[i]) return S2CNN_EINVAL;
    if (misaligned(scales[i], 8) || misaligned(first_out[i], 4) || misaligned(second_out[i], 4)) return S2CNN_EALIGN;
  }
  for_parts(
      count, n,
      [&](Tensors& t, int k, int i) {
        t.first[k] = const_cast<void*>(first[i]), t.second[k] = const_cast<void*>(second[i]);
        t.scales[k] = static_cast<float2*>(const_cast<void*>(scales[i]));
        t.p[k] = first_out[i], t.master[k] = static_cast<float*>(second_out[i]);
      },
      [](const Tensors& t, const void* s) { hipLaunchKernelGGL(states_kernel, dim3(t.part[t.count]), dim3(THREADS), 0, static_cast<hipStream_t>(const_cast<void*>(s)), t); }, stream);
  return launch_status();
}

// Sums of the workgroups of the whole list, 0 for a list that is refused
static long parts_of(const long* n, const int* dtypes, int count) {
  long parts = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || n[i] > MOST_ENTRIES || !known(dtypes[i])) return -1;
    parts += (n[i] + sums_part(dtypes[i]) - 1) / sums_part(dtypes[i]);
  }
  return parts;
}

extern "C" size_t s2cnn_grad_norm_workspace(const long* n, const int* dtypes, int count) {
  const long parts = count < 0 || (count && (!n || !dtypes)) ? -1 : parts_of(n, dtypes, count);
  return parts < 0 ? 0 : (size_t)parts * sizeof(double);
}

extern "C" int s2cnn_grad_norm(const void* const* g, const long* n, const int* dtypes, int count, float* out, void* workspace, size_t workspace_bytes, void* stream_at) {
  clear_stale_error();
  if (count < 0 || !out || (count && (!g || !n || !dtypes))) return S2CNN_EINVAL;
  const long parts = parts_of(n, dtypes, count);
  if (parts < 0) return S2CNN_EINVAL;
  if (misaligned(out, 4)) return S2CNN_EALIGN;
  for (int i = 0; i < count; ++i) {
    if (n[i] && !g[i]) return S2CNN_EINVAL;
    if (n[i] && misaligned(g[i], dtypes[i] == S2CNN_F32 ? 4 : 2)) return S2CNN_EALIGN;
  }
  if (parts && (!workspace || workspace_bytes < (size_t)parts * sizeof(double) || !aligned16(workspace))) return S2CNN_EWORKSPACE;
  double* partial = static_cast<double*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream_at);
  long bytes = 0;
  for (int i = 0; i < count; ++i) bytes += n[i] * (dtypes[i] == S2CNN_F32 ? 4 : 2);
  const bool stream = (size_t)bytes >= STREAM_BYTES;
  Lists t = {};
  const auto run = [&] {
    if (t.count) hipLaunchKernelGGL(squares_kernel, dim3(t.part[t.count]), dim3(THREADS), 0, s, t, partial, stream);
    partial += t.part[t.count];
    t.count = 0;
  };
  for (int i = 0; i < count; ++i) {
    if (!n[i]) continue;
    const unsigned long need = (unsigned long)((n[i] + sums_part(dtypes[i]) - 1) / sums_part(dtypes[i]));
    if (t.count == MOST_SUMS || (t.count && t.part[t.count] + need > MOST_PARTS)) run();
    const int k = t.count++;
    t.g[k] = g[i], t.n[k] = n[i], t.dtype[k] = (unsigned char)dtypes[i];
    t.part[k + 1] = t.part[k] + (unsigned)need;
  }
  run();
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(1024), 0, s, static_cast<const double*>(workspace), parts, out);
  return launch_status();
}
