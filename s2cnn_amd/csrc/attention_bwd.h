// Attention, backward.  The probabilities are recomputed from the scores and the two statistics of each query:
//   p = 2^(x - m) / l (m, l: largest score, sum),  ds = p (dp - delta),  dp = dout v^T,  delta = dout . out (per query),
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T dout,  dtable[head, n] = sum of ds over the pairs of bucket n.
// Where one key holds most of a query's softmax, dp - delta is a small difference: for the 16-bit types delta is formed from
// the output before its rounding (out_f32).
// Two kernels, each with its results in registers to the end and no atomics between workgroups, so that results do not depend
// on the order of execution: one keeps queries and runs over keys (dq, dtable, and delta for the other), one keeps keys and
// runs over the queries of all heads that share them (dk, dv).  The price is that both form x and dp: seven products instead
// of five; storing ds would cost 2 n_q n_k floats of traffic per head, more time than two products.
//
// What bounds them, and what they measured.  float32, 4 signals, 8 heads, 4096 points, D = 64: dq 1.17 ms (176 TFLOP/s of float32 products),
// dk and dv 1.42 ms (193): matrix and vector instructions together take nine tenths of a SIMD's time, and a third of a tile's step goes into
// staging its rows.  bfloat16, 16 signals, 8 heads on 2, 1024 points, those within a radian: 125 and 132 us, vector instructions 0.40 and 0.38 of
// the time, matrix ones 0.11 and 0.16, the rest the latency of a tile's steps with two or three waves a SIMD.  float32, 32 signals, 5 heads,
// 400 points of 20 entries: 62 and 72 us.
#pragma once
#include "attention.h"

namespace s2cnn {
namespace attn {

// float16 has 30 binades: probabilities of a long row and gradients of a scaled loss do not fit it as they are.  Probabilities
// are held times 2^p, 2^p the power of two at n_k (at most 2^15), gradients of scores times 2^(p / 2) and the power of two that brings
// the largest |dout| to one.  Where values are large that is too much: |ds| = P |dp - delta| is at most a half of M = sum_d |dout_d| max |v|,
// and the power is lowered to where M stays below 2^16, ds below 2^15 (float16 ends at 65504; its second part then still reaches 2^-39 of
// that).  Both powers are taken off the results.  All are one for the other types.
struct ScoreScale {
  float p = 1.f, ds = 1.f;                    // of probabilities; of ds on top of that
};
constexpr int ANY_DS = 1000;                  // the exponent of a query without a gradient
__device__ __forceinline__ int p_exponent(int n_k) { return min(15, 31 - __clz(max(n_k, 1))); }
// the exponent of a query's ScoreScale::ds; bound: its M.  Of several queries: the least one
__device__ __forceinline__ int ds_exponent(int n_k, float largest, float bound) {
  if (!(largest > 0.f)) return ANY_DS;
  const int e = p_exponent(n_k), ordinary = -max(-40, min(40, ilogbf(largest) + 1)) - (e + 1) / 2;
  return bound > 0.f && bound < pinf() ? min(ordinary, 15 - e - ilogbf(bound)) : ordinary;
}
template <class T> __device__ __forceinline__ ScoreScale score_scale(int n_k, int exponent) {
  ScoreScale s;
  if constexpr (T::HALF) {
    s.p = ldexpf(1.f, p_exponent(n_k));
    s.ds = ldexpf(1.f, exponent == ANY_DS ? 0 : exponent);
  }
  return s;
}

// The largest |v| that the forward pass saw of a signal's key head: that of its parts.
__device__ __forceinline__ float largest_value(const float* of_parts, int parts) {
  float t = 0.f;
  for (int i = threadIdx.x & 63; i < parts; i += 64) t = fmaxf(t, of_parts[i]);
#pragma unroll
  for (int s = 32; s; s >>= 1) t = fmaxf(t, __shfl_xor(t, s));
  return t;
}

// ---- dq, dtable, delta ----------------------------------------------------------------------------------------------
// Sums of the table's gradient.  LDS adds floats at one lane per three clocks (190 clocks a wave instruction, measured) and
// integers at full rate (7 clocks, 64 bits), and integers give the same sum in any order: a value goes in as a 64-bit integer
// in units of a power of two that the workgroup knows beforehand.  |ds| <= 2 max(sum_d |dout_d|) max |v|, both maxima over what the
// workgroup sees, and a query's |ds| add up to no more than that: 2^50 units for twice the bound leaves room for the queries of a
// workgroup, and a unit is 2^-49 of the bound, 2^-28 of a typical ds in a row of 10^6 keys.
// 32 copies, one per lane of a half and shared by waves, keep lanes from the same address.  Sums of a workgroup are added in 64 bits to the
// end: entries of the table's gradient are small differences of large sums.
struct TableSums {
  static constexpr int COPIES = 32;
  static constexpr double MAGIC = 6755399441055744.0;        // 1.5 * 2^52: adding it rounds to an integer, which its low bits hold
  static __host__ __device__ int words(int n_buckets) { return (n_buckets + 1) * COPIES; }       // one more for excluded pairs
};

// Workgroups of four waves a CU: three at D = 32 and for the 16-bit types at 64, two for the others up to float32 at 64, all without spills but
// float32 at 32 (2 registers; 69 us against 90 with two, 32 signals, 5 heads, 400 points: 640 workgroups at once instead of in two rounds).
// Of one wave: so that two fit a SIMD (135 us against 252 with one, one query a head over 13824 keys of 106, 8 signals, 8 heads, float16).
template <class T, int D, int W> __global__ __launch_bounds__(64 * W, T::PARTS * D > 192 ? 1 : W > 1 && (D == 32 || T::PARTS * D == 64) ? 3 : 2) void grad_q_kernel(Args p) {
  typedef Tile<T, D> Tl;
  constexpr int BUFS = buffers<T, D, W>(3), BUF = 3 * Tl::BYTES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* const lds_kb = reinterpret_cast<float*>(smem + BUFS * BUF);          // [RING][ROWS]
  float* const lds_table = lds_kb + RING * ROWS;                              // [MAX_BUCKETS + 4]
  unsigned long long* const lds_sums = reinterpret_cast<unsigned long long*>(lds_table + MAX_BUCKETS + 4);
  const s2cnn_attention_t& a = p.a;

  const int work = work_of_block(p);
  if (work >= p.workgroups) return;
  const int split = work / p.tiles % p.splits, bh = work / p.tiles / p.splits, tile = tile_of(p, work, bh);
  const Group of = group_of(a, bh, a.heads);
  const int b = of.b, head = of.head, hk = head / (a.heads / a.kv_heads);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6;
  const int query_ = tile * 32 * W + wave * 32 + (lane & 31);
  const bool ok = query_ < a.n_q;
  const int query = ok ? query_ : a.n_q - 1;
  const long row = ((long)b * a.heads + head) * a.n_q + query, rows = (long)a.batch * a.heads * a.n_q;

  int end = a.n_k;
  if (a.lengths) end = max(0, min(end, a.lengths[b]));
  const int chunk = ((end + ROWS - 1) / ROWS + p.splits - 1) / p.splits * ROWS;      // parts of the keys that the signal has
  const int key0 = split * chunk;
  end = min(end, key0 + chunk);

  typedef typename T::type E;
  const Vectors<T> k{static_cast<const E*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[1], a.k_stride[2], a.n_k, a.d};
  const Vectors<T> v{static_cast<const E*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[1], a.v_stride[2], a.n_k, a.d};
  const float* const key_bias = a.key_bias ? a.key_bias + b * a.key_bias_stride : nullptr;
  const signed char* const buckets = a.buckets ? a.buckets + b * a.bucket_stride[0] + query * a.bucket_stride[1] : nullptr;
  unsigned long long* const sums = lds_sums + lane % TableSums::COPIES;
  const bool table_grad = a.gtable != nullptr;
  const float dead = ninf();

  Stage<T, D, 64 * W, BOTH, BY_ROWS> stage;
  unsigned words[4] = {0, 0, 0, 0};
  if (key0 < end) {
    stage.prepare(k, v, tid);
    if (W > 1) stage.fetch(k, v, key0, tid);
    if (buckets) load_buckets(buckets, key0, end, half, words);
  }
  if (tid < 2 * ROWS) lds_kb[tid] = key_value(key0 < end ? load_key_bias(key_bias, key0 + tid, end) : 0.f, key0 + tid, end, p.inv_c, p.most);
  float bias_ahead = tid < ROWS && key0 < end ? load_key_bias(key_bias, key0 + 2 * ROWS + tid, end) : 0.f;
  if (buckets) stage_table<T>(lds_table, a.table, a.n_buckets, head, 1, p.most * p.c, tid, 64 * W);
  if (table_grad)
    for (int n = tid; n < TableSums::words(a.n_buckets); n += 64 * W) lds_sums[n] = 0;

  Frag<T> qf[D / 16], gf[D / 16];
  const E* const g_row = static_cast<const E*>(a.gout) + b * a.gout_stride[0] + head * a.gout_stride[1] + query * a.gout_stride[2];
  const float* const o_row = T::PARTS == 3 ? static_cast<const float*>(a.out) + b * a.out_stride[0] + head * a.out_stride[1] + query * a.out_stride[2] : a.out_f32 + row * a.d;
  const float2 stats = reinterpret_cast<const float2*>(a.stats)[row];
  const Reference ref = reference<T>(ok ? stats.x : pinf(), p.c);
  const float inv_l = ok ? stats.y : 0.f;
  const bool live = inv_l != 0.f, active = __any(live);    // a row without keys takes no part, whatever its gradient holds
  load_column<T, D>(static_cast<const E*>(a.q) + b * a.q_stride[0] + head * a.q_stride[1] + query * a.q_stride[2], a.d, live, half,
                    a.scale * LOG2E, qf);
  // The matrix cores round sums down, not to nearest: a bias of a fraction of a unit in dp's last place, lost in the noise everywhere but
  // in the table's gradient, where the bias of every pair adds up.  Queries of odd lanes form -dp, whose bias has the other sign.
  const float sign = T::PARTS == 3 && (lane & 1) ? -1.f : 1.f;
  load_column<T, D>(g_row, a.d, live, half, sign, gf);
  float delta = 0.f, largest = 0.f, total = 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const int quad = 4 * (i / 2) + 2 * half + i % 2;
    float g4[4], o4[4];
    quad_values<T>(load_quad<T>(g_row, quad, a.d), g4);
    quad_values<F32>(load_quad<F32>(o_row, quad, a.d), o4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      delta = fmaf(g4[j], o4[j], delta);
      total += fabsf(g4[j]);
      if constexpr (T::HALF) largest = fmaxf(largest, fabsf(g4[j]));
    }
  }
  delta = live ? half_sum(delta) : 0.f;
  total = live ? half_sum(total) : 0.f;
  if constexpr (T::HALF) largest = live ? half_max(largest) : 0.f;
  const float vmax = T::HALF || table_grad ? largest_value(a.stats + 2 * rows + (b * a.kv_heads + hk) * p.forward_splits, p.forward_splits) : 0.f;
  const int exponent = T::HALF ? ds_exponent(a.n_k, largest, total * vmax) : 0;
  if (split == 0 && half == 0 && ok) {
    p.delta[row] = delta;
    if constexpr (T::HALF) p.delta[rows + row] = (float)exponent;
  }
  const ScoreScale sc = score_scale<T>(a.n_k, exponent);
  const float rl = inv_l * sc.p * sc.ds * sign, delta_rl = delta * sign * rl;         // ds = p (dp - delta) / l, as p (dp rl - delta rl)
  const float undo = T::HALF ? 1.f / (sc.p * sc.ds) : 1.f;

  // the unit of the table's sums; NaN where the gradient or a value seen by some query is none or infinite: delta is too, then
  double unit = 0.0;
  if (table_grad) {
    double bound = fabsf(delta) < pinf() ? (double)total * vmax : (double)pinf();
#pragma unroll
    for (int i = 32; i; i >>= 1) bound = fmax(bound, __shfl_xor(bound, i));
    double* const at = reinterpret_cast<double*>(smem);
    if (lane == 0) at[wave] = bound;
    __syncthreads();
    for (int i = 0; i < W; ++i) bound = fmax(bound, at[i]);
    __syncthreads();
    unit = bound == 0.0 ? 1.0 : bound < (double)pinf() ? ldexp(1.0, 48 - ilogb(bound)) : (double)__builtin_nanf("");
  }
  const double to_units = unit * undo;
  const auto write = [&](int step) {
    unsigned char* const to = smem + step % BUFS * BUF;
    const float* const kb = lds_kb + step % RING * ROWS;
    const auto keep = [&](int r) { return kb[r] != dead; };
    if constexpr (W == 1) stage.fetch_and_write(k, v, key0 + step * ROWS, to, tid, keep);
    else stage.write(to, tid, keep);
  };
  if (BUFS == 2) {
    __syncthreads();
    if (key0 < end) write(0);
    if (key0 + ROWS < end) stage.fetch(k, v, key0 + ROWS, tid);
  }

  v16f dq[D / 32] = {};
  int step = 0;
  for (int key = key0; key < end; key += ROWS, ++step) {
    const bool more = key + ROWS < end;
    __syncthreads();
    if (BUFS == 1) {
      write(step);
      __syncthreads();
    }
    const unsigned char* const lds_k = smem + step % BUFS * BUF;
    const unsigned char* const lds_kt = lds_k + Tl::BYTES;
    const unsigned char* const lds_v = lds_k + 2 * Tl::BYTES;
    const float* const kb = lds_kb + step % RING * ROWS;

    if (tid < ROWS) lds_kb[(step + 2) % RING * ROWS + tid] = key_value(bias_ahead, key + 2 * ROWS + tid, end, p.inv_c, p.most);
    if (BUFS == 2 && more) write(step + 1);
    unsigned now[4] = {0, 0, 0, 0};
    if (buckets) place_buckets(words, now);
    if (tid < ROWS) bias_ahead = load_key_bias(key_bias, key + 3 * ROWS + tid, end);
    if (W > 1 && key + BUFS * ROWS < end) stage.fetch(k, v, key + BUFS * ROWS, tid);
    if (more && buckets) load_buckets(buckets, key + ROWS, end, half, words);

    if (active && (!buckets || !none_takes_part(now))) {
      v16f s, dp = {};
      start_scores<T>(s, kb, half, buckets != nullptr, now, lds_table, a.n_buckets, p.inv_c);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) mma<T>(Tl::by_rows(lds_k, i, lane), qf[i], s);

#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        if constexpr (T::PARTS == 3) mma_small<T>(Tl::by_rows(lds_v, i, lane), gf[i], dp);
        else mma<T>(Tl::by_rows(lds_v, i, lane), gf[i], dp);
      }
      if constexpr (T::PARTS == 3) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) dp = mfma<T>(Tl::first_by_rows(lds_v, i, lane), gf[i].part[0], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float pr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) pr[i] = exp2_(off_reference<T>(s[r + i], ref));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[r + i] = pr[i] * fmaf(dp[r + i], rl, -delta_rl);
          if (table_grad) {
            const double x = __builtin_fma((double)s[r + i], to_units, TableSums::MAGIC);
            const unsigned long long raw = __builtin_bit_cast(unsigned long long, x);
            const unsigned high = (unsigned)(raw >> 32) - (unsigned)(__builtin_bit_cast(unsigned long long, TableSums::MAGIC) >> 32);   // its low half is zero
            __hip_atomic_fetch_add(sums + bucket_of(now[r / 4], r % 4 + i, a.n_buckets) * TableSums::COPIES, (unsigned long long)high << 32 | (unsigned)raw, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          }
        }
      }

#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const TwoParts<T> f = cut_rows_in_two<T>(s, t);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) mma<T>(Tl::by_entries(lds_kt, i, t, lane), f, dq[i]);
      }
    }
  }

  if (table_grad) {
    __syncthreads();
    double* const part = p.gtable_partial + (((long)b * a.heads + head) * p.splits * p.tiles + split * p.tiles + tile) * a.n_buckets;
    for (int n = tid; n < a.n_buckets; n += 64 * W) {
      unsigned long long t = 0;
      for (int i = 0; i < TableSums::COPIES; ++i) t += lds_sums[n * TableSums::COPIES + ((i + n) % TableSums::COPIES)];   // lanes start at banks of their own
      part[n] = (double)(long long)t / unit;
    }
  }
  if (!ok) return;
  if (p.splits > 1) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dq[i] *= a.scale * undo;
    store_partial<D>(p.partial + (split * rows + row) * D, half, dq);
    return;
  }
  store_column<T, D>(static_cast<E*>(a.gq) + b * a.gq_stride[0] + head * a.gq_stride[1] + query * a.gq_stride[2], a.d, half, dq, a.scale * undo);
}

// dtable[head, n]: a wave adds the workgroups' partial sums, [batch][heads][per][n_buckets], `pair` = head n_buckets + n.  In workgroups of the
// kernel of dk and dv beyond its own: a launch less, 4 us of the host's time and 5 of the card's.
template <class T> __device__ __forceinline__ void sum_table(const s2cnn_attention_t& a, const double* part, int per, int pair) {
  if (pair >= a.heads * a.n_buckets) return;
  const int head = pair / a.n_buckets, n = pair % a.n_buckets;
  double t = 0.0;
  for (unsigned k = threadIdx.x & 63; k < (unsigned)(a.batch * per); k += 64)          // fewer than 2^30, as the workgroups
    t += part[((long)(k / (unsigned)per * a.heads + head) * per + k % (unsigned)per) * a.n_buckets + n];
#pragma unroll
  for (int s = 32; s; s >>= 1) t += __shfl_xor(t, s);
  if ((threadIdx.x & 63) == 0) static_cast<typename T::type*>(a.gtable)[pair] = (typename T::type)(float)t;
}
template <class T> __global__ __launch_bounds__(256) void sum_table_kernel(Args p) { sum_table<T>(p.a, p.gtable_partial, p.gtable_parts, blockIdx.x * 4 + (threadIdx.x >> 6)); }

// ---- dk, dv ---------------------------------------------------------------------------------------------------------
// Columns: keys of one key head.  Rows: the queries of its heads, tile by tile, head by head.
constexpr int BUCKET_LD = 9;
// One tile in LDS, not two, for float32 at D = 32: so three workgroups fit a CU (79 us against 92 with two, at the size above), although 22
// registers are spilled for it.  For the 16-bit types at 64 the third costs 38, and 189 us against 156; at 128 the second costs 36, and is
// worth it (322 us against 409, 4 signals, 8 heads, 2048 points of 100).
template <class T> constexpr int row_arrays = T::PARTS == 3 ? 3 : 4;      // numbers of a row in LDS
template <class T, int D, int W> constexpr int kv_buffers() { return T::PARTS * D == 96 ? 1 : buffers<T, D, W>(4); }

template <class T, int D, int W> __global__ __launch_bounds__(64 * W, T::PARTS * D > 192 || W == 1 ? 1 : D == 32 ? 3 : 2) void grad_kv_kernel(Args p) {
  typedef Tile<T, D> Tl;
  constexpr int BUFS = kv_buffers<T, D, W>(), BUF = 4 * Tl::BYTES, ARRAYS = row_arrays<T>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* const lds_rows = reinterpret_cast<float*>(smem + BUFS * BUF);        // [RING][ARRAYS][ROWS]: -reference, 1 / l, -delta, factor (16-bit types)
  unsigned* const lds_buckets = reinterpret_cast<unsigned*>(lds_rows + ARRAYS * RING * ROWS);      // [2][32 W keys][8 words of four queries, one unused]
  float* const lds_table = lds_rows + ARRAYS * RING * ROWS + 2 * 32 * W * BUCKET_LD;
  const s2cnn_attention_t& a = p.a;

  const int own = blocks_for(p.workgroups);
  if ((int)blockIdx.x >= own) return sum_table<T>(a, p.gtable_partial, p.gtable_parts, ((int)blockIdx.x - own) * W + (threadIdx.x >> 6));
  const int work = work_of_block(p);
  if (work >= p.workgroups) return;
  const int split = work / p.tiles % p.splits, bh = work / p.tiles / p.splits, tile = tile_of(p, work, bh);
  const Group of = group_of(a, bh, a.kv_heads);
  const int b = of.b, hk = of.head, group = a.heads / a.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6;
  const int key_ = tile * 32 * W + wave * 32 + (lane & 31);
  const bool ok = key_ < a.n_k;
  const int key = ok ? key_ : a.n_k - 1;
  const long column = ((long)b * a.kv_heads + hk) * a.n_k + key;

  int end = a.n_k;
  if (a.lengths) end = max(0, min(end, a.lengths[b]));
  // the rows: tiles of 32 queries of each head in turn
  const int per_head = (a.n_q + ROWS - 1) / ROWS, all = group * per_head;
  const int chunk = (all + p.splits - 1) / p.splits;
  const int first = split * chunk;
  const int last = tile * 32 * W < end ? min(all, first + chunk) : first;     // past the length: zeros

  typedef typename T::type E;
  const float* const key_bias = a.key_bias ? a.key_bias + b * a.key_bias_stride : nullptr;
  const signed char* const buckets = a.buckets ? a.buckets + b * a.bucket_stride[0] : nullptr;
  const float dead = ninf(), kb_c = ok ? key_value(load_key_bias(key_bias, key, a.n_k), key, end, p.inv_c, p.most) : dead;
  const bool live = kb_c != dead, active = __any(live);

  Frag<T> kf[D / 16], vf[D / 16];
  load_column<T, D>(static_cast<const E*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[1] + key * a.k_stride[2], a.d, live, half,
                    T::PARTS == 3 ? 1.f : a.scale, kf);
  load_column<T, D>(static_cast<const E*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[1] + key * a.v_stride[2], a.d, live, half, 1.f, vf);

  ScoreScale sc;
  if constexpr (T::HALF) {                                 // one for all heads and queries: they are summed
    float* const lds_min = lds_rows;
    const float* const exponents = p.delta + (long)a.batch * a.heads * a.n_q + ((long)b * a.heads + hk * group) * a.n_q;
    float t = ANY_DS;
    for (long i = tid; i < (long)group * a.n_q; i += 64 * W) t = fminf(t, exponents[i]);
#pragma unroll
    for (int s = 32; s; s >>= 1) t = fminf(t, __shfl_xor(t, s));
    if (lane == 0) lds_min[wave] = t;
    __syncthreads();
    for (int w = 0; w < W; ++w) t = fminf(t, lds_min[w]);
    __syncthreads();
    sc = score_scale<T>(a.n_k, (int)t);
  }

  Stage<T, D, 64 * W, BOTH, BOTH, T::PARTS == 3> stage;
  stage.factor = a.scale * LOG2E;
  struct Place {                                           // of a tile: its head of the group, its first query
    int head, query;
    __device__ __forceinline__ Place next(int n_q) const { return query + ROWS < n_q ? Place{head, query + ROWS} : Place{head + 1, 0}; }
  };
  const auto queries = [&](const Place& at, const void* base, const long (&stride)[3]) -> Vectors<T> {
    return {static_cast<const E*>(base) + b * stride[0] + (hk * group + at.head) * stride[1], stride[2], a.n_q, a.d};
  };
  const auto fetch = [&](const Place& at) { stage.fetch(queries(at, a.q, a.q_stride), queries(at, a.gout, a.gout_stride), at.query, tid); };
  // what thread tid < ROWS brings for row tid of tile r: the load, and what is made of it (as load_key_bias, key_value)
  struct Row { float2 stats; float delta; };
  const auto load_row = [&](const Place& at) -> Row {
    const long row = ((long)b * a.heads + hk * group + min(at.head, group - 1)) * a.n_q + min(at.query + tid, a.n_q - 1);
    return {reinterpret_cast<const float2*>(a.stats)[row], p.delta[row]};
  };
  const auto put_row = [&](int step, const Place& at, const Row& x) {
    float* const to = lds_rows + step % RING * ARRAYS * ROWS + tid;
    const bool none = at.head >= group || at.query + tid >= a.n_q;
    const Reference ref = reference<T>(x.stats.x, p.c);
    if constexpr (T::PARTS == 1) to[3 * ROWS] = ref.c;
    to[0] = none ? ninf() : -ref.at, to[ROWS] = none ? 0.f : x.stats.y * sc.p, to[2 * ROWS] = none ? 0.f : -x.delta;
  };
  const auto write = [&](int step, const Place& at) {
    unsigned char* const to = smem + step % BUFS * BUF;
    const float* const rows = lds_rows + step % RING * ARRAYS * ROWS;
    const auto keep = [&](int i) { return rows[ROWS + i] != 0.f; };
    if constexpr (W == 1) stage.fetch_and_write(queries(at, a.q, a.q_stride), queries(at, a.gout, a.gout_stride), at.query, to, tid, keep);
    else stage.write(to, tid, keep);
  };
  // The tile's buckets pass through LDS too: a thread fetches those of 4 queries and 4 keys, and writes them the other way round, a word
  // of four queries per key.
  unsigned bucket_words[4];
  const int block_query = 4 * (tid / (8 * W)), block_key = 4 * (tid % (8 * W));
  const unsigned bucket_stride = (unsigned)a.bucket_stride[1], bucket_offset = block_query * bucket_stride + block_key;
  const auto fetch_buckets = [&](const Place& place) {
    const int left = a.n_q - 1 - place.query, key0 = tile * 32 * W + block_key;
    const signed char* const at = buckets + (unsigned long long)(unsigned)place.query * bucket_stride + tile * 32 * W;
    if (left >= ROWS - 1 && (tile + 1) * 32 * W <= a.n_k) {                // for all threads alike
#pragma unroll
      for (int i = 0; i < 4; ++i) bucket_words[i] = load_word_at(at + i * bucket_stride, bucket_offset);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const signed char* const from = at + (unsigned)(min(block_query + i, left) * (int)a.bucket_stride[1] + block_key);
      if (key0 + 4 <= a.n_k) __builtin_memcpy(&bucket_words[i], from, 4);
      else {
        bucket_words[i] = 0;
        for (int e = 0; e < 4; ++e) bucket_words[i] |= (key0 + e < a.n_k ? (unsigned)(unsigned char)from[e] : 255u) << (8 * e);
      }
    }
  };
  const auto write_buckets = [&](int step) {
    unsigned* const to = lds_buckets + step % 2 * 32 * W * BUCKET_LD + block_key * BUCKET_LD + block_query / 4;
    const unsigned a0 = __builtin_amdgcn_perm(bucket_words[1], bucket_words[0], 0x05010400u), a1 = __builtin_amdgcn_perm(bucket_words[1], bucket_words[0], 0x07030602u);
    const unsigned b0 = __builtin_amdgcn_perm(bucket_words[3], bucket_words[2], 0x05010400u), b1 = __builtin_amdgcn_perm(bucket_words[3], bucket_words[2], 0x07030602u);
    to[0] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
    to[BUCKET_LD] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
    to[2 * BUCKET_LD] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
    to[3 * BUCKET_LD] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
  };
  Place here{first / per_head, first % per_head * ROWS}, next = here.next(a.n_q), after = next.next(a.n_q);     // of this step, the next, the one after
  Row ahead = {};
  if (first < last) {
    stage.prepare(queries(here, a.q, a.q_stride), queries(here, a.gout, a.gout_stride), tid);
    if (W > 1) fetch(here);
    if (buckets) fetch_buckets(here);
    if (tid < ROWS) put_row(0, here, load_row(here)), put_row(1, next, load_row(next)), ahead = load_row(after);
  }
  if (buckets) stage_table<T>(lds_table, a.table, a.n_buckets, hk * group, group, p.most * p.c, tid, 64 * W);
  if (BUFS == 2) {
    __syncthreads();
    if (first < last) write(0, here);
    if (first + 1 < last) fetch(next);
    if (buckets && first < last) write_buckets(0);
    if (buckets && first + 1 < last) fetch_buckets(next);
  }

  v16f dk[D / 32] = {}, dv[D / 32] = {};
  for (int r = first, step = 0; r < last; ++r, ++step) {
    const float* const rows = lds_rows + step % RING * ARRAYS * ROWS;
    const unsigned char* const lds_q = smem + step % BUFS * BUF;
    const unsigned char* const lds_qt = lds_q + Tl::BYTES;
    const unsigned char* const lds_g = lds_q + 2 * Tl::BYTES;
    const unsigned char* const lds_gt = lds_q + 3 * Tl::BYTES;
    __syncthreads();
    if (tid < ROWS) put_row(step + 2, after, ahead);
    if (BUFS == 1) {
      write(step, here);
      if (buckets) write_buckets(step);
      __syncthreads();
    } else if (r + 1 < last) {
      write(step + 1, next);
      if (buckets) write_buckets(step + 1);
    }
    const float* const table = lds_table + here.head * (a.n_buckets + 1);
    if (tid < ROWS) ahead = load_row(after.next(a.n_q));
    if (r + BUFS < last) {
      if (W > 1) fetch(BUFS == 1 ? next : after);
      if (buckets) fetch_buckets(BUFS == 1 ? next : after);
    }
    unsigned words[4] = {0, 0, 0, 0};
    if (buckets) {
      const unsigned* const from = lds_buckets + (step % 2 * 32 * W + wave * 32 + (lane & 31)) * BUCKET_LD + half;
#pragma unroll
      for (int g = 0; g < 4; ++g) words[g] = from[2 * g];
    }
    if (active && (!buckets || !none_takes_part(words))) {
      // the scores start from the biases, dp from -delta
      v16f s, dp;
      if (buckets) {
        float t[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) t[j] = table[bucket_of(words[j / 4], j % 4, a.n_buckets)];
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = T::PARTS == 3 ? kb_c + t[j] : fmaf(t[j], p.inv_c, kb_c);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = kb_c;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float start[4];
        read16(rows + 2 * ROWS + 8 * g + 4 * half, start);
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[4 * g + i] = start[i];
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) mma<T, true>(Tl::by_rows(lds_q, i, lane), kf[i], s);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float ms[4], cs[4] = {1.f, 1.f, 1.f, 1.f};
        read16(rows + 8 * g + 4 * half, ms);
        if constexpr (T::PARTS == 1) read16(rows + 3 * ROWS + 8 * g + 4 * half, cs);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * g + i] = exp2_(off_reference<T>(s[4 * g + i], Reference{-ms[i], cs[i]}));
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) mma<T>(Tl::by_rows(lds_g, i, lane), vf[i], dp);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float ls[4];
        read16(rows + ROWS + 8 * g + 4 * half, ls);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 4 * g + i;
          s[j] *= ls[i];
          dp[j] = s[j] * (T::HALF ? dp[j] * sc.ds : dp[j]);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const TwoParts<T> pf = cut_rows_in_two<T>(s, t), df = cut_rows_in_two<T>(dp, t);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          mma<T>(Tl::by_entries(lds_gt, i, t, lane), pf, dv[i]);
          mma<T>(Tl::by_entries(lds_qt, i, t, lane), df, dk[i]);
        }
      }
    }
    here = next, next = after, after = after.next(a.n_q);
  }

  if (!ok) return;
  const float fk = T::PARTS == 3 ? 1.f / LOG2E : T::HALF ? a.scale / (sc.p * sc.ds) : a.scale, fv = T::HALF ? 1.f / sc.p : 1.f;
  if (p.splits > 1) {
    const long columns = (long)a.batch * a.kv_heads * a.n_k;
    float* const part = p.partial;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dk[i] *= fk, dv[i] *= fv;
    store_partial<D>(part + (split * columns + column) * D, half, dk);
    store_partial<D>(part + ((p.splits + split) * columns + column) * D, half, dv);
    return;
  }
  store_column<T, D>(static_cast<E*>(a.gk) + b * a.gk_stride[0] + hk * a.gk_stride[1] + key * a.gk_stride[2], a.d, half, dk, fk);
  store_column<T, D>(static_cast<E*>(a.gv) + b * a.gv_stride[0] + hk * a.gv_stride[1] + key * a.gv_stride[2], a.d, half, dv, fv);
}

// ---- sums of partial results, in a fixed order ----------------------------------------------------------------------
// Vectors: D / 4 lanes each, a quad a lane; [tensor][splits][vectors][D] -> the tensors (dk and dv, or dq alone).
struct Sums {
  const float* part;
  void* to[2];
  long stride[2][3];
  int splits, heads, n, d;
  long vectors;
};
template <class T, int D> __global__ __launch_bounds__(256) void sum_vectors_kernel(Sums p) {
  constexpr int LANES = D / 4;
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int q = threadIdx.x % LANES, which = blockIdx.y;
  if (i >= p.vectors || 4 * q >= p.d) return;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.splits; ++s) {
    float x[4];
    read16(p.part + ((which * p.splits + s) * p.vectors + i) * D + 4 * q, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += x[e];
  }
  const long (&st)[3] = p.stride[which];
  store_quad<T>(static_cast<typename T::type*>(p.to[which]) + i / p.n / p.heads * st[0] + i / p.n % p.heads * st[1] + i % p.n * st[2], q, p.d, t[0], t[1], t[2], t[3]);
}
template <class T, int D> void sum_vectors(const float* part, int splits, int tensors, void* const (&to)[2], const long* s0, const long* s1, int batch, int heads, int n, int d,
                                           hipStream_t stream) {
  const Sums p{part, {to[0], to[1]}, {{s0[0], s0[1], s0[2]}, {s1[0], s1[1], s1[2]}}, splits, heads, n, d, (long)batch * heads * n};
  hipLaunchKernelGGL((sum_vectors_kernel<T, D>), dim3((unsigned)((p.vectors * (D / 4) + 255) / 256), (unsigned)tensors), dim3(256), 0, stream, p);
}

template <class T, int D> void backward_d(Args& p, const Plans& plans, float* partial_q, float* partial_kv, hipStream_t stream) {
  const s2cnn_attention_t& a = p.a;
  const auto use = [&](const Plan& f, float* partial) {
    p.splits = f.splits, p.tiles = f.tiles, p.workgroups = (int)f.workgroups, p.partial = partial;
  };
  use(plans.grad_q, partial_q);
  const int waves_q = plans.grad_q.waves;
  const size_t lds_q = (waves_q == 1 ? buffers<T, D, 1>(3) : buffers<T, D, 4>(3)) * 3 * Tile<T, D>::BYTES + (RING * ROWS + MAX_BUCKETS + 4) * sizeof(float) +
                       (a.gtable ? TableSums::words(a.n_buckets) * sizeof(unsigned long long) : 0);
  if constexpr (few_waves<T, D>) {
    if (waves_q == 1) launch(grad_q_kernel<T, D, 1>, p, 1, lds_q, stream);
  }
  if (waves_q != 1) launch(grad_q_kernel<T, D, 4>, p, 4, lds_q, stream);
  if (plans.grad_q.splits > 1) sum_vectors<T, D>(partial_q, plans.grad_q.splits, 1, {a.gq, nullptr}, a.gq_stride, a.gq_stride, a.batch, a.heads, a.n_q, a.d, stream);
  p.gtable_parts = plans.grad_q.splits * plans.grad_q.tiles;
  const int pairs = a.gtable ? a.heads * a.n_buckets : 0;
  if (!a.gk) {
    if (pairs) hipLaunchKernelGGL(sum_table_kernel<T>, dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, stream, p);
    return;
  }
  use(plans.grad_kv, partial_kv);
  const size_t lds_kv = (plans.grad_kv.waves == 1 ? kv_buffers<T, D, 1>() : kv_buffers<T, D, 4>()) * 4 * Tile<T, D>::BYTES + (row_arrays<T> * RING * ROWS + 2 * 32 * plans.grad_kv.waves * BUCKET_LD + (a.buckets ? a.heads / a.kv_heads * (a.n_buckets + 1) : 0)) * sizeof(float);
  if constexpr (few_waves<T, D>) {
    if (plans.grad_kv.waves == 1) launch(grad_kv_kernel<T, D, 1>, p, 1, lds_kv, stream, pairs);
  }
  if (plans.grad_kv.waves != 1) launch(grad_kv_kernel<T, D, 4>, p, 4, lds_kv, stream, (pairs + 3) / 4);
  if (plans.grad_kv.splits > 1)
    sum_vectors<T, D>(partial_kv, plans.grad_kv.splits, 2, {a.gk, a.gv}, a.gk_stride, a.gv_stride, a.batch, a.kv_heads, a.n_k, a.d, stream);
}
template <class T> void backward(Args p, const Plans& plans, float* partial_q, float* partial_kv, hipStream_t stream) {
  if (plans.D == 32) backward_d<T, 32>(p, plans, partial_q, partial_kv, stream);
  else if (plans.D == 64) backward_d<T, 64>(p, plans, partial_q, partial_kv, stream);
  else backward_d<T, 128>(p, plans, partial_q, partial_kv, stream);
}

}  // namespace attn
}  // namespace s2cnn
