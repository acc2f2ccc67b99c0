// Attention, backward.  The probabilities are recomputed from the scores and the two statistics of each query:
//   p = 2^(x - m) / l,  ds = p (dp - delta),  dp = dout v^T,  delta = dout . out (per query),
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T dout,  dtable[head, n] = sum of ds over the pairs of bucket n.
// Where one key holds most of a query's softmax, dp - delta is a small difference: for the 16-bit types delta is formed from
// the output before its rounding (out_f32), and the probabilities are the rounded ones that made it.
// Two kernels, each with its results in registers to the end and no atomics between workgroups, so that results do not depend
// on the order of execution: one keeps queries and runs over keys (dq, dtable, and delta for the other), one keeps keys and
// runs over the queries of all heads that share them (dk, dv).  The price is that both form x and dp: seven products instead
// of five; storing ds would cost 2 n_q n_k floats of traffic per head, more time than two products.
#pragma once
#include "attention.h"

namespace s2cnn {
namespace attn {

// float16 has 30 binades: probabilities of a long row and gradients of a scaled loss do not fit it as they are.  Probabilities
// are held times 2^p, 2^p the power of two at n_k (at most 2^15), gradients of scores times 2^(p / 2) and the power of two that brings
// the largest |dout| to one.  Both are taken off the results.  All are one for the other types.
struct ScoreScale {
  float p = 1.f, ds = 1.f;                    // of probabilities; of ds on top of that
};
template <class T> __device__ __forceinline__ ScoreScale score_scale(int n_k, float largest) {
  ScoreScale s;
  if constexpr (T::HALF) {
    const int e = min(15, 31 - __clz(max(n_k, 1)));
    const int g = largest > 0.f ? max(-40, min(40, ilogbf(largest) + 1)) : 0;
    s.p = ldexpf(1.f, e);
    s.ds = ldexpf(1.f, -g - (e + 1) / 2);
  }
  return s;
}

// ---- dq, dtable, delta ----------------------------------------------------------------------------------------------
// Columns: queries of one head.  dtable: every lane adds to sums of its own in LDS, [wave][bucket][lane], one more bucket for
// pairs that have none; a wave's instructions run in order, so no sum depends on timing.
template <class T, int D, int W> __global__ __launch_bounds__(64 * W, 1) void grad_q_kernel(Args p) {
  typedef Tile<T, D> Tl;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* const lds_k = smem;
  unsigned char* const lds_kt = smem + Tl::BYTES;
  unsigned char* const lds_v = smem + 2 * Tl::BYTES;
  float* const lds_kb = reinterpret_cast<float*>(smem + 3 * Tl::BYTES);       // [2][ROWS]
  float* const lds_table = lds_kb + 2 * ROWS;                                 // [MAX_BUCKETS + 4]
  float* const lds_sums = lds_table + MAX_BUCKETS + 4;
  const s2cnn_attention_t& a = p.a;

  const int work = work_of_block(p.workgroups);
  if (work >= p.workgroups) return;
  const int tile = work % p.tiles, split = work / p.tiles % p.splits, bh = work / p.tiles / p.splits;
  const int b = bh / a.heads, head = bh % a.heads, hk = head / (a.heads / a.kv_heads);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = tid >> 6;
  const int query_ = tile * 32 * W + wave * 32 + (lane & 31);
  const bool ok = query_ < a.n_q;
  const int query = ok ? query_ : a.n_q - 1;
  const long row = ((long)b * a.heads + head) * a.n_q + query;

  int end = a.n_k;
  if (a.lengths) end = max(0, min(end, a.lengths[b]));
  const int chunk = ((a.n_k + ROWS - 1) / ROWS + p.splits - 1) / p.splits * ROWS;
  const int key0 = split * chunk;
  end = min(end, key0 + chunk);

  typedef typename T::type E;
  const Vectors<T> k{static_cast<const E*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[1], a.k_stride[2], a.n_k, a.d, (p.wide & WIDE_K) != 0};
  const Vectors<T> v{static_cast<const E*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[1], a.v_stride[2], a.n_k, a.d, (p.wide & WIDE_V) != 0};
  const float* const key_bias = a.key_bias ? a.key_bias + b * a.key_bias_stride : nullptr;
  const signed char* const buckets = a.buckets ? a.buckets + b * a.bucket_stride[0] + query * a.bucket_stride[1] : nullptr;
  float* const sums = lds_sums + (wave * (a.n_buckets + 1)) * 64 + lane;
  const bool table_grad = a.gtable != nullptr;

  Stage<T, D, 64 * W> stage;
  unsigned words[4] = {0, 0, 0, 0};
  if (key0 < end) {
    stage.fetch(k, v, key0, tid);
    if (buckets) load_buckets(buckets, key0, end, half, words);
  }
  if (tid < ROWS) lds_kb[tid] = key_value(key_bias, key0 + tid, end);
  if (buckets) stage_table<T>(lds_table, a.table, a.n_buckets, head, 1, tid, 64 * W);
  if (table_grad)
    for (int n = 0; n <= a.n_buckets; ++n) sums[n * 64] = 0.f;

  Frag<T> qf[D / 16], gf[D / 16];
  const E* const g_row = static_cast<const E*>(a.gout) + b * a.gout_stride[0] + head * a.gout_stride[1] + query * a.gout_stride[2];
  const float* const o_row = T::PARTS == 3 ? static_cast<const float*>(a.out) + b * a.out_stride[0] + head * a.out_stride[1] + query * a.out_stride[2] : a.out_f32 + row * a.d;
  const bool wide_g = (p.wide & WIDE_GOUT) != 0;
  const bool wide_o = T::PARTS == 3 ? (p.wide & WIDE_OUT) != 0 : a.d % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out_f32) & 15) == 0;
  const float2 stats = reinterpret_cast<const float2*>(a.stats)[row];
  const float m = ok ? stats.x : pinf(), inv_l = ok ? stats.y : 0.f;
  const bool live = inv_l != 0.f;                          // a row without keys takes no part, whatever its gradient holds
  load_column<T, D>(static_cast<const E*>(a.q) + b * a.q_stride[0] + head * a.q_stride[1] + query * a.q_stride[2], a.d, (p.wide & WIDE_Q) != 0, live, half, qf);
  load_column<T, D>(g_row, a.d, wide_g, live, half, gf);
  float delta = 0.f, largest = 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const int quad = 4 * (i / 2) + 2 * half + i % 2;
    float g4[4], o4[4];
    quad_values<T>(load_quad<T>(g_row, quad, a.d, wide_g), g4);
    quad_values<F32>(load_quad<F32>(o_row, quad, a.d, wide_o), o4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      delta = fmaf(g4[j], o4[j], delta);
      if constexpr (T::HALF) largest = fmaxf(largest, fabsf(g4[j]));
    }
  }
  delta = live ? half_sum(delta) : 0.f;
  if constexpr (T::HALF) largest = live ? half_max(largest) : 0.f;
  if (split == 0 && half == 0 && ok) {
    p.delta[row] = delta;
    if constexpr (T::HALF) p.delta[(long)a.batch * a.heads * a.n_q + row] = largest;
  }
  const ScoreScale sc = score_scale<T>(a.n_k, largest);
  const float rl = inv_l * sc.p, delta_s = delta * sc.ds;

  const float scale = a.scale * LOG2E;
  v16f dq[D / 32] = {};
  int slot = 0;
  for (int key = key0; key < end; key += ROWS, slot ^= 1) {
    const float* const kb = lds_kb + slot * ROWS;
    __syncthreads();
    stage.write(lds_k, lds_kt, lds_v, nullptr, tid, [&](int r) { return kb[r] != ninf(); });
    __syncthreads();
    unsigned now[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) now[g] = words[g];
    float kb_next = 0.f;
    const bool more = key + ROWS < end;
    if (more) {
      stage.fetch(k, v, key + ROWS, tid);
      if (buckets) load_buckets(buckets, key + ROWS, end, half, words);
      if (tid < ROWS) kb_next = key_value(key_bias, key + ROWS + tid, end);
    }

    v16f s = {}, dp = {};
    int n_of[16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      mma<T>(Tl::by_rows(lds_k, i, lane), qf[i], s);
      mma<T>(Tl::by_rows(lds_v, i, lane), gf[i], dp);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 kb4 = *reinterpret_cast<const float4*>(kb + 8 * g + 4 * half);
      const float kbs[4] = {kb4.x, kb4.y, kb4.z, kb4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * g + i;
        float x;
        int n = 0;
        if (buckets) {
          n = bucket_of(now[g], i, a.n_buckets);
          x = fmaf(s[r], scale, lds_table[n]) + kbs[i];
          if (n == a.n_buckets) x = ninf();
        } else {
          x = fmaf(s[r], scale, kbs[i]);
        }
        s[r] = exp2_(x - m);
        n_of[r] = n;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      float pr[2] = {s[r], s[r + 1]};
      round_pair<T>(pr[0], pr[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[r + i] = pr[i] * rl * (T::HALF ? fmaf(dp[r + i], sc.ds, -delta_s) : dp[r + i] - delta);
        if (table_grad) __hip_atomic_fetch_add(sums + n_of[r + i] * 64, s[r + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> f = cut_rows<T>(s, t);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) mma<T>(Tl::by_entries(lds_kt, i, t, lane), f, dq[i]);
    }
    if (more && tid < ROWS) lds_kb[(slot ^ 1) * ROWS + tid] = kb_next;
  }

  const float undo = T::HALF ? 1.f / (sc.p * sc.ds) : 1.f;
  if (table_grad) {
    if constexpr (T::HALF)
      for (int n = 0; n < a.n_buckets; ++n) sums[n * 64] *= undo;
    __syncthreads();
    float* const part = p.gtable_partial + ((long)bh * p.splits * p.tiles + split * p.tiles + tile) * a.n_buckets;
    for (int n = tid; n < a.n_buckets; n += 64 * W) {
      float t = 0.f;
      for (int w = 0; w < W; ++w)
        for (int i = 0; i < 64; ++i) t += lds_sums[(w * (a.n_buckets + 1) + n) * 64 + ((i + n) & 63)];   // lanes start at banks of their own
      part[n] = t;
    }
  }
  if (!ok) return;
  if (p.splits > 1) {
    const long rows = (long)a.batch * a.heads * a.n_q;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dq[i] *= a.scale * undo;
    store_partial<D>(p.partial + (split * rows + row) * D, half, dq);
    return;
  }
  store_column<T, D>(static_cast<E*>(a.gq) + b * a.gq_stride[0] + head * a.gq_stride[1] + query * a.gq_stride[2], a.d, (p.wide & WIDE_GQ) != 0, half, dq, a.scale * undo);
}

// ---- dk, dv ---------------------------------------------------------------------------------------------------------
// Columns: keys of one key head.  Rows: the queries of its heads, tile by tile, head by head.
template <class T, int D, int W> __global__ __launch_bounds__(64 * W, 1) void grad_kv_kernel(Args p) {
  typedef Tile<T, D> Tl;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* const lds_q = smem;
  unsigned char* const lds_qt = smem + Tl::BYTES;
  unsigned char* const lds_g = smem + 2 * Tl::BYTES;
  unsigned char* const lds_gt = smem + 3 * Tl::BYTES;
  float* const lds_rows = reinterpret_cast<float*>(smem + 4 * Tl::BYTES);     // [2][3][ROWS]: m, 1 / l, delta
  float* const lds_table = lds_rows + 6 * ROWS;
  const s2cnn_attention_t& a = p.a;

  const int work = work_of_block(p.workgroups);
  if (work >= p.workgroups) return;
  const int tile = work % p.tiles, split = work / p.tiles % p.splits, bh = work / p.tiles / p.splits;
  const int b = bh / a.kv_heads, hk = bh % a.kv_heads, group = a.heads / a.kv_heads;
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
  const signed char* const buckets = a.buckets ? a.buckets + b * a.bucket_stride[0] + key : nullptr;
  const float kb = ok ? key_value(key_bias, key, end) : ninf();
  const bool live = kb != ninf();

  Frag<T> kf[D / 16], vf[D / 16];
  load_column<T, D>(static_cast<const E*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[1] + key * a.k_stride[2], a.d, (p.wide & WIDE_K) != 0, live, half, kf);
  load_column<T, D>(static_cast<const E*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[1] + key * a.v_stride[2], a.d, (p.wide & WIDE_V) != 0, live, half, vf);

  ScoreScale sc;
  if constexpr (T::HALF) {                                 // one for all heads and queries: they are summed
    float* const lds_max = lds_rows;
    const float* const largest = p.delta + (long)a.batch * a.heads * a.n_q + ((long)b * a.heads + hk * group) * a.n_q;
    float t = 0.f;
    for (long i = tid; i < (long)group * a.n_q; i += 64 * W) t = fmaxf(t, largest[i]);
#pragma unroll
    for (int s = 32; s; s >>= 1) t = fmaxf(t, __shfl_xor(t, s));
    if (lane == 0) lds_max[wave] = t;
    __syncthreads();
    for (int w = 0; w < W; ++w) t = fmaxf(t, lds_max[w]);
    __syncthreads();
    sc = score_scale<T>(a.n_k, t);
  }

  Stage<T, D, 64 * W> stage;
  const auto fetch = [&](int r) {
    const int head = hk * group + r / per_head;
    const Vectors<T> q{static_cast<const E*>(a.q) + b * a.q_stride[0] + head * a.q_stride[1], a.q_stride[2], a.n_q, a.d, (p.wide & WIDE_Q) != 0};
    const Vectors<T> g{static_cast<const E*>(a.gout) + b * a.gout_stride[0] + head * a.gout_stride[1], a.gout_stride[2], a.n_q, a.d, (p.wide & WIDE_GOUT) != 0};
    stage.fetch(q, g, r % per_head * ROWS, tid);
  };
  struct Row { float m, rl, delta; };
  const auto row_of = [&](int r) -> Row {                  // what thread tid < ROWS brings for row tid of tile r
    const int query = r % per_head * ROWS + tid;
    if (query >= a.n_q) return {pinf(), 0.f, 0.f};
    const long row = ((long)b * a.heads + hk * group + r / per_head) * a.n_q + query;
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    return {st.x, st.y * sc.p, p.delta[row] * sc.ds};
  };
  const auto put_row = [&](int slot, const Row& x) {
    float* const to = lds_rows + slot * 3 * ROWS + tid;
    to[0] = x.m, to[ROWS] = x.rl, to[2 * ROWS] = x.delta;
  };
  if (first < last) {
    fetch(first);
    if (tid < ROWS) put_row(0, row_of(first));
  }
  if (buckets) stage_table<T>(lds_table, a.table, a.n_buckets, hk * group, group, tid, 64 * W);

  const float scale = a.scale * LOG2E;
  v16f dk[D / 32] = {}, dv[D / 32] = {};
  int slot = 0;
  for (int r = first; r < last; ++r, slot ^= 1) {
    const float* const rows = lds_rows + slot * 3 * ROWS;
    __syncthreads();
    stage.write(lds_q, lds_qt, lds_g, lds_gt, tid, [&](int i) { return rows[ROWS + i] != 0.f; });
    __syncthreads();
    const int query0 = r % per_head * ROWS;
    unsigned n_of[16];
    if (buckets) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        n_of[i] = (unsigned char)buckets[min(query0 + 8 * (i / 4) + 4 * half + i % 4, a.n_q - 1) * a.bucket_stride[1]];
    }
    Row next = {};
    const bool more = r + 1 < last;
    if (more) {
      fetch(r + 1);
      if (tid < ROWS) next = row_of(r + 1);
    }
    const float* const table = lds_table + r / per_head * (a.n_buckets + 1);

    v16f s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      mma<T>(Tl::by_rows(lds_q, i, lane), kf[i], s);
      mma<T>(Tl::by_rows(lds_g, i, lane), vf[i], dp);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 m4 = *reinterpret_cast<const float4*>(rows + 8 * g + 4 * half), l4 = *reinterpret_cast<const float4*>(rows + ROWS + 8 * g + 4 * half),
                   d4 = *reinterpret_cast<const float4*>(rows + 2 * ROWS + 8 * g + 4 * half);
      const float ms[4] = {m4.x, m4.y, m4.z, m4.w}, ls[4] = {l4.x, l4.y, l4.z, l4.w}, ds[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * g + i;
        float x;
        if (buckets) {
          const int n = min((int)n_of[j], a.n_buckets);
          x = fmaf(s[j], scale, table[n]) + kb;
          if (n == a.n_buckets) x = ninf();
        } else {
          x = fmaf(s[j], scale, kb);
        }
        s[j] = exp2_(x - ms[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float pr[2] = {s[4 * g + i], s[4 * g + i + 1]};
        round_pair<T>(pr[0], pr[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 4 * g + i + e;
          s[j] = pr[e] * ls[i + e];
          dp[j] = s[j] * (T::HALF ? fmaf(dp[j], sc.ds, -ds[i + e]) : dp[j] - ds[i + e]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag<T> pf = cut_rows<T>(s, t), df = cut_rows<T>(dp, t);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        mma<T>(Tl::by_entries(lds_gt, i, t, lane), pf, dv[i]);
        mma<T>(Tl::by_entries(lds_qt, i, t, lane), df, dk[i]);
      }
    }
    if (more && tid < ROWS) put_row(slot ^ 1, next);
  }

  if (!ok) return;
  const float fk = T::HALF ? a.scale / (sc.p * sc.ds) : a.scale, fv = T::HALF ? 1.f / sc.p : 1.f;
  if (p.splits > 1) {
    const long columns = (long)a.batch * a.kv_heads * a.n_k;
    float* const part = p.partial;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dk[i] *= fk, dv[i] *= fv;
    store_partial<D>(part + (split * columns + column) * D, half, dk);
    store_partial<D>(part + ((p.splits + split) * columns + column) * D, half, dv);
    return;
  }
  store_column<T, D>(static_cast<E*>(a.gk) + b * a.gk_stride[0] + hk * a.gk_stride[1] + key * a.gk_stride[2], a.d, (p.wide & WIDE_GK) != 0, half, dk, fk);
  store_column<T, D>(static_cast<E*>(a.gv) + b * a.gv_stride[0] + hk * a.gv_stride[1] + key * a.gv_stride[2], a.d, (p.wide & WIDE_GV) != 0, half, dv, fv);
}

// ---- sums of partial results, in a fixed order ----------------------------------------------------------------------
// Vectors: one wave each; [splits][vectors][D] -> the tensor.
template <class T, int D> __global__ __launch_bounds__(256) void sum_vectors_kernel(const float* part, int splits, typename T::type* to, long s0, long s1, long s2,
                                                                                   int heads, int n, int d, long vectors) {
  const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= vectors) return;
  typename T::type* const out = to + i / n / heads * s0 + i / n % heads * s1 + i % n * s2;
  for (int e = threadIdx.x & 63; e < d; e += 64) {
    float t = 0.f;
    for (int s = 0; s < splits; ++s) t += part[(s * vectors + i) * D + e];
    out[e] = (typename T::type)t;
  }
}
// dtable: one wave per (head, bucket); partials [batch][heads][per][n_buckets]
template <class T> __global__ __launch_bounds__(64) void sum_table_kernel(const float* part, int batch, int heads, int per, int n_buckets, typename T::type* out) {
  const int head = blockIdx.x / n_buckets, n = blockIdx.x % n_buckets;
  float t = 0.f;
  for (long k = threadIdx.x; k < (long)batch * per; k += 64) t += part[((k / per * heads + head) * per + k % per) * n_buckets + n];
#pragma unroll
  for (int s = 32; s; s >>= 1) t += __shfl_xor(t, s);
  if (threadIdx.x == 0) out[blockIdx.x] = (typename T::type)t;
}

template <class T> void sum_vectors(const float* part, int splits, int D, void* to, const long* stride, int batch, int heads, int n, int d, hipStream_t stream) {
  const long vectors = (long)batch * heads * n;
  const auto kernel = D == 32 ? sum_vectors_kernel<T, 32> : D == 64 ? sum_vectors_kernel<T, 64> : sum_vectors_kernel<T, 128>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((vectors + 3) / 4)), dim3(256), 0, stream, part, splits, static_cast<typename T::type*>(to), stride[0], stride[1],
                     stride[2], heads, n, d, vectors);
}

template <class T, int D> void backward_d(Args& p, const Plans& plans, float* partial_q, float* partial_kv, hipStream_t stream) {
  const s2cnn_attention_t& a = p.a;
  const auto use = [&](const Plan& f, float* partial) {
    p.splits = f.splits, p.tiles = f.tiles, p.workgroups = (int)f.workgroups, p.partial = partial;
  };
  use(plans.grad_q, partial_q);
  const int waves_q = plans.grad_q.waves;
  const size_t lds_q = 3 * Tile<T, D>::BYTES + (2 * ROWS + MAX_BUCKETS + 4 + (a.gtable ? waves_q * (a.n_buckets + 1) * 64 : 0)) * sizeof(float);
  if (waves_q == 1) launch(grad_q_kernel<T, D, 1>, p, 1, lds_q, stream);
  else launch(grad_q_kernel<T, D, 4>, p, 4, lds_q, stream);
  if (plans.grad_q.splits > 1) sum_vectors<T>(partial_q, plans.grad_q.splits, D, a.gq, a.gq_stride, a.batch, a.heads, a.n_q, a.d, stream);
  if (a.gtable)
    hipLaunchKernelGGL(sum_table_kernel<T>, dim3((unsigned)(a.heads * a.n_buckets)), dim3(64), 0, stream, p.gtable_partial, a.batch, a.heads,
                       plans.grad_q.splits * plans.grad_q.tiles, a.n_buckets, static_cast<typename T::type*>(a.gtable));
  if (!a.gk) return;
  use(plans.grad_kv, partial_kv);
  const size_t lds_kv = 4 * Tile<T, D>::BYTES + (6 * ROWS + (a.buckets ? a.heads / a.kv_heads * (a.n_buckets + 1) : 0)) * sizeof(float);
  if (plans.grad_kv.waves == 1) launch(grad_kv_kernel<T, D, 1>, p, 1, lds_kv, stream);
  else launch(grad_kv_kernel<T, D, 4>, p, 4, lds_kv, stream);
  if (plans.grad_kv.splits > 1) {
    const long columns = (long)a.batch * a.kv_heads * a.n_k;
    sum_vectors<T>(partial_kv, plans.grad_kv.splits, D, a.gk, a.gk_stride, a.batch, a.kv_heads, a.n_k, a.d, stream);
    sum_vectors<T>(partial_kv + plans.grad_kv.splits * columns * D, plans.grad_kv.splits, D, a.gv, a.gv_stride, a.batch, a.kv_heads, a.n_k, a.d, stream);
  }
}
template <class T> void backward(Args p, const Plans& plans, float* partial_q, float* partial_kv, hipStream_t stream) {
  if (plans.D == 32) backward_d<T, 32>(p, plans, partial_q, partial_kv, stream);
  else if (plans.D == 64) backward_d<T, 64>(p, plans, partial_q, partial_kv, stream);
  else backward_d<T, 128>(p, plans, partial_q, partial_kv, stream);
}

}  // namespace attn
}  // namespace s2cnn
