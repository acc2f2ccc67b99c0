// Attention, forward: out = softmax(scale q k^T + table[bucket] + key bias) v in one pass over the keys.
//
// A wave keeps 32 queries, a workgroup of W waves stages tiles of 32 keys and values for all of them.  Per tile: scores (rows:
// keys), running maximum and sum per query, probabilities as they are in registers into the product with the transposed
// values.  The columns run over all queries of the heads that share a key head, so that a single query of 8 heads reads its
// keys once; few columns and many keys: the keys are split over workgroups, and a second kernel joins their results.
//
// What bounds it, and what it measured.  float32, 4 signals, 8 heads, 4096 points, D = 64: 0.79 ms, 174 TFLOP/s of float32 products (1046 of
// bf16 ones; a library product of 8192^3 reaches 1238): matrix and vector instructions take 0.44 and 0.50 of a SIMD's time, and of the vector
// ones a third cut the staged rows into parts.  bfloat16, 16 signals, 8 heads on 2, 1024 points, those within a radian, D = 64: 77 us,
// bound by vector instructions (half of the SIMDs' time; matrix instructions 0.14) and the latency of a tile's steps.  One query a
// head, float32, 8 signals, 8 heads on 2, 32768 keys of 50: 60 us and 6 for the join, 3.5 TB/s of keys and values.  A kernel of one tile
// takes 8.5 us: the launch and one trip to memory after another.
#pragma once
#include "attention.h"

namespace s2cnn {
namespace attn {

// Workgroups of four waves a CU: four for the 16-bit types up to D = 64 (128 registers, none spilled), three for float32 at 64 (4 spilled; 868 us
// against 906 with two, 4 signals, 8 heads, 4096 points, on one card), two for the others; float32 at 32 takes 128 and gets four.  Three for the
// 16-bit types at 128 cost 14 registers, and 135 us against 101 (7 sets of 1009 queries and up to 2501 keys, 6 heads of 100); one for
// float32 at 128 leaves more registers, and takes 537 us against 397 (4 signals, 8 heads, 2048 points of 100).
template <class T, int D, int W> __global__ __launch_bounds__(64 * W, T::PARTS * D == 192 && W > 1 ? 3 : W == 1 || T::PARTS * D > 64 ? 2 : 4) void forward_kernel(Args p) {
  typedef Tile<T, D> Tl;
  constexpr int BUFS = buffers<T, D, W>(2), BUF = 2 * Tl::BYTES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* const lds_kb = reinterpret_cast<float*>(smem + BUFS * BUF);          // [RING][ROWS]
  float* const lds_table = lds_kb + RING * ROWS;
  const s2cnn_attention_t& a = p.a;

  const int work = work_of_block(p);
  if (work >= p.workgroups) return;
  const int split = work / p.tiles % p.splits, bh = work / p.tiles / p.splits, tile = tile_of(p, work, bh);
  const Group of = group_of(a, bh, a.kv_heads);
  const int b = of.b, hk = of.head, group = a.heads / a.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int columns = group * a.n_q, column0 = tile * 32 * W;
  const int column = column0 + (tid >> 6) * 32 + (lane & 31);
  const bool ok = column < columns, active = __any(ok);     // a wave without columns only stages
  const int c = ok ? column : columns - 1;
  const int head = hk * group + c / a.n_q, query = c % a.n_q;
  const int head0 = hk * group + column0 / a.n_q, heads = hk * group + min(columns - 1, column0 + 32 * W - 1) / a.n_q - head0 + 1;

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
  const float* const table = lds_table + (head - head0) * (a.n_buckets + 1);
  const bool measure = a.stats && tile == 0;                // this workgroup finds the largest |v| of its keys for the backward pass
  const float dead = ninf();

  Stage<T, D, 64 * W, BY_ROWS, BY_ENTRIES> stage;
  unsigned words[4] = {0, 0, 0, 0};
  if (key0 < end) {
    stage.prepare(k, v, tid);
    if (W > 1) stage.fetch(k, v, key0, tid);
    if (buckets) load_buckets(buckets, key0, end, half, words);
  }
  if (tid < 2 * ROWS) lds_kb[tid] = key_value(key0 < end ? load_key_bias(key_bias, key0 + tid, end) : 0.f, key0 + tid, end, p.inv_c, p.most);
  float bias_ahead = tid < ROWS && key0 < end ? load_key_bias(key_bias, key0 + 2 * ROWS + tid, end) : 0.f;
  if (buckets) stage_table<T>(lds_table, a.table, a.n_buckets, head0, heads, p.most * p.c, tid, 64 * W);
  Frag<T> qf[D / 16];
  load_column<T, D>(static_cast<const E*>(a.q) + b * a.q_stride[0] + head * a.q_stride[1] + query * a.q_stride[2], a.d, ok, half,
                    a.scale * LOG2E, qf);
  float largest = 0.f;
  const auto write = [&](int step) {
    unsigned char* const to = smem + step % BUFS * BUF;
    const float* const kb = lds_kb + step % RING * ROWS;
    const auto keep = [&](int r) { return kb[r] != dead; };
    if constexpr (W == 1) stage.fetch_and_write(k, v, key0 + step * ROWS, to, tid, keep);
    else stage.write(to, tid, keep);
    if (measure) largest = fmaxf(largest, stage.largest_second(tid));
  };
  if (BUFS == 2) {
    __syncthreads();
    if (key0 < end) write(0);
    if (key0 + ROWS < end) stage.fetch(k, v, key0 + ROWS, tid);
  }

  float m = ninf(), l = 0.f;
  Reference ref = reference<T>(0.f, p.c);
  v16f o[D / 32] = {};
  int step = 0;
  for (int key = key0; key < end; key += ROWS, ++step) {
    const bool more = key + ROWS < end;
    __syncthreads();
    if (BUFS == 1) {
      write(step);
      __syncthreads();
    }
    const unsigned char* const lds_k = smem + step % BUFS * BUF;
    const unsigned char* const lds_v = lds_k + Tl::BYTES;
    const float* const kb = lds_kb + step % RING * ROWS;

    if (tid < ROWS) lds_kb[(step + 2) % RING * ROWS + tid] = key_value(bias_ahead, key + 2 * ROWS + tid, end, p.inv_c, p.most);
    if (BUFS == 2 && more) write(step + 1);
    if (tid < ROWS) bias_ahead = load_key_bias(key_bias, key + 3 * ROWS + tid, end);
    if (W > 1 && key + BUFS * ROWS < end) stage.fetch(k, v, key + BUFS * ROWS, tid);
    unsigned now[4] = {0, 0, 0, 0};
    if (buckets) place_buckets(words, now);
    if (more && buckets) load_buckets(buckets, key + ROWS, end, half, words);

    if (active && (!buckets || !none_takes_part(now))) {
      v16f s;
      start_scores<T>(s, kb, half, buckets != nullptr, now, table, a.n_buckets, p.inv_c);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) mma<T>(Tl::by_rows(lds_k, i, lane), qf[i], s);
      float top = ninf();
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
      top = ceilf(fmaxf(T::PARTS == 3 ? half_max(top) : half_max(top) * p.c, m));
      if (__any(top != m)) {
        const float fade = top == m ? 1.f : fade_to<T>(top, m);       // a power of two
        l *= fade;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= fade;
        m = top;
        ref = reference<T>(top == ninf() ? 0.f : top, p.c);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = exp2_(off_reference<T>(s[i], ref));
        if constexpr (T::PARTS == 3) l += s[i];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const TwoParts<T> pf = cut_rows_in_two<T>(s, t);
        if constexpr (T::PARTS == 1) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned w[4] = {pf.part[i].part[0].x, pf.part[i].part[0].y, pf.part[i].part[0].z, pf.part[i].part[0].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) l = add_pair<T>(w[j], l);
          }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) mma<T>(Tl::by_entries(lds_v, i, t, lane), pf, o[i]);
      }
    }
  }

  const long row = ((long)b * a.heads + head) * a.n_q + query, rows = (long)a.batch * a.heads * a.n_q;
  if (measure) {
#pragma unroll
    for (int i = 32; i; i >>= 1) largest = fmaxf(largest, __shfl_xor(largest, i));
    __syncthreads();
    if (lane == 0) lds_kb[tid >> 6] = largest;
    __syncthreads();
    for (int i = 0; i < W; ++i) largest = fmaxf(largest, lds_kb[i]);
    if (tid == 0) a.stats[2 * rows + (b * a.kv_heads + hk) * p.splits + split] = largest;
  }
  l = half_sum(l);
  if (!ok) return;
  if (p.splits > 1) {
    float* const part = p.partial;
    store_partial<D>(part + (split * rows + row) * D, half, o);
    if (half == 0) reinterpret_cast<float2*>(part + p.splits * rows * D)[split * rows + row] = make_float2(m, l);
    return;
  }
  // a row without keys: zeros, and statistics by which every probability is zero
  const bool any = l != 0.f;
  const float inv = any ? 1.f / l : 0.f;
  store_column<T, D>(static_cast<E*>(a.out) + b * a.out_stride[0] + head * a.out_stride[1] + query * a.out_stride[2], a.d, half, o, inv);
  if (T::PARTS == 1 && a.out_f32) store_column<F32, D>(a.out_f32 + row * a.d, a.d, half, o, inv);
  if (half == 0 && a.stats) reinterpret_cast<float2*>(a.stats)[row] = any ? make_float2(m, inv) : make_float2(pinf(), 0.f);
}

// A workgroup joins the parts of one query, shared out to sixteen waves: lane s of a wave has the maximum and the sum of its part s (of 64
// at a time), and so its weight, 2^(its maximum - the maximum of all).
constexpr int JOIN_WAVES = 16;
template <class T, int D> __global__ __launch_bounds__(64 * JOIN_WAVES) void join_kernel(Args p) {
  __shared__ float lds_o[JOIN_WAVES][D], lds_l[JOIN_WAVES];
  const s2cnn_attention_t& a = p.a;
  const long rows = (long)a.batch * a.heads * a.n_q, row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* const part = p.partial;
  const float2* const ml = reinterpret_cast<const float2*>(part + p.splits * rows * D);
  constexpr int PER = (D + 63) / 64;
  float m = ninf();
  for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, ml[s * rows + row].x);
#pragma unroll
  for (int i = 32; i; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
  const float top = m == ninf() ? 0.f : m;
  const int per_wave = (p.splits + JOIN_WAVES - 1) / JOIN_WAVES, first = wave * per_wave, last = min(p.splits, first + per_wave);
  float l = 0.f, o[PER] = {};
  for (int s0 = first; s0 < last; s0 += 64) {
    float w = 0.f;
    if (s0 + lane < last) {
      const float2 x = ml[(s0 + lane) * rows + row];
      w = fade_to<T>(top, x.x);
      l = fmaf(x.y, w, l);
    }
    const int n = min(64, last - s0);
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 64 * i < D) o[i] = fmaf(part[((s0 + s) * rows + row) * D + lane + 64 * i], ws, o[i]);
    }
  }
#pragma unroll
  for (int i = 32; i; i >>= 1) l += __shfl_xor(l, i);
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < D) lds_o[wave][lane + 64 * i] = o[i];
  if (lane == 0) lds_l[wave] = l;
  __syncthreads();
  if (wave) return;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < JOIN_WAVES; ++w) l += lds_l[w];
  const bool any = l != 0.f;
  const float inv = any ? 1.f / l : 0.f;
  const int query = (int)(row % a.n_q), head = (int)(row / a.n_q % a.heads), b = (int)(row / a.n_q / a.heads);
  const long at = b * a.out_stride[0] + head * a.out_stride[1] + query * a.out_stride[2];
  typedef typename T::type E;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    if (e >= a.d) continue;
    const int slot = slot_of(e, a.d);
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN_WAVES; ++w) x += lds_o[w][slot];
    x *= inv;
    static_cast<E*>(a.out)[at + e] = (E)x;
    if (T::PARTS == 1 && a.out_f32) a.out_f32[row * a.d + e] = x;
  }
  if (lane == 0 && a.stats) reinterpret_cast<float2*>(a.stats)[row] = any ? make_float2(m, inv) : make_float2(pinf(), 0.f);
}

// The same for few parts, where what is read is many queries: D / 4 lanes a query, four entries a lane.  42378 queries of 128 entries in two
// parts: 11 us, by a workgroup a query 49; 64 queries in 96 parts: 6 us by a workgroup each, which here would be two wavefronts' chain of 96.
constexpr int FEW_PARTS = 8;
template <class T, int D> __global__ __launch_bounds__(256) void join_few_kernel(Args p) {
  const s2cnn_attention_t& a = p.a;
  constexpr int LANES = D / 4;
  const long rows = (long)a.batch * a.heads * a.n_q, row = ((long)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int q = threadIdx.x % LANES;
  if (row >= rows) return;
  const float* const part = p.partial;
  const float2* const ml = reinterpret_cast<const float2*>(part + p.splits * rows * D);
  float m = ninf();
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[s * rows + row].x);
  const float top = m == ninf() ? 0.f : m;
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.splits; ++s) {
    const float2 x = ml[s * rows + row];
    const float w = fade_to<T>(top, x.x);
    float y[4];
    read16(part + (s * rows + row) * D + 4 * q, y);
    l = fmaf(x.y, w, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(y[e], w, o[e]);
  }
  const bool any = l != 0.f;
  const float inv = any ? 1.f / l : 0.f;
  const int query = (int)(row % a.n_q), head = (int)(row / a.n_q % a.heads), b = (int)(row / a.n_q / a.heads);
  typedef typename T::type E;
  store_quad<T>(static_cast<E*>(a.out) + b * a.out_stride[0] + head * a.out_stride[1] + query * a.out_stride[2], q, a.d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (T::PARTS == 1 && a.out_f32) store_quad<F32>(a.out_f32 + row * a.d, q, a.d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (q == 0 && a.stats) reinterpret_cast<float2*>(a.stats)[row] = any ? make_float2(m, inv) : make_float2(pinf(), 0.f);
}

template <class T, int D> void forward_d(const Args& p, const Plans& plans, hipStream_t stream) {
  const s2cnn_attention_t& a = p.a;
  const Plan& f = plans.fwd;
  const int heads = min(a.heads / a.kv_heads, (32 * f.waves - 1) / a.n_q + 2);
  const size_t lds = (f.waves == 1 ? buffers<T, D, 1>(2) : buffers<T, D, 4>(2)) * 2 * Tile<T, D>::BYTES + (RING * ROWS + (a.buckets ? heads * (a.n_buckets + 1) : 0)) * sizeof(float);
  if constexpr (few_waves<T, D>) {
    if (f.waves == 1) launch(forward_kernel<T, D, 1>, p, 1, lds, stream);
  }
  if (f.waves != 1) launch(forward_kernel<T, D, 4>, p, 4, lds, stream);
  const long rows = (long)a.batch * a.heads * a.n_q;
  if (f.splits > FEW_PARTS) hipLaunchKernelGGL((join_kernel<T, D>), dim3((unsigned)rows), dim3(64 * JOIN_WAVES), 0, stream, p);
  else if (f.splits > 1) hipLaunchKernelGGL((join_few_kernel<T, D>), dim3((unsigned)((rows * (D / 4) + 255) / 256)), dim3(256), 0, stream, p);
}
template <class T> void forward(const Args& p, const Plans& plans, hipStream_t stream) {
  if (plans.D == 32) forward_d<T, 32>(p, plans, stream);
  else if (plans.D == 64) forward_d<T, 64>(p, plans, stream);
  else forward_d<T, 128>(p, plans, stream);
}

}  // namespace attn
}  // namespace s2cnn
