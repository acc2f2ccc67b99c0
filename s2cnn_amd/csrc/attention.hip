// Entry points of the attention kernels: checks, the layout of the work, workspaces.
#include "attention.h"

namespace s2cnn {
namespace attn {
extern template void forward<F32>(const Args&, const Plans&, hipStream_t);
extern template void forward<BF16>(const Args&, const Plans&, hipStream_t);
extern template void forward<F16>(const Args&, const Plans&, hipStream_t);
extern template void backward<F32>(Args, const Plans&, float*, float*, hipStream_t);
extern template void backward<BF16>(Args, const Plans&, float*, float*, hipStream_t);
extern template void backward<F16>(Args, const Plans&, float*, float*, hipStream_t);

namespace {

constexpr int CUS = 256;

// Columns of one group of heads, groups, and tiles of the long axis.  A workgroup of one wave where one wave holds all columns.
// The long axis is cut where there are less than six workgroups of one wave, or two of four, for each compute unit, into parts of at
// least four tiles, or sixteen where every unit has a workgroup without: the parts are written and read again.  Six is what a unit's LDS
// holds at float32, D = 64: 61 us for one query a head over 32768 keys, 8 signals, 2 key heads of 50; with five 69, with seven 93.
Plan plan(long columns, long groups, long long_tiles, bool few) {
  Plan p;
  p.waves = few && columns <= 32 ? 1 : 4;
  p.tiles = columns < 1 ? 1 : (int)((columns + 32 * p.waves - 1) / (32 * p.waves));
  const long base = p.tiles * groups, want = p.waves == 1 ? 6 * CUS : 2 * CUS;
  const long splits = min((want + base - 1) / base, long_tiles / (base > CUS ? 16 : 4));
  p.splits = splits < 1 ? 1 : (int)splits;
  p.workgroups = base * p.splits;
  return p;
}

long tiles_of(long n) { return (n + ROWS - 1) / ROWS; }

Plans plans_of(const s2cnn_attention_t& a) {
  Plans p;
  p.D = a.d <= 32 ? 32 : a.d <= 64 ? 64 : 128;
  const long group = a.heads / a.kv_heads;
  const bool few = a.dtype != S2CNN_F32 || p.D <= 64;       // few_waves
  p.fwd = plan(group * a.n_q, (long)a.batch * a.kv_heads, tiles_of(a.n_k), few);
  p.grad_q = plan(a.n_q, (long)a.batch * a.heads, tiles_of(a.n_k), few);
  p.grad_kv = plan(a.n_k, (long)a.batch * a.kv_heads, group * tiles_of(a.n_q), few);
  return p;
}

long stats_floats(const s2cnn_attention_t& a, const Plans& p) { return 2L * a.batch * a.heads * a.n_q + (long)a.batch * a.kv_heads * p.fwd.splits; }

bool sizes_ok(const s2cnn_attention_t* a) {
  if (!a) return false;
  if (a->dtype != S2CNN_F32 && a->dtype != S2CNN_BF16 && a->dtype != S2CNN_F16) return false;
  if (a->batch < 1 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->n_q < 1 || a->n_k < 0 || a->d < 4 || a->d > 128) return false;
  const bool bias = a->buckets || a->table || a->n_buckets;
  if (bias && ((!a->buckets && a->n_k > 0) || !a->table || a->n_buckets < 1 || a->n_buckets > MAX_BUCKETS || a->heads / a->kv_heads > MAX_GROUP)) return false;
  if (a->buckets && (a->bucket_stride[1] < 0 || a->bucket_stride[1] >= S2CNN_ATTENTION_STRIDE_LIMIT)) return false;
  const long limit = 1L << 30;
  if ((long)a->heads / a->kv_heads * a->n_q > limit || a->n_k > limit || (long)a->batch * a->heads > limit) return false;
  for (const long* s : {a->q_stride, a->k_stride, a->v_stride, a->gout_stride})
    if (s[2] < 0 || s[2] >= S2CNN_ATTENTION_STRIDE_LIMIT) return false;
  const Plans p = plans_of(*a);
  return p.fwd.workgroups < limit && p.grad_q.workgroups < limit && p.grad_kv.workgroups < limit && (long)a->batch * a->heads * a->n_q < 4 * limit &&
         (long)a->batch * a->kv_heads * a->n_k < 4 * limit;
}

// Heads that share a key head, as one head of all their queries, where no bucket tells them apart and their vectors follow each other evenly:
// a tile of rows or columns holds more than one head's, and the keys are read once.  Gradients of 5 queries of 12 heads on 3 over 5832
// keys of 90, 31 signals, float32: a quarter of the tiles.  The statistics, [batch, heads, n_q], are the same array.
s2cnn_attention_t joined(const s2cnn_attention_t& a, bool gradients) {
  const int group = a.heads / a.kv_heads;
  if (group == 1 || a.buckets) return a;
  s2cnn_attention_t c = a;
  c.heads = a.kv_heads, c.n_q = group * a.n_q;
  for (long(*s)[3] : {&c.q_stride, &c.out_stride, &c.gout_stride, &c.gq_stride}) {
    if (!gradients && (s == &c.gout_stride || s == &c.gq_stride)) continue;
    long(&x)[3] = *s;
    if (a.n_q > 1 ? x[1] != a.n_q * x[2] : x[1] < 0 || x[1] >= S2CNN_ATTENTION_STRIDE_LIMIT) return a;
    if (a.n_q == 1) x[2] = x[1];
    x[1] *= group;
  }
  return c;
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

size_t forward_bytes(const s2cnn_attention_t& a, const Plans& p) {
  return p.fwd.splits > 1 ? up((size_t)p.fwd.splits * a.batch * a.heads * a.n_q * (p.D + 2) * sizeof(float)) : 0;
}
struct Backward { size_t delta, table, q, kv, bytes; };   // where the parts of the workspace begin
Backward backward_layout(const s2cnn_attention_t& a, const Plans& p) {
  const size_t queries = (size_t)a.batch * a.heads * a.n_q, keys = (size_t)a.batch * a.kv_heads * a.n_k;
  Backward w;
  w.delta = 0;
  w.table = up(queries * (a.dtype == S2CNN_F16 ? 2 : 1) * sizeof(float));
  w.q = w.table + up((size_t)p.grad_q.workgroups * a.n_buckets * sizeof(double));
  w.kv = w.q + (p.grad_q.splits > 1 ? up((size_t)p.grad_q.splits * queries * p.D * sizeof(float)) : 0);
  w.bytes = w.kv + (p.grad_kv.splits > 1 ? up((size_t)p.grad_kv.splits * 2 * keys * p.D * sizeof(float)) : 0);
  return w;
}

Args args_of(const s2cnn_attention_t& a, const Plans& plans) {
  Args p{};
  p.a = a;
  p.forward_splits = plans.fwd.splits;
  // float32 takes the factor into its columns; the others into the scores, and its inverse into the biases: never zero
  const float c = a.dtype == S2CNN_F32 ? 1.f : fabsf(a.scale) * LOG2E;
  p.c = c < 1e-30f ? 1e-30f : c;
  p.inv_c = 1.f / p.c;
  p.most = 1.5e38f / (p.c > 1.f ? p.c : 1.f);              // twice it is finite, times c too
  return p;
}

bool aligned_to_type(const s2cnn_attention_t& a) {
  const uintptr_t mask = a.dtype == S2CNN_F32 ? 3 : 1;
  for (const void* p : {a.q, a.k, a.v, a.table, (const void*)a.out, a.gout, (const void*)a.gq, (const void*)a.gk, (const void*)a.gv, (const void*)a.gtable})
    if (reinterpret_cast<uintptr_t>(p) & mask) return false;
  return !((reinterpret_cast<uintptr_t>(a.key_bias) | reinterpret_cast<uintptr_t>(a.out_f32) | reinterpret_cast<uintptr_t>(a.lengths)) & 3) && aligned8(a.stats);
}

}  // namespace
}  // namespace attn
}  // namespace s2cnn

using namespace s2cnn;
using namespace s2cnn::attn;

extern "C" size_t s2cnn_attention_workspace(const s2cnn_attention_t* a, int backward) {
  if (!sizes_ok(a)) return 0;
  const size_t own = backward ? backward_layout(*a, plans_of(*a)).bytes : forward_bytes(*a, plans_of(*a));
  if (!backward || a->heads == a->kv_heads || a->buckets) return own;
  s2cnn_attention_t c = *a;                                // whether heads are joined depends on strides that may not be known yet
  c.heads = a->kv_heads, c.n_q = a->heads / a->kv_heads * a->n_q;
  const size_t other = backward_layout(c, plans_of(c)).bytes;
  return own > other ? own : other;
}

extern "C" size_t s2cnn_attention_stats_floats(const s2cnn_attention_t* a) { return sizes_ok(a) ? (size_t)stats_floats(*a, plans_of(*a)) : 0; }

extern "C" int s2cnn_attention_fwd(const s2cnn_attention_t* a, void* workspace, size_t workspace_bytes, void* stream) {
  clear_stale_error();
  if (!sizes_ok(a) || !a->q || !a->out || (a->n_k > 0 && (!a->k || !a->v))) return S2CNN_EINVAL;
  if (!aligned_to_type(*a)) return S2CNN_EALIGN;
  const s2cnn_attention_t c = joined(*a, false);
  const Plans plans = plans_of(c);
  const size_t need = forward_bytes(c, plans);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return S2CNN_EWORKSPACE;
  Args p = args_of(c, plans);
  p.splits = plans.fwd.splits, p.tiles = plans.fwd.tiles, p.workgroups = (int)plans.fwd.workgroups;
  p.partial = static_cast<float*>(workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->dtype == S2CNN_F32) forward<F32>(p, plans, st);
  else if (a->dtype == S2CNN_BF16) forward<BF16>(p, plans, st);
  else forward<F16>(p, plans, st);
  return launch_status();
}

extern "C" int s2cnn_attention_bwd(const s2cnn_attention_t* a, void* workspace, size_t workspace_bytes, void* stream) {
  clear_stale_error();
  if (!sizes_ok(a) || a->n_k < 1 || !a->q || !a->k || !a->v || !a->out || !a->stats || !a->gout || !a->gq || !a->gk != !a->gv) return S2CNN_EINVAL;
  if ((a->gtable && !a->table) || (a->dtype != S2CNN_F32 && !a->out_f32)) return S2CNN_EINVAL;
  if (!aligned_to_type(*a)) return S2CNN_EALIGN;
  const s2cnn_attention_t c = joined(*a, true);
  const Plans plans = plans_of(c);
  const Backward w = backward_layout(c, plans);
  if (!workspace || workspace_bytes < w.bytes || !aligned16(workspace)) return S2CNN_EWORKSPACE;
  char* const at = static_cast<char*>(workspace);
  Args p = args_of(c, plans);
  p.delta = reinterpret_cast<float*>(at + w.delta);
  p.gtable_partial = reinterpret_cast<double*>(at + w.table);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  float* const q = reinterpret_cast<float*>(at + w.q);
  float* const kv = reinterpret_cast<float*>(at + w.kv);
  if (a->dtype == S2CNN_F32) backward<F32>(p, plans, q, kv, st);
  else if (a->dtype == S2CNN_BF16) backward<BF16>(p, plans, q, kv, st);
  else backward<F16>(p, plans, q, kv, st);
  return launch_status();
}
