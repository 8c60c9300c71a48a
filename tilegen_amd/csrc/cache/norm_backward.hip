// The gradients of norms that turn (launch_norm_rope_backward).
//
// With g the gradient of a turned row, u = g turned back (the pair (a, b) becomes
// (a cos + b sin, b cos - a sin)), v = u w and r = (mean of x^2 + epsilon)^-1/2:
//
//   dx = r (v - x r^2 (mean of v x)),     dw = the sum over rows of u x r
//
// A wave keeps to the same heads and goes over tokens, so that every lane sums the elements of
// its own heads in registers.  A workgroup's sums go to the workspace, by head or, of a weight
// that all heads share, as one row; a second kernel adds them up.  All in 32 bits, in an order
// that the sizes alone decide.
//
// Memory bounds it: 16384 tokens of 40 heads of 128 in bfloat16 (503 MB) take 96 us, 5.2 TB/s, and
// adding up the sums of 5 x 153 workgroups 4.8; 4095 of 25 heads of 96 in float32 (118 MB) 23.6 and
// 4.0.  Sums over tokens in registers cost no traffic; atomics would cost the order.  Of 8 or 64
// tokens it takes 8.3 and 2.6 us, behind a call that costs the host 19.
#include "rows.h"

namespace tg {
namespace {

constexpr int kWavesOf = 4;

struct Back {
  const void *grad_query, *grad_key, *query, *key;
  void *query_out, *key_out;
  const void *query_weight, *key_weight;
  const int64_t* positions;
  const double* frequency;
  float *query_part, *key_part;     // null: not wanted
  i64 gq_token, gq_head, gk_token, gk_head, q_token, q_head, k_token, k_head;
  i64 qo_token, qo_head, ko_token, ko_head, qw_head, kw_head;
  int tokens, heads, kv_heads, dim, half, layout, wide;
  int rows, eights, blocks;         // groups of 64 / G rows; workgroups that share the tokens
  int key_first;                    // the first group with a row of the keys
  int query_each, key_each;         // weights by head (0: one for all)
  Div by_eights;
  float magnitude, epsilon, inverse;
};

template <typename T, typename P>
__global__ __launch_bounds__(64 * kWavesOf) void norm_rows_backward(Back a) {
  __shared__ Turns s_turns[kWavesOf];
  __shared__ float s_sum[kWavesOf][2 * P::NP][64];
  constexpr int R = 64 / P::G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int block = a.by_eights(blockIdx.x), group = blockIdx.x - block * a.eights;
  const P place(lane & (P::G - 1), a.dim, a.half, a.layout);
  using Raw = typename P::template Raw<T>;

  const int row = group * R + lane / P::G;
  const bool live = row < a.rows, is_query = row < a.heads;
  const int head = live ? is_query ? row : row - a.heads : 0;
  const T* x_at = static_cast<const T*>(is_query ? a.query : a.key) +
                  head * (is_query ? a.q_head : a.k_head);
  const T* g_at = static_cast<const T*>(is_query ? a.grad_query : a.grad_key) +
                  head * (is_query ? a.gq_head : a.gk_head);
  T* to = static_cast<T*>(is_query ? a.query_out : a.key_out) +
          head * (is_query ? a.qo_head : a.ko_head);
  const i64 x_token = is_query ? a.q_token : a.k_token;
  const i64 g_token = is_query ? a.gq_token : a.gk_token;
  const i64 to_token = is_query ? a.qo_token : a.ko_token;
  const Pairs<P::NP> w = weight_of<T>(place, is_query ? a.query_weight : a.key_weight, a.wide,
                                      head * (is_query ? a.qw_head : a.kw_head), live);
  float da[P::NP], db[P::NP];
#pragma unroll
  for (int i = 0; i < P::NP; ++i) da[i] = db[i] = 0.f;

  const int step = a.blocks * kWavesOf;
  int token = block * kWavesOf + wave;
  Raw next_x, next_g;
  i64 next_position = 0;
  auto load = [&](int t) {
    place.load(x_at + t * x_token, live, next_x);
    place.load(g_at + t * g_token, live, next_g);
    if (a.half) next_position = a.positions[t];
  };
  if (token < a.tokens) load(token);
  Turns& turns = s_turns[wave];
  for (; token < a.tokens; token += step) {
    Raw x = next_x;
    const Raw g = next_g;
    turns_of(turns, next_position, a.frequency, a.half, a.magnitude);
    if (token + step < a.tokens) load(token + step);
    float ua[P::NP], ub[P::NP];
    float square = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < P::NP; ++i) {
      const int pair = place.turn(i);
      const float p = g.first(i), q = g.second(i), y = x.first(i), z = x.second(i);
      ua[i] = p;
      ub[i] = q;
      if (pair < a.half) {
        const float c = turns.c[pair], s = turns.s[pair];
        ua[i] = p * c + q * s;
        ub[i] = q * c - p * s;
      }
      if (place.counts(i)) {
        square = __builtin_fmaf(y, y, square);
        square = __builtin_fmaf(z, z, square);
        dot = __builtin_fmaf(ua[i] * w.a[i], y, dot);
        dot = __builtin_fmaf(ub[i] * w.b[i], z, dot);
      }
    }
    const float r = rsqrtf(__builtin_fmaf(lanes_sum<P::G>(square), a.inverse, a.epsilon));
    const float back = lanes_sum<P::G>(dot) * a.inverse * r * r;
#pragma unroll
    for (int i = 0; i < P::NP; ++i) {
      const float y = x.first(i), z = x.second(i);
      da[i] = __builtin_fmaf(ua[i], y * r, da[i]);
      db[i] = __builtin_fmaf(ub[i], z * r, db[i]);
      x.set(i, r * (ua[i] * w.a[i] - y * back), r * (ub[i] * w.b[i] - z * back));
    }
    if (live) place.store(to + token * to_token, x);
  }

  // the workgroup's sums: by head, or the rows of one weight together
  if (!a.query_part && !a.key_part) return;
#pragma unroll
  for (int i = 0; i < P::NP; ++i) {
    s_sum[wave][i][lane] = live ? da[i] : 0.f;
    s_sum[wave][P::NP + i][lane] = live ? db[i] : 0.f;
  }
  __syncthreads();
  const int row0 = group * R;
  for (int at = threadIdx.x; at < 64 * 2 * P::NP; at += 64 * kWavesOf) {
    const int j = at / 64, l = at & 63, unit = l & (P::G - 1), r = row0 + l / P::G;
    const P mine(unit, a.dim, a.half, a.layout);
    const int d = mine.element(j < P::NP ? j : j - P::NP, j >= P::NP);
    if (d < 0 || r >= a.rows) continue;
    const bool q = r < a.heads;
    float* part = q ? a.query_part : a.key_part;
    if (!part) continue;
    if (q ? a.query_each : a.key_each) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWavesOf; ++w) sum += s_sum[w][j][l];
      const int h = q ? r : r - a.heads, heads = q ? a.heads : a.kv_heads;
      part[(static_cast<i64>(block) * heads + h) * a.dim + d] = sum;
    } else if (r == row0 || r == a.heads) {     // the first of its weight in the group
      float sum = 0.f;
      for (int m = l; m < 64 && (m / P::G + row0 < a.heads) == q; m += P::G)
#pragma unroll
        for (int w = 0; w < kWavesOf; ++w) sum += s_sum[w][j][m];
      const int groups = q ? (a.heads + R - 1) / R : a.eights - a.key_first;
      const int nth = q ? group : group - a.key_first;
      part[(static_cast<i64>(block) * groups + nth) * a.dim + d] = sum;
    }
  }
}

// Columns summed over parts: 16 columns a workgroup, 64 parts side by side.
struct Sums {
  const float *query, *key;
  void *query_out, *key_out;
  int query_columns, key_columns, query_parts, key_parts;
  int query_groups;     // workgroups of the query's columns
};

constexpr int kColumns = 16, kSlices = 64;

template <typename W>
__global__ __launch_bounds__(kColumns* kSlices) void sum_parts(Sums a) {
  __shared__ float s_sum[kSlices][kColumns];
  const bool q = static_cast<int>(blockIdx.x) < a.query_groups;
  const int columns = q ? a.query_columns : a.key_columns;
  const int parts = q ? a.query_parts : a.key_parts;
  const float* from = q ? a.query : a.key;
  const int column = (blockIdx.x - (q ? 0 : a.query_groups)) * kColumns + threadIdx.x % kColumns;
  const int slice = threadIdx.x / kColumns;
  float sum = 0.f;
  if (column < columns) {
#pragma unroll 8
    for (int p = slice; p < parts; p += kSlices) sum += from[static_cast<i64>(p) * columns + column];
  }
  s_sum[slice][threadIdx.x % kColumns] = sum;
  __syncthreads();
  for (int n = kSlices / 2; n; n /= 2) {
    if (slice < n) s_sum[slice][threadIdx.x % kColumns] += s_sum[slice + n][threadIdx.x % kColumns];
    __syncthreads();
  }
  if (slice == 0 && column < columns)
    static_cast<W*>(q ? a.query_out : a.key_out)[column] =
        static_cast<W>(s_sum[0][threadIdx.x % kColumns]);
}

template <typename T, typename P>
const void* kernel_of() {
  return reinterpret_cast<const void*>(&norm_rows_backward<T, P>);
}

template <typename T, int LAYOUT, bool EDGE>
const void* kernel_of(int lanes) {
  switch (lanes) {
    case 4: return kernel_of<T, Whole<T, LAYOUT, 4, EDGE>>();
    case 8: return kernel_of<T, Whole<T, LAYOUT, 8, EDGE>>();
    case 16: return kernel_of<T, Whole<T, LAYOUT, 16, EDGE>>();
    case 32: return kernel_of<T, Whole<T, LAYOUT, 32, EDGE>>();
    default: return kernel_of<T, Whole<T, LAYOUT, 64, EDGE>>();
  }
}

template <typename T>
const void* kernel_of(int64_t layout, Lanes l) {
  if (l.cut == kRagged) return kernel_of<T, Ragged<T>>();
  if (layout == TG_HALF)
    return l.cut == kEdge ? kernel_of<T, TG_HALF, true>(l.lanes)
                          : kernel_of<T, TG_HALF, false>(l.lanes);
  return l.cut == kEdge ? kernel_of<T, TG_INTERLEAVED, true>(l.lanes)
                        : kernel_of<T, TG_INTERLEAVED, false>(l.lanes);
}

struct Plan {
  Back a;
  Sums sums;
  Lanes lanes;
  int64_t query_floats, key_floats;
};

int plan(const tg_norm_rope_backward* r, Plan* p) {
  const char* what = "launch_norm_rope_backward";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (const int rc = check_norm(what, r->dtype, r->weight_dtype, r->tokens, r->heads, r->kv_heads,
                                r->dim, r->rotary, r->layout, r->epsilon))
    return rc;
  if ((r->query_weight_out && !r->query_weight) || (r->key_weight_out && !r->key_weight))
    return refuse(-1, what, "a weight's gradient without the weight", 0);
  *p = Plan{};
  Back& a = p->a;
  a.tokens = static_cast<int>(r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.dim = static_cast<int>(r->dim);
  a.half = static_cast<int>(r->rotary / 2);
  a.layout = static_cast<int>(r->layout);
  a.rows = a.heads + a.kv_heads;
  p->lanes = lanes_of(r->dtype, a.dim, a.half, a.layout);
  const int R = 64 / p->lanes.lanes;
  a.eights = (a.rows + R - 1) / R;
  a.key_first = a.heads / R;
  a.by_eights = Div(a.eights ? a.eights : 1);
  // Workgroups that share the tokens, as many in all as the chip holds of them at once: by their
  // registers 768, or twice that where a lane has few pairs.  16384 tokens of 40 heads of 128 in
  // bfloat16: 100 us by 768, 108 by 1536; 4095 of 25 heads of 96 in float32, interleaved: 29.2 and
  // 25.9; 8192 of 128 elements with 62 turned: 210 and 145.
  const int64_t most = (r->tokens + kWavesOf - 1) / kWavesOf;
  const bool many = p->lanes.cut == kRagged || (r->dtype == TG_F32 && a.layout == TG_INTERLEAVED);
  int64_t blocks = a.eights ? (many ? 1536 : 768) / a.eights : 1;
  blocks = blocks < 1 ? 1 : blocks < most ? blocks : most;
  a.blocks = static_cast<int>(blocks);
  a.query_each = r->query_weight_head != 0;
  a.key_each = r->key_weight_head != 0;
  Sums& s = p->sums;
  s.query_columns = a.query_each ? a.heads * a.dim : a.dim;
  s.key_columns = a.key_each ? a.kv_heads * a.dim : a.dim;
  s.query_parts = a.blocks * (a.query_each ? 1 : (a.heads + R - 1) / R);
  s.key_parts = a.blocks * (a.key_each ? 1 : a.eights - a.key_first);
  if (!a.heads) s.query_parts = 0;
  if (!a.kv_heads) s.key_parts = 0;
  if (r->query_weight_out)
    p->query_floats = static_cast<int64_t>(s.query_columns) * s.query_parts;
  if (r->key_weight_out)
    p->key_floats = static_cast<int64_t>(s.key_columns) * s.key_parts;
  return 0;
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" __attribute__((visibility("default"))) int64_t norm_rope_backward_workspace(
    const tg_norm_rope_backward* r) {
  Plan p;
  if (const int rc = plan(r, &p)) return rc < 0 ? rc : -1;
  return (p.query_floats + p.key_floats) * 4;
}

extern "C" __attribute__((visibility("default"))) int launch_norm_rope_backward(
    const tg_norm_rope_backward* r, void* stream) {
  const char* what = "launch_norm_rope_backward";
  Plan p;
  if (const int rc = plan(r, &p)) return rc;
  Back& a = p.a;
  const Operand query = {"query", r->query, 3, {r->tokens, r->heads, r->dim},
                         {r->query_token, r->query_head, 1}};
  const Operand key = {"key", r->key, 3, {r->tokens, r->kv_heads, r->dim},
                       {r->key_token, r->key_head, 1}};
  const Operand grad_query = {"grad_query", r->grad_query, 3, {r->tokens, r->heads, r->dim},
                              {r->grad_query_token, r->grad_query_head, 1}};
  const Operand grad_key = {"grad_key", r->grad_key, 3, {r->tokens, r->kv_heads, r->dim},
                            {r->grad_key_token, r->grad_key_head, 1}};
  const Operand query_out = {"query_out", r->query_out, 3, {r->tokens, r->heads, r->dim},
                             {r->qout_token, r->qout_head, 1}};
  const Operand key_out = {"key_out", r->key_out, 3, {r->tokens, r->kv_heads, r->dim},
                           {r->kout_token, r->kout_head, 1}};
  const int bytes = r->dtype == TG_F32 ? 4 : 2;
  if (const int rc = once(what, query_out)) return rc;
  if (const int rc = once(what, key_out)) return rc;
  if (const int rc = apart(what, query_out, key_out, bytes)) return rc;
  for (const Operand* x : {&query, &grad_query, &key, &grad_key}) {
    if (x == &key || x == &grad_key || !same(query_out, *x))
      if (const int rc = apart(what, query_out, *x, bytes)) return rc;
    if (x == &query || x == &grad_query || !same(key_out, *x))
      if (const int rc = apart(what, key_out, *x, bytes)) return rc;
  }
  if (a.tokens && a.rows &&
      ((r->heads && (!r->query || !r->grad_query || !r->query_out)) ||
       (r->kv_heads && (!r->key || !r->grad_key || !r->key_out)) ||
       (r->rotary && (!r->frequency || !r->positions))))
    return refuse(-1, what, "null array", r->tokens);
  const int64_t need = (p.query_floats + p.key_floats) * 4;
  if (r->workspace_bytes < need || (need && !r->workspace))
    return refuse(-1, what, "the workspace is too small; bytes needed", need);
  if (reinterpret_cast<uintptr_t>(r->workspace) % 16)
    return refuse(-1, what, "the workspace is not 16-byte aligned", 0);
  a.grad_query = r->grad_query;
  a.grad_key = r->grad_key;
  a.query = r->query;
  a.key = r->key;
  a.query_out = r->query_out;
  a.key_out = r->key_out;
  a.query_weight = r->query_weight;
  a.key_weight = r->key_weight;
  a.positions = r->positions;
  a.frequency = r->frequency;
  a.gq_token = r->grad_query_token;
  a.gq_head = r->grad_query_head;
  a.gk_token = r->grad_key_token;
  a.gk_head = r->grad_key_head;
  a.q_token = r->query_token;
  a.q_head = r->query_head;
  a.k_token = r->key_token;
  a.k_head = r->key_head;
  a.qo_token = r->qout_token;
  a.qo_head = r->qout_head;
  a.ko_token = r->kout_token;
  a.ko_head = r->kout_head;
  a.qw_head = r->query_weight_head;
  a.kw_head = r->key_weight_head;
  a.wide = r->weight_dtype == TG_F32;
  a.magnitude = static_cast<float>(r->magnitude);
  a.epsilon = static_cast<float>(r->epsilon);
  a.inverse = 1.f / a.dim;
  float* space = static_cast<float*>(r->workspace);
  a.query_part = p.query_floats ? space : nullptr;
  a.key_part = p.key_floats ? space + p.query_floats : nullptr;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t groups = static_cast<int64_t>(a.blocks) * a.eights;
  const void* k = r->dtype == TG_F32   ? kernel_of<float>(a.layout, p.lanes)
                  : r->dtype == TG_F16 ? kernel_of<_Float16>(a.layout, p.lanes)
                                       : kernel_of<__bf16>(a.layout, p.lanes);
  if (a.tokens && a.rows) {
    void* args[] = {&a};
    const hipError_t e = launch(k, groups, 64 * kWavesOf, args, s);
    if (e != hipSuccess) return hip_failed(e, what);
  }
  // (without tokens or heads the sums have no parts and come out as 0)
  Sums& u = p.sums;
  const bool q = r->query_weight_out && u.query_columns, w = r->key_weight_out && u.key_columns;
  if (!q && !w) return 0;
  u.query = a.query_part;
  u.key = a.key_part;
  u.query_out = r->query_weight_out;
  u.key_out = r->key_weight_out;
  u.query_groups = q ? (u.query_columns + kColumns - 1) / kColumns : 0;
  const int key_groups = w ? (u.key_columns + kColumns - 1) / kColumns : 0;
  void* args[] = {&u};
  const void* sum = r->weight_dtype == TG_F32   ? reinterpret_cast<const void*>(&sum_parts<float>)
                    : r->weight_dtype == TG_F16 ? reinterpret_cast<const void*>(&sum_parts<_Float16>)
                                                : reinterpret_cast<const void*>(&sum_parts<__bf16>);
  const hipError_t e = launch(sum, u.query_groups + key_groups, kColumns * kSlices, args, s);
  return e == hipSuccess ? 0 : hip_failed(e, what);
}
