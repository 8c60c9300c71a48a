// Norms of query and key heads that turn on the way (launch_norm_rope), alone or in front of the
// append to a paged cache (launch_paged_append_normed).
//
// z = x r w, r = (mean of x^2 + epsilon)^-1/2, then the pairs (a, b) of z become
// (a cos - b sin, b cos + a sin).  All in 32 bits, rounded once.
//
// Every head is read and written once and memory bounds it: 16384 tokens of 40 heads of 128 in
// bfloat16 (336 MB) take 67 us, 5.0 TB/s, a large copy's rate; float32 likewise.  A head's sum is 2
// to 6 exchanges between the lanes that hold it.  The append of 4 prompts of up to 4096 tokens, 8194
// in all, of 48 rows (201 MB) takes 44 us; of small calls (4.5 to 5 us) launch and lookups are all.
#include "rows.h"

namespace tg {
namespace {

constexpr int kWavesOf = 4;   // of a workgroup; each works by itself

struct Normed {
  const void *query, *key, *value;
  void *query_out, *key_out, *value_out;     // append: the last two are the caches
  const void *query_weight, *key_weight;
  const int64_t *positions, *shift;
  const double* frequency;
  i64 q_token, q_head, k_token, k_head, v_token, v_head;
  i64 qo_token, qo_head, ko_token, ko_head;  // rows of the outputs (append: of the queries')
  i64 kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  i64 qw_head, kw_head, offset;
  Table table;
  int tokens, heads, kv_heads, dim, half, layout, wide, normed;
  int rows, eights, splits, each;   // of a token: rows, groups of 64 / G, tasks, groups of a task
  Div by_splits;
  float magnitude, epsilon, inverse;
};

// A wave's task: some groups of rows of one token.
template <typename T, typename P, bool APPEND>
__global__ __launch_bounds__(64 * kWavesOf) void norm_rows(Normed a) {
  __shared__ Turns s_turns[kWavesOf];
  constexpr int R = 64 / P::G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kWavesOf + wave;
  if (task >= static_cast<int64_t>(a.tokens) * a.splits) return;
  const int token = a.by_splits(static_cast<uint32_t>(task));
  const int first = (static_cast<int>(task) - token * a.splits) * a.each;
  const int last = min(first + a.each, a.eights);
  const P place(lane & (P::G - 1), a.dim, a.half, a.layout);

  using Raw = typename P::template Raw<T>;
  // row `row` of the token: where it is read, whether it is at all
  auto from = [&](int row) -> const T* {
    if (row < a.heads)
      return static_cast<const T*>(a.query) + token * a.q_token + row * a.q_head;
    row -= a.heads;
    if (!APPEND || row < a.kv_heads)
      return static_cast<const T*>(a.key) + token * a.k_token + row * a.k_head;
    return static_cast<const T*>(a.value) + token * a.v_token + (row - a.kv_heads) * a.v_head;
  };
  auto live = [&](int row) { return row < a.rows; };
  Raw next;
  int row = first * R + lane / P::G;
  place.load(from(live(row) ? row : 0), live(row), next);

  // the token's position, and (append) its slots in the caches, if it has any: two rounds of
  // lookups, which the rows' loads do not wait for
  i64 position = 0, key_at = 0, value_at = 0;
  bool lost = false, placed = false;
  if (APPEND) {
    const Table& t = a.table;
    int b = token;
    if (t.ends) b = sequence_of(t.ends, t.sequences, token);
    lost = b >= t.sequences;
    if (!lost) {
      const i64 start = t.ends ? t.ends[b] : token, stop = t.ends ? t.ends[b + 1] : token + 1;
      const i64 length = t.lengths[b], shift = a.shift ? a.shift[b] : 0;
      const i64 begin = t.indptr[b], end = min(static_cast<i64>(t.indptr[b + 1]), t.n_indices);
      const i64 p = length - (stop - start) + (token - start);
      position = a.offset + p + shift;
      if (p >= 0 && p <= INT32_MAX && begin >= 0 && begin < end) {
        const uint32_t nth = t.by_page(static_cast<uint32_t>(p));
        if (begin + nth < end) {
          const i64 page = t.indices[begin + nth], slot = p - static_cast<i64>(nth) * t.page;
          if (page >= 0 && page < t.pages) {
            placed = true;
            key_at = page * a.kc_page + slot * a.kc_slot;
            value_at = page * a.vc_page + slot * a.vc_slot;
          }
        }
      }
    }
  } else if (a.half) {
    position = a.positions[token];
  }
  Turns& turns = s_turns[wave];
  turns_of(turns, position, a.frequency, a.half, a.magnitude);

  for (int group = first; group < last; ++group, row += R) {
    Raw x = next;
    if (group + 1 < last) place.load(from(live(row + R) ? row + R : 0), live(row + R), next);
    const bool is_query = row < a.heads, is_value = APPEND && row >= a.heads + a.kv_heads;
    float r = 1.f;
    if (a.normed) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < P::NP; ++i) {
        const float u = x.first(i), w = x.second(i);
        if (place.counts(i)) {
          sum = __builtin_fmaf(u, u, sum);
          sum = __builtin_fmaf(w, w, sum);
        }
      }
      r = rsqrtf(__builtin_fmaf(lanes_sum<P::G>(sum), a.inverse, a.epsilon));
    }
    if (!is_value) {
      const int head = is_query ? row : row - a.heads;
      const Pairs<P::NP> weight =
          weight_of<T>(place, is_query ? a.query_weight : a.key_weight, a.wide,
                       head * (is_query ? a.qw_head : a.kw_head), live(row));
#pragma unroll
      for (int i = 0; i < P::NP; ++i) {
        const int pair = place.turn(i);
        const float u = x.first(i) * r * weight.a[i], w = x.second(i) * r * weight.b[i];
        if (pair < a.half) {
          const float c = turns.c[pair], s = turns.s[pair];
          x.set(i, u * c - w * s, w * c + u * s);
        } else {
          x.set(i, u, w);
        }
      }
    }
    if (row >= a.rows) continue;
    if (APPEND) {
      if (is_query) {
        if (lost) {
#pragma unroll
          for (int i = 0; i < P::NP; ++i) x.set(i, 0.f, 0.f);
        }
      } else if (!placed) {
        continue;
      }
    }
    T* to;
    if (is_query)
      to = static_cast<T*>(a.query_out) + token * a.qo_token + row * a.qo_head;
    else if (!APPEND)
      to = static_cast<T*>(a.key_out) + token * a.ko_token + (row - a.heads) * a.ko_head;
    else if (!is_value)
      to = static_cast<T*>(a.key_out) + key_at + (row - a.heads) * a.kc_head;
    else
      to = static_cast<T*>(a.value_out) + value_at + (row - a.heads - a.kv_heads) * a.vc_head;
    place.store(to, x);
  }
}

template <typename T, typename P>
const void* kernel_of(bool append) {
  return append ? reinterpret_cast<const void*>(&norm_rows<T, P, true>)
                : reinterpret_cast<const void*>(&norm_rows<T, P, false>);
}

template <typename T, int LAYOUT, bool EDGE>
const void* kernel_of(int lanes, bool append) {
  switch (lanes) {
    case 4: return kernel_of<T, Whole<T, LAYOUT, 4, EDGE>>(append);
    case 8: return kernel_of<T, Whole<T, LAYOUT, 8, EDGE>>(append);
    case 16: return kernel_of<T, Whole<T, LAYOUT, 16, EDGE>>(append);
    case 32: return kernel_of<T, Whole<T, LAYOUT, 32, EDGE>>(append);
    default: return kernel_of<T, Whole<T, LAYOUT, 64, EDGE>>(append);
  }
}

template <typename T>
const void* kernel_of(int64_t layout, Lanes l, bool append) {
  if (l.cut == kRagged) return kernel_of<T, Ragged<T>>(append);
  if (layout == TG_HALF)
    return l.cut == kEdge ? kernel_of<T, TG_HALF, true>(l.lanes, append)
                          : kernel_of<T, TG_HALF, false>(l.lanes, append);
  return l.cut == kEdge ? kernel_of<T, TG_INTERLEAVED, true>(l.lanes, append)
                        : kernel_of<T, TG_INTERLEAVED, false>(l.lanes, append);
}

int enqueue(Normed& a, int64_t dtype, bool append, const char* what, hipStream_t stream) {
  const Lanes l = lanes_of(dtype, a.dim, a.half, a.layout);
  a.rows = a.heads + (append ? 2 : 1) * a.kv_heads;
  a.eights = (a.rows + 64 / l.lanes - 1) / (64 / l.lanes);
  // Tasks of one group of rows while there are few, else of three (of pairs of halves, 32 bytes a lane;
  // five of 16 bytes): waves start with the token's lookups and angles, and long ones end in an uneven
  // last turn.  16384 tokens of 40 heads of 128 in bfloat16: 73.6 us by 5 groups, 66.0 by 3, 66.5 by 1;
  // interleaved 73.2 by 5, 77.0 by 3, 94.9 by 1.  Appending 8194 tokens of 48 rows: 53.0 by 1,
  // 43.9 by 3, 46.9 by 5; interleaved 56.9 by 3, 55.2 by 4.  3000 tokens of 40 heads: 14.5 by 1, 12.7
  // by 3.
  const int64_t groups = static_cast<int64_t>(a.tokens) * a.eights;
  int64_t each = groups / 4096, most = a.layout == TG_HALF ? 3 : 5;
  each = each < 1 ? 1 : each < most ? each : most;
  const int64_t room = kWavesOf * kMostGroups / a.tokens, splits = (a.eights + each - 1) / each;
  a.splits = static_cast<int>(splits < room ? splits : room);     // (one launch: at least 8 fit)
  a.each = (a.eights + a.splits - 1) / a.splits;
  a.by_splits = Div(a.splits);
  const int64_t tasks = static_cast<int64_t>(a.tokens) * a.splits;
  const void* k = dtype == TG_F32   ? kernel_of<float>(a.layout, l, append)
                  : dtype == TG_F16 ? kernel_of<_Float16>(a.layout, l, append)
                                    : kernel_of<__bf16>(a.layout, l, append);
  void* args[] = {&a};
  const hipError_t e = launch(k, (tasks + kWavesOf - 1) / kWavesOf, 64 * kWavesOf, args, stream);
  return e == hipSuccess ? 0 : hip_failed(e, what);
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" __attribute__((visibility("default"))) int launch_norm_rope(const tg_norm_rope* r,
                                                                       void* stream) {
  const char* what = "launch_norm_rope";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (const int rc = check_norm(what, r->dtype, r->weight_dtype, r->tokens, r->heads, r->kv_heads,
                                r->dim, r->rotary, r->layout, r->epsilon))
    return rc;
  if (r->tokens == 0 || r->heads + r->kv_heads == 0) return 0;
  const Operand query = {"query", r->query, 3, {r->tokens, r->heads, r->dim},
                         {r->query_token, r->query_head, 1}};
  const Operand key = {"key", r->key, 3, {r->tokens, r->kv_heads, r->dim},
                       {r->key_token, r->key_head, 1}};
  const Operand query_out = {"query_out", r->query_out, 3, {r->tokens, r->heads, r->dim},
                             {r->qout_token, r->qout_head, 1}};
  const Operand key_out = {"key_out", r->key_out, 3, {r->tokens, r->kv_heads, r->dim},
                           {r->kout_token, r->kout_head, 1}};
  const int bytes = r->dtype == TG_F32 ? 4 : 2;
  if (const int rc = once(what, query_out)) return rc;
  if (const int rc = once(what, key_out)) return rc;
  if (const int rc = apart(what, query_out, key_out, bytes)) return rc;
  if (!same(query_out, query))
    if (const int rc = apart(what, query_out, query, bytes)) return rc;
  if (!same(key_out, key))
    if (const int rc = apart(what, key_out, key, bytes)) return rc;
  if (const int rc = apart(what, query_out, key, bytes)) return rc;
  if (const int rc = apart(what, key_out, query, bytes)) return rc;
  if ((r->heads && (!r->query || !r->query_out)) || (r->kv_heads && (!r->key || !r->key_out)) ||
      (r->rotary && (!r->frequency || !r->positions)))
    return refuse(-1, what, "null array", r->tokens);
  Normed a = {};
  a.query = r->query;
  a.key = r->key;
  a.query_out = r->query_out;
  a.key_out = r->key_out;
  a.query_weight = r->query_weight;
  a.key_weight = r->key_weight;
  a.positions = r->positions;
  a.frequency = r->frequency;
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
  a.tokens = static_cast<int>(r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.dim = static_cast<int>(r->dim);
  a.half = static_cast<int>(r->rotary / 2);
  a.layout = static_cast<int>(r->layout);
  a.wide = r->weight_dtype == TG_F32;
  a.normed = 1;
  a.magnitude = static_cast<float>(r->magnitude);
  a.epsilon = static_cast<float>(r->epsilon);
  a.inverse = 1.f / a.dim;
  return enqueue(a, r->dtype, false, what, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) int launch_paged_append_normed(
    const tg_paged_append_normed* r, void* stream) {
  const char* what = "launch_paged_append_normed";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (const int rc = check_norm(what, r->dtype, r->weight_dtype, r->tokens, r->heads, r->kv_heads,
                                r->dim, r->rotary, r->layout, r->epsilon))
    return rc;
  if (r->kv_heads < 1) return refuse(-1, what, "kv_heads must be 1 to 65536", r->kv_heads);
  if (r->normed != 0 && r->normed != 1)
    return refuse(-1, what, "normed must be 0 or 1", r->normed);
  if (!r->normed && (r->query_weight || r->key_weight))
    return refuse(-1, what, "weights without a norm", 0);
  if (const int rc = check_table(what, r->sequences, r->pages, r->page, r->n_indices, 0)) return rc;
  if (!r->query_indptr && r->tokens > r->sequences)
    return refuse(-1, what, "more tokens than sequences without query_indptr", r->tokens);
  if (r->tokens == 0) return 0;
  // As in launch_paged_append: what is written shares no memory with what else is written, or
  // with the rows of new tokens (which may stand in the caches, in slots that are not written).
  const Operand key = {"key", r->key, 3, {r->tokens, r->kv_heads, r->dim},
                       {r->key_token, r->key_head, 1}};
  const Operand value = {"value", r->value, 3, {r->tokens, r->kv_heads, r->dim},
                         {r->value_token, r->value_head, 1}};
  const Operand query = {"query", r->query, 3, {r->tokens, r->heads, r->dim},
                         {r->query_token, r->query_head, 1}};
  const Operand out = {"query_out", r->query_out, 3, {r->tokens, r->heads, r->dim},
                       {r->out_token, r->out_head, 1}};
  const Operand kc = {"key_cache", r->key_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->kc_page, r->kc_slot, r->kc_head, 1}};
  const Operand vc = {"value_cache", r->value_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->vc_page, r->vc_slot, r->vc_head, 1}};
  const int bytes = r->dtype == TG_F32 ? 4 : 2;
  for (const Operand* x : {&kc, &vc})
    if (const int rc = once(what, *x)) return rc;
  if (r->heads) {
    if (const int rc = once(what, out)) return rc;
    if (!same(out, query))
      if (const int rc = apart(what, out, query, bytes)) return rc;
    for (const Operand* x : {&key, &value, &kc, &vc})
      if (const int rc = apart(what, out, *x, bytes)) return rc;
  }
  if (const int rc = apart(what, vc, kc, bytes)) return rc;
  if (!r->key || !r->value || (r->pages && (!r->key_cache || !r->value_cache)) || !r->indptr ||
      !r->lengths || (r->n_indices && !r->indices) ||
      (r->heads && (!r->query || !r->query_out)) || (r->rotary && !r->frequency))
    return refuse(-1, what, "null array", r->tokens);
  Normed a = {};
  a.query = r->query;
  a.key = r->key;
  a.value = r->value;
  a.query_out = r->query_out;
  a.key_out = r->key_cache;
  a.value_out = r->value_cache;
  a.query_weight = r->query_weight;
  a.key_weight = r->key_weight;
  a.shift = r->shift;
  a.frequency = r->frequency;
  a.q_token = r->query_token;
  a.q_head = r->query_head;
  a.k_token = r->key_token;
  a.k_head = r->key_head;
  a.v_token = r->value_token;
  a.v_head = r->value_head;
  a.qo_token = r->out_token;
  a.qo_head = r->out_head;
  a.kc_page = r->kc_page;
  a.kc_slot = r->kc_slot;
  a.kc_head = r->kc_head;
  a.vc_page = r->vc_page;
  a.vc_slot = r->vc_slot;
  a.vc_head = r->vc_head;
  a.qw_head = r->query_weight_head;
  a.kw_head = r->key_weight_head;
  a.offset = r->offset;
  a.table.indptr = r->indptr;
  a.table.indices = r->indices;
  a.table.lengths = r->lengths;
  a.table.ends = r->query_indptr;
  a.table.pages = r->pages;
  a.table.n_indices = r->n_indices;
  a.table.tokens = static_cast<int>(r->tokens);
  a.table.sequences = static_cast<int>(r->sequences);
  a.table.page = static_cast<int>(r->page);
  a.table.by_page = Div(a.table.page);
  a.tokens = static_cast<int>(r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.dim = static_cast<int>(r->dim);
  a.half = static_cast<int>(r->rotary / 2);
  a.layout = static_cast<int>(r->layout);
  a.wide = r->weight_dtype == TG_F32;
  a.normed = static_cast<int>(r->normed);
  a.magnitude = static_cast<float>(r->magnitude);
  a.epsilon = static_cast<float>(r->epsilon);
  a.inverse = 1.f / a.dim;
  return enqueue(a, r->dtype, true, what, static_cast<hipStream_t>(stream));
}
