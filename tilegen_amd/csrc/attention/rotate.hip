// Rotary positions (launch_rope) and the append to a paged cache that turns keys and queries
// on the way (launch_paged_append): one kernel, whose rows are the heads of a token.
//
// Memory bounds it: every value is read and written once, in 16-byte units, and the cosines and
// sines are computed once a token for all its heads.  16384 tokens of 40 heads of 128 in
// bfloat16 (336 MB) take 59 us, 5.7 TB/s; an append of 16384 tokens with their queries (403 MB)
// 75 to 79, 5.1 to 5.4 TB/s; a plain copy of 1 GiB reaches 4.8.  8 tokens take 3.2 us, an append of
// 32 with its page lookups 4.1: the latency of the loads that follow from one another.
#include "attention.h"

namespace tg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;
constexpr int kMaxSequences = 1 << 30;   // sequence_of's places stay within 32 bits
constexpr int kMostTokens = 4;   // tokens of one workgroup

struct Rows {
  // rows turned from x to y (the input of rope, the queries of append)
  const void* x;
  void* y;
  i64 x_token, x_head, y_token, y_head;
  const double* frequency;
  const int64_t* positions;      // rope; append finds them
  int tokens, heads, dim, half, sign;
  float magnitude;
  int per_token;                 // units of work of one token
  int turned, plain;             // units of a turned row, of a copied row
  Div by_token, by_turned, by_plain, by_page;
  // append alone
  const void *key, *value;
  void *key_cache, *value_cache;
  i64 key_token, key_head, value_token, value_head;
  i64 kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  const int64_t *indptr, *indices, *lengths, *query_indptr;
  int sequences, kv_heads, page;
  i64 pages, n_indices, offset;
};

// A unit is one 16-byte chunk of a copied row, one chunk of interleaved pairs, or one chunk of
// first halves with the chunk of their second halves.  WHOLE: rows consist of whole chunks
// (dim, and for halves rotary/2, are multiples of a chunk).
template <typename T, bool WHOLE>
__device__ __forceinline__ void copy_unit(const T* __restrict__ src, T* __restrict__ dst, int off,
                                          int dim, bool zero) {
  using C = Chunk<T>;
  typename C::Vec v;
  if (WHOLE || off + C::N <= dim) {
    v = C::load(src + off);
    if (zero) v = typename C::Vec(T(0));
    C::store(dst + off, v);
  } else {
    for (int i = off; i < dim; ++i) dst[i] = zero ? T(0) : src[i];
  }
}

// src and dst may be the same row, so neither is __restrict__: a unit reads all that it writes
// before it writes, and no unit reads another's.
template <typename T, int LAYOUT, bool WHOLE>
__device__ __forceinline__ void turn_unit(const T* src, T* dst, int unit, int half, int dim,
                                          const float* cs, const float* sn, bool zero) {
  using C = Chunk<T>;
  using Vec = typename C::Vec;
  if (LAYOUT == TG_HALF) {
    const int first = (half + C::N - 1) / C::N;
    if (unit >= first) {
      const int off = 2 * half + (unit - first) * C::N;
      if (WHOLE || off + C::N <= dim) {
        Vec v = C::load(src + off);
        if (zero) v = Vec(T(0));
        C::store(dst + off, v);
      } else {
        for (int i = off; i < dim; ++i) dst[i] = zero ? T(0) : src[i];
      }
      return;
    }
    const int off = unit * C::N;
    if (WHOLE || off + C::N <= half) {
      const Vec a = C::load(src + off), b = C::load(src + half + off);
      Vec p, q;
#pragma unroll
      for (int i = 0; i < C::N; ++i) {
        const float c = cs[off + i], s = sn[off + i];
        const float u = static_cast<float>(a[i]), w = static_cast<float>(b[i]);
        p[i] = zero ? T(0) : static_cast<T>(u * c - w * s);
        q[i] = zero ? T(0) : static_cast<T>(w * c + u * s);
      }
      C::store(dst + off, p);
      C::store(dst + half + off, q);
    } else {
      for (int i = off; i < half; ++i) {
        const float u = static_cast<float>(src[i]), w = static_cast<float>(src[half + i]);
        dst[i] = zero ? T(0) : static_cast<T>(u * cs[i] - w * sn[i]);
        dst[half + i] = zero ? T(0) : static_cast<T>(w * cs[i] + u * sn[i]);
      }
    }
  } else {
    const int off = unit * C::N;
    if (WHOLE || off + C::N <= dim) {
      Vec v = C::load(src + off);
#pragma unroll
      for (int i = 0; i < C::N; i += 2) {
        const int pair = off / 2 + i / 2;
        if (pair < half) {
          const float c = cs[pair], s = sn[pair];
          const float u = static_cast<float>(v[i]), w = static_cast<float>(v[i + 1]);
          v[i] = static_cast<T>(u * c - w * s);
          v[i + 1] = static_cast<T>(w * c + u * s);
        }
      }
      if (zero) v = Vec(T(0));
      C::store(dst + off, v);
    } else {
      for (int i = off; i < dim; i += 2) {
        const float u = static_cast<float>(src[i]);
        const float w = i + 1 < dim ? static_cast<float>(src[i + 1]) : 0.f;
        float p = u, q = w;
        if (i / 2 < half) {
          p = u * cs[i / 2] - w * sn[i / 2];
          q = w * cs[i / 2] + u * sn[i / 2];
        }
        dst[i] = zero ? T(0) : static_cast<T>(p);
        if (i + 1 < dim) dst[i + 1] = zero ? T(0) : static_cast<T>(q);
      }
    }
  }
}

// One workgroup takes n_tokens tokens: their positions, the cosine and sine of every pair of
// each token once into LDS, then all heads' rows in 16-byte units.
//
// Angles: positions reach 2^17 and more, where position * frequency in 32 bits would be off by
// 2^-8 radians.  The product is taken in 64 bits as turns (one multiplication a pair), and its
// fraction, at most half a turn and exact to 2^-25 of itself in 32 bits, goes to sincospi.
template <typename T, int LAYOUT, bool WHOLE, bool APPEND>
__global__ __launch_bounds__(kThreads) void rotate_rows(Rows a, int n_tokens) {
  __shared__ float s_cos[kMostTokens * kMaxDim / 2], s_sin[kMostTokens * kMaxDim / 2];
  __shared__ i64 s_position[kMostTokens], s_key[kMostTokens], s_value[kMostTokens];
  const int tid = threadIdx.x;
  const int t0 = static_cast<int>(blockIdx.x) * n_tokens;
  const int count = min(n_tokens, a.tokens - t0);
  if (APPEND) {
    // wave w finds token w's place: s_key/s_value its slot in the caches, or -1; s_position -1
    // for a token of no sequence
    const int w = tid / 64;
    if (w < count) {
      const int t = t0 + w;
      int b = t;
      i64 start = t, n = 1;
      if (a.query_indptr) {
        b = sequence_of(a.query_indptr, a.sequences, t);
        if (b < a.sequences) {
          start = a.query_indptr[b];
          n = a.query_indptr[b + 1] - start;
        }
      }
      i64 position = -1, key = -1, value = -1;
      if (b < a.sequences) {
        const i64 p = a.lengths[b] - n + (t - start);
        position = a.offset + p;
        const i64 begin = a.indptr[b], end = min(static_cast<i64>(a.indptr[b + 1]), a.n_indices);
        if (p >= 0 && p <= INT32_MAX && begin >= 0 && begin < end) {
          const uint32_t nth = a.by_page(static_cast<uint32_t>(p));
          const i64 at = begin + nth;
          if (at < end) {
            const i64 pg = a.indices[at], slot = p - static_cast<i64>(nth) * a.page;
            if (pg >= 0 && pg < a.pages) {
              key = pg * a.kc_page + slot * a.kc_slot;
              value = pg * a.vc_page + slot * a.vc_slot;
            }
          }
        }
      }
      if ((tid & 63) == 0) {
        s_position[w] = b < a.sequences ? position : INT64_MIN;
        s_key[w] = key;
        s_value[w] = value;
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < count * a.half; i += kThreads) {
    const int t = i / a.half, pair = i - t * a.half;
    const i64 position = APPEND ? s_position[t] : a.positions[t0 + t];
    constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
    const double turns = static_cast<double>(position) * (a.frequency[pair] * kPerTurn);
    const float f = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.f * f, &s, &c);
    s_cos[i] = c * a.magnitude;
    s_sin[i] = s * a.magnitude * static_cast<float>(a.sign);
  }
  __syncthreads();
  const int units = count * a.per_token;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  for (int i = tid; i < units; i += kThreads) {
    const int t = a.by_token(i);
    int u = i - t * a.per_token;
    const int token = t0 + t;
    const float *cs = s_cos + t * a.half, *sn = s_sin + t * a.half;
    if (!APPEND) {
      const int h = a.by_turned(u);
      turn_unit<T, LAYOUT, WHOLE>(x + token * a.x_token + h * a.x_head,
                                  y + token * a.y_token + h * a.y_head, u - h * a.turned, a.half,
                                  a.dim, cs, sn, false);
    } else {
      const int rows = (a.heads + a.kv_heads) * a.turned;
      if (u < rows) {
        const int h = a.by_turned(u);
        const T* src;
        T* dst;
        bool zero = false;
        if (h < a.heads) {
          src = x + token * a.x_token + h * a.x_head;
          dst = y + token * a.y_token + h * a.y_head;
          zero = s_position[t] == INT64_MIN;
        } else {
          if (s_key[t] < 0) continue;
          src = static_cast<const T*>(a.key) + token * a.key_token + (h - a.heads) * a.key_head;
          dst = static_cast<T*>(a.key_cache) + s_key[t] + (h - a.heads) * a.kc_head;
        }
        turn_unit<T, LAYOUT, WHOLE>(src, dst, u - h * a.turned, a.half, a.dim, cs, sn, zero);
      } else {
        if (s_value[t] < 0) continue;
        u -= rows;
        const int h = a.by_plain(u);
        copy_unit<T, WHOLE>(
            static_cast<const T*>(a.value) + token * a.value_token + h * a.value_head,
            static_cast<T*>(a.value_cache) + s_value[t] + h * a.vc_head,
            (u - h * a.plain) * Chunk<T>::N, a.dim, false);
      }
    }
  }
}

template <typename T, int LAYOUT, bool WHOLE>
const void* kernel_of(bool append) {
  return append ? reinterpret_cast<const void*>(&rotate_rows<T, LAYOUT, WHOLE, true>)
                : reinterpret_cast<const void*>(&rotate_rows<T, LAYOUT, WHOLE, false>);
}

template <typename T>
const void* kernel_of(int64_t layout, bool whole, bool append) {
  if (layout == TG_HALF)
    return whole ? kernel_of<T, TG_HALF, true>(append) : kernel_of<T, TG_HALF, false>(append);
  return whole ? kernel_of<T, TG_INTERLEAVED, true>(append)
               : kernel_of<T, TG_INTERLEAVED, false>(append);
}

int enqueue(Rows a, int64_t dtype, int64_t layout, bool append, const char* what,
            hipStream_t stream) {
  const int n = dtype == TG_F32 ? 4 : 8;
  const bool halves = layout == TG_HALF;
  a.plain = (a.dim + n - 1) / n;
  a.turned = halves ? (a.half + n - 1) / n + (a.dim - 2 * a.half + n - 1) / n : a.plain;
  a.per_token = (a.heads + a.kv_heads) * a.turned + a.kv_heads * a.plain;
  a.by_turned = Div(a.turned);
  a.by_plain = Div(a.plain);
  a.by_token = Div(a.per_token);
  a.by_page = Div(append ? a.page : 1);
  const bool whole = a.dim % n == 0 && (!halves || a.half % n == 0);
  // Workgroups of one token fill the chip best while there are few tokens, and where a token's
  // heads are work for all threads; else four share a workgroup's start.  16384 tokens of 40
  // heads of 128: 59 us by one, 63 by four; of 4 heads: 13.2 and 7.7.  An append looks up its
  // place first: 4096 tokens of 32 and 8 heads 19.1 and 17.9, 16384 77.7 and 79.1.
  const int tokens =
      a.tokens < 4096 || (!append && a.per_token >= kThreads) ? 1 : kMostTokens;
  const void* k = dtype == TG_F32   ? kernel_of<float>(layout, whole, append)
                  : dtype == TG_F16 ? kernel_of<_Float16>(layout, whole, append)
                                    : kernel_of<__bf16>(layout, whole, append);
  int n_tokens = tokens;
  void* args[] = {&a, &n_tokens};
  const hipError_t e = hipLaunchKernel(k, dim3((a.tokens + tokens - 1) / tokens), dim3(kThreads),
                                       args, 0, stream);
  return e == hipSuccess ? 0 : hip_failed(e, what);
}

// The checks that both entries share; 0 or a status.
int check(const char* what, int64_t dtype, int64_t tokens, int64_t heads, int64_t dim,
          int64_t rotary, int64_t layout) {
  if (dtype < TG_BF16 || dtype > TG_F32) return refuse(-1, what, "unknown dtype", dtype);
  if (layout != TG_HALF && layout != TG_INTERLEAVED)
    return refuse(-1, what, "unknown layout", layout);
  if (tokens < 0 || heads < 0)
    return refuse(-1, what, "negative size", tokens < 0 ? tokens : heads);
  if (dim < 1 || dim > kMaxDim) return refuse(-1, what, "dim must be 1 to 1024", dim);
  if (rotary < 0 || rotary > dim || rotary % 2)
    return refuse(-1, what, "rotary must be even and at most dim", rotary);
  if (tokens > 0x7FFFFF) return refuse(-2, what, "more than 8388607 tokens in one launch", tokens);
  if (heads > 0x10000) return refuse(-2, what, "more than 65536 heads", heads);
  return 0;
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" __attribute__((visibility("default"))) int launch_rope(const tg_rope* r, void* stream) {
  const char* what = "launch_rope";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (const int rc = check(what, r->dtype, r->tokens, r->heads, r->dim, r->rotary, r->layout))
    return rc;
  if (r->sign != 1 && r->sign != -1) return refuse(-1, what, "sign must be 1 or -1", r->sign);
  if (r->tokens == 0 || r->heads == 0) return 0;
  const Operand x = {"x", r->x, 3, {r->tokens, r->heads, r->dim}, {r->x_token, r->x_head, 1}};
  const Operand y = {"out", r->y, 3, {r->tokens, r->heads, r->dim}, {r->y_token, r->y_head, 1}};
  if (const int rc = once(what, y)) return rc;
  if (!same(y, x))
    if (const int rc = apart(what, y, x, r->dtype == TG_F32 ? 4 : 2)) return rc;
  if (!r->x || !r->y || !r->positions || (r->rotary && !r->frequency))
    return refuse(-1, what, "null array", r->tokens);
  Rows a = {};
  a.x = r->x;
  a.y = r->y;
  a.x_token = r->x_token;
  a.x_head = r->x_head;
  a.y_token = r->y_token;
  a.y_head = r->y_head;
  a.frequency = r->frequency;
  a.positions = r->positions;
  a.tokens = static_cast<int>(r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.dim = static_cast<int>(r->dim);
  a.half = static_cast<int>(r->rotary / 2);
  a.sign = static_cast<int>(r->sign);
  a.magnitude = static_cast<float>(r->magnitude);
  return enqueue(a, r->dtype, r->layout, false, what, static_cast<hipStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) int launch_paged_append(const tg_paged_append* r,
                                                                          void* stream) {
  const char* what = "launch_paged_append";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (const int rc = check(what, r->dtype, r->tokens, r->heads, r->dim, r->rotary, r->layout))
    return rc;
  if (r->kv_heads < 1 || r->kv_heads > 0x10000)
    return refuse(-1, what, "kv_heads must be 1 to 65536", r->kv_heads);
  if (r->sequences < 0 || r->sequences > kMaxSequences)
    return refuse(-1, what, "sequences must be 0 to 2^30", r->sequences);
  if (r->page < 1 || r->page > 0x7FFFFFFF)
    return refuse(-1, what, "page must be 1 to 2^31 - 1", r->page);
  if (r->pages < 0 || r->n_indices < 0) return refuse(-1, what, "negative size", r->pages);
  if (!r->query_indptr && r->tokens > r->sequences)
    return refuse(-1, what, "more tokens than sequences without query_indptr", r->tokens);
  if (r->tokens == 0) return 0;
  // What is written shares no memory with what else is written, or with the rows of new tokens.
  // (Rows of new tokens may stand in the caches themselves: which slots are written is known on
  // the device alone.)
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
  // one cache for both holds the same values twice where nothing is turned and value is key
  if (!(r->rotary == 0 && same(key, value) && same(kc, vc)))
    if (const int rc = apart(what, vc, kc, bytes)) return rc;
  if (!r->key || !r->value || !r->key_cache || !r->value_cache || !r->indptr || !r->lengths ||
      (r->n_indices && !r->indices) || (r->heads && (!r->query || !r->query_out)) ||
      (r->rotary && !r->frequency))
    return refuse(-1, what, "null array", r->tokens);
  Rows a = {};
  a.x = r->query;
  a.y = r->query_out;
  a.x_token = r->query_token;
  a.x_head = r->query_head;
  a.y_token = r->out_token;
  a.y_head = r->out_head;
  a.frequency = r->frequency;
  a.tokens = static_cast<int>(r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.dim = static_cast<int>(r->dim);
  a.half = static_cast<int>(r->rotary / 2);
  a.sign = 1;
  a.magnitude = static_cast<float>(r->magnitude);
  a.key = r->key;
  a.value = r->value;
  a.key_cache = r->key_cache;
  a.value_cache = r->value_cache;
  a.key_token = r->key_token;
  a.key_head = r->key_head;
  a.value_token = r->value_token;
  a.value_head = r->value_head;
  a.kc_page = r->kc_page;
  a.kc_slot = r->kc_slot;
  a.kc_head = r->kc_head;
  a.vc_page = r->vc_page;
  a.vc_slot = r->vc_slot;
  a.vc_head = r->vc_head;
  a.indptr = r->indptr;
  a.indices = r->indices;
  a.lengths = r->lengths;
  a.query_indptr = r->query_indptr;
  a.sequences = static_cast<int>(r->sequences);
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.page = static_cast<int>(r->page);
  a.pages = r->pages;
  a.n_indices = r->n_indices;
  a.offset = r->offset;
  return enqueue(a, r->dtype, r->layout, true, what, static_cast<hipStream_t>(stream));
}
