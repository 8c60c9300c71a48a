// The parts that prefix attention is split into, and what its kernels and host code share.
#pragma once

#include "attention.h"

namespace tg {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct Attention {
  const void *q, *k, *v;
  const int64_t *prefix, *indptr, *indices, *lengths, *ends;  // ends: query_indptr or null
  void* out;
  float* lse;
  float* part;        // [slots, tokens * heads, dim]: each part's sums, not yet divided
  float2* part_ml;    // [slots, tokens * heads]: what its exponents are taken against, and its sum
  i64 q_token, q_head, o_token, o_head;
  i64 kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  i64 pages, n_indices;
  int tokens, sequences, heads, kv_heads, group, dim, page, prefix_length;
  float scale;        // scale * log2 e
  Div by_group, by_page;
  // the prefix's slots come first, then the own pages'
  int prefix_splits, prefix_chunk, prefix_tiles;
  int own_splits, own_chunk, own_tiles;
  int slots;
  int prefix_eights, own_eights;    // workgroups, in eights
  int even;           // the wide kernel's scalar addresses hold (wide.h)
  int sorted;         // own parts go from the longest sequence to the shortest (parts.h)
};

// The new tokens of sequence b and the keys of its own pages.
struct Sequence {
  int first, count;   // its tokens
  int before;         // token j sees before + j + 1 keys, 0 to keys
  int keys;           // keys that its pages hold
  const int64_t* list;
};

__device__ __forceinline__ Sequence sequence(const Attention& a, int b) {
  Sequence s;
  i64 first = b, last = b + 1;
  if (a.ends) {
    first = a.ends[b];
    last = a.ends[b + 1];
    first = first < 0 ? 0 : first > a.tokens ? a.tokens : first;
    last = last < first ? first : last > a.tokens ? a.tokens : last;
  }
  s.first = static_cast<int>(first);
  s.count = static_cast<int>(last - first);
  i64 begin = a.indptr[b], end = a.indptr[b + 1];
  begin = begin < 0 ? 0 : begin > a.n_indices ? a.n_indices : begin;
  end = end < begin ? begin : end > a.n_indices ? a.n_indices : end;
  s.list = a.indices + begin;
  i64 length = a.lengths[b];
  length = length < 0 ? 0 : length > INT32_MAX / 2 ? INT32_MAX / 2 : length;
  const i64 held = (end - begin) * a.page;
  s.before = static_cast<int>(length) - s.count;
  s.keys = static_cast<int>(length < held ? length : held);
  return s;
}

// Keys of its own pages that token j of the sequence sees.
__device__ __forceinline__ int seen(const Sequence& s, int j) {
  const int n = s.before + j + 1;
  return n < 0 ? 0 : n > s.keys ? s.keys : n;
}

// Parts of a row's own pages: those whose first key it sees; the last takes all that is left.
__device__ __forceinline__ int own_parts(const Attention& a, int keys) {
  const int n = (keys + a.own_chunk - 1) / a.own_chunk;
  return n < a.own_splits ? n : a.own_splits;
}

// Enqueue the parts, or the whole of a small call, for one type and padded head size.
template <typename T, int DP>
hipError_t launch_parts(const Attention& a, int prefix_rows, int own_rows, hipStream_t stream);
template <typename T, int DP>
hipError_t launch_whole(const Attention& a, hipStream_t stream);

}  // namespace tg
