/*
 * tilegen_cache.h -- libtgcache.so (tilegen_amd/csrc/cache/): a paged cache of bounded length, for
 * gfx950, beside include/tilegen_attention.h.
 *
 * No counterpart in the reference.  Each operator is enqueued on `stream` (NULL = the null
 * stream) without waiting:
 *
 *   launch_norm_rope            root mean square norms of query and key heads, turned in the same
 *                               pass
 *   launch_norm_rope_backward   their gradients, and the weights'
 *   launch_paged_append_normed  launch_paged_append with those norms, at positions that count
 *                               tokens that are no longer there
 *   launch_attention_weights    the attention weight that each cached key receives
 *   launch_paged_evict          all but the heaviest tokens leave their sequences' pages
 *
 * Every pointer is a device pointer of the caller's; nothing is allocated.  Strides count
 * elements; the elements of a head are contiguous, and no two of an output share memory.  dtype
 * is 0 (bfloat16), 1 (float16) or 2 (float32).  Structures hold 8-byte fields only, so that a
 * binding packs them flat.
 *
 * Returns 0 on success, -1 for a bad argument, -2 for a size beyond one launch, or a hipError_t;
 * the message is in libtgrt's tg_last_error().  What the device arrays hold is checked where it
 * is used: a page outside the cache, a position outside a sequence's pages or a row pointer
 * outside `indices` is never read or written.  A page belongs to one sequence alone where a call
 * writes to it.
 */
#ifndef TILEGEN_CACHE_H
#define TILEGEN_CACHE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* query_out[t,h] = turn(x r w), x = query[t,h], r = (mean of x^2 + epsilon)^-1/2, w = query_weight
 * (NULL: ones; of head h at query_weight + h query_weight_head, stride 0: one for all heads), and
 * the same for key.  turn is launch_rope's: pairs of the first `rotary` elements by positions[t] *
 * frequency[i], times magnitude.  Weights are of weight_dtype: dtype or 2.  Each output may be its
 * own input (the same strides); it may not overlap the operands otherwise.  heads or kv_heads may
 * be 0 (its arrays NULL). */
typedef struct {
  const void *query, *key;
  void *query_out, *key_out;
  const void *query_weight, *key_weight;
  const int64_t* positions; /* [tokens]; NULL where rotary is 0 */
  const double* frequency;  /* [rotary / 2], radians per position */
  int64_t dtype, weight_dtype, tokens, heads, kv_heads, dim, rotary, layout;
  int64_t query_token, query_head, key_token, key_head;
  int64_t qout_token, qout_head, kout_token, kout_head;
  int64_t query_weight_head, key_weight_head;
  double magnitude, epsilon;
} tg_norm_rope;

int launch_norm_rope(const tg_norm_rope* a, void* stream);

/* The gradients of launch_norm_rope from those of its outputs, grad_query and grad_key: of query
 * and key into query_out and key_out, of the weights into query_weight_out and key_weight_out
 * (contiguous, of weight_dtype: [dim], or [heads, dim] where the stride is not 0; NULL: not
 * wanted), each summed in 32 bits in an order that the sizes alone decide; zeros where there are no
 * tokens or no heads.  query_out may be grad_query or query (the same strides), and key_out
 * likewise.  workspace holds norm_rope_backward_workspace(a) bytes, 16-byte aligned, until the
 * kernels have run; calls that overlap need one each. */
typedef struct {
  const void *grad_query, *grad_key, *query, *key;
  void *query_out, *key_out, *query_weight_out, *key_weight_out;
  const void *query_weight, *key_weight;
  const int64_t* positions;
  const double* frequency;
  void* workspace;
  int64_t workspace_bytes;
  int64_t dtype, weight_dtype, tokens, heads, kv_heads, dim, rotary, layout;
  int64_t grad_query_token, grad_query_head, grad_key_token, grad_key_head;
  int64_t query_token, query_head, key_token, key_head;
  int64_t qout_token, qout_head, kout_token, kout_head;
  int64_t query_weight_head, key_weight_head;
  double magnitude, epsilon;
} tg_norm_rope_backward;

/* Bytes, or a negative status for arguments that launch_norm_rope_backward refuses. */
int64_t norm_rope_backward_workspace(const tg_norm_rope_backward* a);
int launch_norm_rope_backward(const tg_norm_rope_backward* a, void* stream);

/* launch_paged_append (include/tilegen_attention.h), with two additions.  Where `normed` is 1, keys
 * and queries are normed as by launch_norm_rope before they are turned (query_weight, key_weight,
 * epsilon).  Where shift is given, tokens of sequence b are turned at offset + shift[b] + p: shift[b]
 * tokens that came before are no longer in its pages.  The slot is p's all the same.  dim is at
 * most 256. */
typedef struct {
  const void *key, *value, *query;
  void *key_cache, *value_cache, *query_out;
  const int64_t *indptr, *indices, *lengths, *query_indptr, *shift;
  const double* frequency;
  const void *query_weight, *key_weight;
  int64_t dtype, weight_dtype, tokens, sequences, heads, kv_heads, dim, rotary, layout;
  int64_t pages, page, n_indices, offset, normed;
  int64_t key_token, key_head, value_token, value_head;
  int64_t query_token, query_head, out_token, out_head;
  int64_t kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  int64_t query_weight_head, key_weight_head;
  double magnitude, epsilon;
} tg_paged_append_normed;

int launch_paged_append_normed(const tg_paged_append_normed* a, void* stream);

/* weights[slot of p, h] = (p < lengths[b] - n ? decay weights[slot of p, h] : 0) + the sum of
 * exp(scale q . k - lse) over the n new tokens of sequence b that see position p (as in
 * launch_prefix_attention) and the query heads of kv head h, for every position p of each
 * sequence's own pages.  lse is what that call left: of a row whose logarithm is -inf nothing is
 * added.  A sequence without new tokens keeps its weights as they are.  weights may not overlap
 * the other operands; max_query and max_length as there. */
typedef struct {
  const void* query;
  const float* lse;
  const void* key_cache;
  float* weights;
  const int64_t *indptr, *indices, *lengths, *query_indptr;
  void* workspace;
  int64_t workspace_bytes;
  int64_t dtype, tokens, sequences, heads, kv_heads, dim;
  int64_t pages, page, n_indices, max_query, max_length;
  int64_t query_token, query_head, lse_token, lse_head;
  int64_t kc_page, kc_slot, kc_head, w_page, w_slot, w_head;
  double scale, decay;
} tg_attention_weights;

/* Bytes, or a negative status for arguments that launch_attention_weights refuses. */
int64_t attention_weights_workspace(const tg_attention_weights* a);
int launch_attention_weights(const tg_attention_weights* a, void* stream);

/* Each sequence of L > keep tokens loses all but `keep`, by kv head; L = lengths[b], or what its
 * pages hold where that is less: the first `first` and the last `recent` stay, and of those between
 * the heaviest by `weights` (of equal ones the first; NaN counts as the heaviest).  Kept tokens at
 * positions below front = keep - recent do not move; the others but the last `recent` go, in order,
 * to the positions below front that became free, in order; the last `recent` go to front and on, in
 * order.  kept[b,h,i] is where the token at position i was, -1 where there is none; lengths_out[b] =
 * min(L, keep).  Slots from there on hold anything.  With move_weights the weights move with their
 * tokens; without they are only read, and may share memory.  A slot whose page is outside the cache
 * counts as one of the least weight, and what would come from it or go there does not move.  The
 * caches and weights may not overlap one another; kept and lengths_out are contiguous and overlap
 * nothing. */
typedef struct {
  void *key_cache, *value_cache;
  float* weights;
  const int64_t *indptr, *indices, *lengths;
  int64_t* lengths_out; /* [sequences] */
  int32_t* kept;        /* [sequences, kv_heads, keep] */
  int64_t dtype, sequences, kv_heads, dim, pages, page, n_indices, max_length;
  int64_t keep, recent, first, move_weights;
  int64_t kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, w_page, w_slot, w_head;
} tg_paged_evict;

int launch_paged_evict(const tg_paged_evict* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TILEGEN_CACHE_H */
