/*
 * tilegen_attention.h -- libtgattn.so (tilegen_amd/csrc/attention/): attention over a paged
 * cache whose page table is a CSR structure, for gfx950.
 *
 * No counterpart in the reference.  Three operators, each enqueued on `stream` (NULL = the
 * null stream) without waiting:
 *
 *   launch_rope              rotary positions, forward and backward
 *   launch_paged_append      new keys and values into their sequences' pages, keys (and the
 *                            queries) rotated on the way
 *   launch_prefix_attention  attention of a batch whose sequences share a prefix, over the
 *                            prefix's pages and each sequence's own
 *
 * Every pointer is a device pointer of the caller's; nothing is allocated.  Strides count
 * elements; the elements of a head are contiguous, and no two of an output share memory.  dtype is 0 (bfloat16), 1 (float16) or 2
 * (float32).  Structures hold 8-byte fields only, so that a binding packs them flat.
 *
 * Returns 0 on success, -1 for a bad argument, -2 for a size beyond one launch, or a hipError_t;
 * the message is in libtgrt's tg_last_error().  What the device arrays hold is checked where it
 * is used: a page outside the cache, a position outside a sequence's pages or a row pointer
 * outside `indices` is never read or written (see each operator).
 */
#ifndef TILEGEN_ATTENTION_H
#define TILEGEN_ATTENTION_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { TG_BF16 = 0, TG_F16 = 1, TG_F32 = 2 };
enum { TG_HALF = 0, TG_INTERLEAVED = 1 };

/* y[t,h] = x[t,h] with its pairs turned by sign * positions[t] * frequency[i] and multiplied by
 * magnitude; a pair is (i, i + rotary/2) (TG_HALF) or (2i, 2i + 1) (TG_INTERLEAVED); elements
 * from `rotary` on are copied.  sign -1 is the backward pass (the transposed map).  y may be x
 * (the same strides); it may not overlap it otherwise. */
typedef struct {
  const void* x;
  void* y;
  const int64_t* positions; /* [tokens] */
  const double* frequency;  /* [rotary / 2], radians per position */
  int64_t dtype, tokens, heads, dim, rotary, layout;
  int64_t x_token, x_head, y_token, y_head; /* strides */
  double magnitude;
  int64_t sign;
} tg_rope;

int launch_rope(const tg_rope* a, void* stream);

/* Sequence b's n new tokens, rows query_indptr[b] .. query_indptr[b+1] of key and value (row b
 * alone where query_indptr is NULL), go to positions lengths[b] - n .. lengths[b] - 1 of the
 * pages indices[indptr[b]:indptr[b+1]]: position p to slot p % page of the page numbered
 * p / page.  Keys are turned at offset + p first, and so are the same rows of `query` into
 * query_out (heads = 0: none).  rotary = 0: nothing is turned.  A token whose position falls
 * outside its sequence's pages, or whose page is outside the cache, is not written; one before
 * query_indptr[0] or past query_indptr[sequences] belongs to no sequence (slices of a larger
 * batch's row pointers, or a padded batch): it is not written and its query comes back zero.
 * query_out may be query (the same strides); it may not overlap it otherwise, or key, value or a
 * cache, and the caches may not overlap one another (they may be one where rotary is 0 and value
 * is key).  Rows that stand in the caches may not be among the slots that are written. */
typedef struct {
  const void *key, *value, *query;
  void *key_cache, *value_cache, *query_out;
  const int64_t *indptr, *indices, *lengths, *query_indptr;
  const double* frequency;
  int64_t dtype, tokens, sequences, heads, kv_heads, dim, rotary, layout;
  int64_t pages, page, n_indices, offset;
  int64_t key_token, key_head, value_token, value_head;
  int64_t query_token, query_head, out_token, out_head;
  int64_t kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  double magnitude;
} tg_paged_append;

int launch_paged_append(const tg_paged_append* a, void* stream);

/* out[t,h] = softmax(scale q[t,h] . k) v over the first prefix_length keys of the pages
 * `prefix`, which every token sees, and those of its sequence's own pages up to its own
 * position: with n new tokens (as above), token j sees positions 0 .. lengths[b] - n + j.  Query
 * head h reads kv head h / (heads / kv_heads).  lse (may be NULL): the logarithm of each row's
 * sum of exponentials, [tokens, heads].  A row that sees no key, or whose scores are all -inf,
 * gives 0 and -inf, and so does one of no sequence (as above).  A key whose page is outside the
 * cache counts as hidden.
 *
 * max_query and max_length are the host's bounds on n and lengths[b]; they size the launch,
 * and larger values on the device are still right.  workspace holds
 * prefix_attention_workspace(a) bytes, 16-byte aligned, until the kernels have run; calls
 * that overlap need one each.  out may be query (the same strides); it may not overlap it
 * otherwise, or a cache. */
typedef struct {
  const void *query, *key_cache, *value_cache;
  const int64_t *prefix, *indptr, *indices, *lengths, *query_indptr;
  void* out;
  float* lse;
  void* workspace;
  int64_t workspace_bytes;
  int64_t dtype, tokens, sequences, heads, kv_heads, dim;
  int64_t pages, page, n_prefix, prefix_length, n_indices, max_query, max_length;
  int64_t query_token, query_head, out_token, out_head;
  int64_t kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  double scale;
} tg_prefix_attention;

/* Bytes, or a negative status for arguments that launch_prefix_attention refuses. */
int64_t prefix_attention_workspace(const tg_prefix_attention* a);
int launch_prefix_attention(const tg_prefix_attention* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TILEGEN_ATTENTION_H */
