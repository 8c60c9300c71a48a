// What the kernels of libtgcache share: a sequence's pages, and the overlap of operands whose
// elements differ in size.
#pragma once

#include "../attention/attention.h"
#include "tilegen_cache.h"

namespace tg {

// A page table and the tokens that a call brings.
struct Table {
  const int64_t *indptr, *indices, *lengths, *ends;   // ends: query_indptr or null
  i64 pages, n_indices;
  int tokens, sequences, page;
  Div by_page;
};

// Sequence b: its new tokens (rows first .. first + count), the keys that its pages hold, and how
// many of them stood there before.
struct Own {
  int first, count, before, keys;
  const int64_t* list;
};

__device__ __forceinline__ Own own_of(const Table& t, int b) {
  Own s;
  i64 first = b, last = b + 1;
  if (t.ends) {
    first = t.ends[b];
    last = t.ends[b + 1];
    first = first < 0 ? 0 : first > t.tokens ? t.tokens : first;
    last = last < first ? first : last > t.tokens ? t.tokens : last;
  }
  s.first = static_cast<int>(first);
  s.count = static_cast<int>(last - first);
  i64 begin = t.indptr[b], end = t.indptr[b + 1];
  begin = begin < 0 ? 0 : begin > t.n_indices ? t.n_indices : begin;
  end = end < begin ? begin : end > t.n_indices ? t.n_indices : end;
  s.list = t.indices + begin;
  i64 length = t.lengths[b];
  length = length < 0 ? 0 : length > INT32_MAX / 2 ? INT32_MAX / 2 : length;
  const i64 held = (end - begin) * t.page;
  s.before = static_cast<int>(length) - s.count;
  s.keys = static_cast<int>(length < held ? length : held);
  return s;
}

// The sum of a value over a wave's lanes up to each.
__device__ __forceinline__ int upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // from 1, 2, 4, 8 lanes below,
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);   // within 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // the last lane of each 16 to
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // the next, of 32 to the other
  return v;
}

// N elements that stand anywhere.
template <typename S, int N>
struct Loose {
  typedef S Vec __attribute__((ext_vector_type(N)));
  struct __attribute__((packed, aligned(sizeof(S)))) Held {
    Vec v;
  };
  static __device__ __forceinline__ Vec load(const S* p) {
    return reinterpret_cast<const Held*>(p)->v;
  }
  static __device__ __forceinline__ void store(S* p, Vec v) {
    reinterpret_cast<Held*>(p)->v = v;
  }
};

constexpr int64_t kMostKeys = INT32_MAX / 2;
constexpr int64_t kMostStride = int64_t(1) << 60;
constexpr int64_t kMostGroups = 0xFFFFFF;   // workgroups of a launch

// An operand of 4-byte elements in units of 2 bytes, to compare with others of 2.
inline Operand in_halves(Operand x) {
  for (int i = 0; i < x.axes; ++i) x.stride[i] *= 2;
  x.size[x.axes] = 2;
  x.stride[x.axes++] = 1;
  return x;
}

// The checks of a page table; 0 or a status.
inline int check_table(const char* what, int64_t sequences, int64_t pages, int64_t page,
                       int64_t n_indices, int64_t max_length) {
  if (sequences < 0 || pages < 0 || n_indices < 0 || max_length < 0)
    return refuse(-1, what, "negative size", 0);
  if (page < 1 || page > INT32_MAX) return refuse(-1, what, "page must be 1 to 2^31 - 1", page);
  if (pages > INT32_MAX) return refuse(-2, what, "more than 2^31 pages", pages);
  if (sequences > (1 << 24)) return refuse(-2, what, "more than 2^24 sequences", sequences);
  if (max_length > kMostKeys) return refuse(-2, what, "more than 2^30 keys", max_length);
  return 0;
}

inline int check_strides(const char* what, const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] > kMostStride || s[i] < -kMostStride)
      return refuse(-2, what, "a stride of more than 2^60", s[i]);
  return 0;
}

inline hipError_t launch(const void* kernel, int64_t groups, int threads, void** args,
                         hipStream_t stream) {
  return hipLaunchKernel(kernel, dim3(static_cast<unsigned>(groups)), dim3(threads), args, 0,
                         stream);
}

}  // namespace tg
