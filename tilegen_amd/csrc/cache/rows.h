// How the heads of queries and keys lie over the lanes of a wave in norms: 64 / G rows side by
// side, G lanes each, every lane with NP pairs of elements, in registers from their load to their
// store.  A row's sums are then a few exchanges between neighbouring lanes, and every value
// is read once.
#pragma once

#include "../attention/parts.h"
#include "cache.h"

namespace tg {

constexpr int kMostDim = 256;

// v + the same lane's value in another order of its 16 lanes
template <int ORDER>
__device__ __forceinline__ float plus(float v) {
  const int x = __builtin_bit_cast(int, v);
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, x, ORDER, 0xF, 0xF, true));
}

// The sum over each G lanes, in all of them.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(G == 4 || G == 8 || G == 16 || G == 32 || G == 64, "");
  v = plus<0xB1>(v);                    // neighbours: lanes 1 0 3 2
  v = plus<0x4E>(v);                    // pairs: lanes 2 3 0 1
  if (G >= 8) v = plus<0x141>(v);       // quads: the mirror of each 8
  if (G >= 16) v = plus<0x140>(v);      // the mirror of each 16
  if (G >= 32) {
    const Both q = quarters(v);
    v = q.a + q.b;
  }
  if (G == 64) {
    const Both h = halves(v);
    v = h.a + h.b;
  }
  return v;
}

// Rows in 16-byte chunks.  Halves: a lane's unit is a chunk of the first half with its partners, or
// a chunk of what is not turned.  Interleaved: a chunk, whose pairs are neighbours.  EDGE: a part of
// the row that does not end with a chunk has a last one that reaches back over the one before; the
// pairs that both have count once (and are written twice, the same).
template <typename T, int LAYOUT, int LANES, bool EDGE>
struct Whole {
  static constexpr int G = LANES, N = Chunk<T>::N, NP = LAYOUT == TG_HALF ? N : N / 2;
  int at, partner, pair;    // elements; the first pair's number; partner -1: none
  int again;                // pairs that the unit before has
  bool active;
  static __host__ __device__ __forceinline__ int chunks(int n) {
    return EDGE ? (n + N - 1) / N : n / N;
  }
  __device__ __forceinline__ Whole(int unit, int dim, int half, int)
      : Whole(unit, unit - chunks(half), dim, half, true) {}
  // past: the units of pairs of halves, negative for those
  __device__ __forceinline__ Whole(int unit, int past, int dim, int half, bool)
      : Whole(LAYOUT != TG_HALF || past < 0 ? unit * N : 2 * half + past * N,
              LAYOUT != TG_HALF || past >= 0 ? dim : half, LAYOUT == TG_HALF && past < 0, half,
              LAYOUT != TG_HALF ? unit < chunks(dim) : past < chunks(dim - 2 * half)) {}
  __device__ __forceinline__ Whole(int from, int end, bool two, int half, bool active)
      : at(EDGE && from + N > end ? end - N : from),
        partner(LAYOUT != TG_HALF ? 0 : two ? half + at : -1),
        pair(LAYOUT != TG_HALF ? at / 2 : two ? at : half),
        again(LAYOUT != TG_HALF ? (from - at) / 2 : from - at),
        active(active) {}
  static int units(int dim, int half) {
    return LAYOUT == TG_HALF ? chunks(half) + chunks(dim - 2 * half) : chunks(dim);
  }
  __device__ __forceinline__ bool counts(int i) const { return !EDGE || i >= again; }
  template <typename S>
  struct Raw {
    typename Loose<S, N>::Vec a, b;
    __device__ __forceinline__ float first(int i) const {
      return static_cast<float>(LAYOUT == TG_HALF ? a[i] : a[2 * i]);
    }
    __device__ __forceinline__ float second(int i) const {
      return static_cast<float>(LAYOUT == TG_HALF ? b[i] : a[2 * i + 1]);
    }
    __device__ __forceinline__ void set(int i, float x, float y) {
      if (LAYOUT == TG_HALF) {
        a[i] = static_cast<S>(x);
        b[i] = static_cast<S>(y);
      } else {
        a[2 * i] = static_cast<S>(x);
        a[2 * i + 1] = static_cast<S>(y);
      }
    }
  };
  template <typename S>
  __device__ __forceinline__ void load(const S* row, bool live, Raw<S>& r) const {
    r.a = r.b = typename Loose<S, N>::Vec(S(0));
    if (!live || !active) return;
    r.a = Loose<S, N>::load(row + at);
    if (LAYOUT == TG_HALF && partner >= 0) r.b = Loose<S, N>::load(row + partner);
  }
  __device__ __forceinline__ void store(T* row, const Raw<T>& r) const {
    if (!active) return;
    Loose<T, N>::store(row + at, r.a);
    if (LAYOUT == TG_HALF && partner >= 0) Loose<T, N>::store(row + partner, r.b);
  }
  // the number of pair i, at least `half` where it is not turned
  __device__ __forceinline__ int turn(int i) const { return pair + i; }
  // where element (first or second) of pair i of `unit` stands in its row, or -1
  __device__ __forceinline__ int element(int i, bool second) const {
    if (!active || !counts(i) || (LAYOUT == TG_HALF && second && partner < 0)) return -1;
    return LAYOUT == TG_HALF ? (second ? partner : at) + i : at + 2 * i + second;
  }
};

// Any row up to 256 elements, one by one: lane l has the pairs l, l + 64, ..; what is not turned
// counts on as pairs of one.
template <typename T>
struct Ragged {
  static constexpr int G = 64, NP = kMostDim / 64;
  int lane, dim, half, layout;
  __device__ __forceinline__ Ragged(int unit, int dim, int half, int layout)
      : lane(unit), dim(dim), half(half), layout(layout) {}
  __device__ __forceinline__ bool counts(int) const { return true; }
  template <typename S>
  struct Raw {
    typedef S Vec __attribute__((ext_vector_type(NP)));
    Vec a, b;
    __device__ __forceinline__ float first(int i) const { return static_cast<float>(a[i]); }
    __device__ __forceinline__ float second(int i) const { return static_cast<float>(b[i]); }
    __device__ __forceinline__ void set(int i, float x, float y) {
      a[i] = static_cast<S>(x);
      b[i] = static_cast<S>(y);
    }
  };
  __device__ __forceinline__ int turn(int i) const { return lane + 64 * i; }
  __device__ __forceinline__ int element(int i, bool second) const {
    const int p = turn(i);
    if (p < half) return layout == TG_HALF ? (second ? half + p : p) : 2 * p + second;
    const int at = half + p;
    return second || at >= dim ? -1 : at;
  }
  template <typename S>
  __device__ __forceinline__ void load(const S* row, bool live, Raw<S>& r) const {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int x = element(i, false), y = element(i, true);
      r.a[i] = live && x >= 0 ? row[x] : S(0);
      r.b[i] = live && y >= 0 ? row[y] : S(0);
    }
  }
  __device__ __forceinline__ void store(T* row, const Raw<T>& r) const {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int x = element(i, false), y = element(i, true);
      if (x >= 0) row[x] = r.a[i];
      if (y >= 0) row[y] = r.b[i];
    }
  }
};

// A norm's weight for one row: NP pairs of 32-bit values.
template <int NP>
struct Pairs {
  typedef float Vec __attribute__((ext_vector_type(NP)));
  Vec a, b;
};
template <typename T, typename P>
__device__ __forceinline__ Pairs<P::NP> weight_of(const P& place, const void* weight, bool wide,
                                                  i64 at, bool live) {
  Pairs<P::NP> w = {typename Pairs<P::NP>::Vec(1.f), typename Pairs<P::NP>::Vec(1.f)};
  if (!weight) return w;
  if (sizeof(T) == 4 || wide) {
    typename P::template Raw<float> r;
    place.load(static_cast<const float*>(weight) + at, live, r);
#pragma unroll
    for (int i = 0; i < P::NP; ++i) {
      w.a[i] = r.first(i);
      w.b[i] = r.second(i);
    }
  } else {
    typename P::template Raw<T> r;
    place.load(static_cast<const T*>(weight) + at, live, r);
#pragma unroll
    for (int i = 0; i < P::NP; ++i) {
      w.a[i] = r.first(i);
      w.b[i] = r.second(i);
    }
  }
  return w;
}

// (cosine, sine) of f turns, |f| <= 1/2: the nearest quarter turn is taken off, exactly, and what is
// left, at most pi/4, goes through the two Taylor series, whose next terms are under 2^-29.
__device__ __forceinline__ float2 turned_by(float f) {
  const float n = rintf(4.f * f);
  const float x = (f - 0.25f * n) * 6.28318530717958647692f, y = x * x;
  const float s = x * (1.f + y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 +
                                                                   y * (1.f / 362880)))));
  const float c = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 +
                                                          y * (1.f / 40320 -
                                                               y * (1.f / 3628800)))));
  const int quarter = static_cast<int>(n) & 3;
  const float u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
  return make_float2(quarter == 1 || quarter == 2 ? -u : u, quarter & 2 ? -v : v);
}

// The cosines and sines of one position's pairs, by a wave into LDS of its own.  Angles are taken
// in 64 bits as turns, of which the fraction is exact to 2^-25 of itself in 32.
struct Turns {
  float c[kMostDim / 2], s[kMostDim / 2];
};
__device__ __forceinline__ void turns_of(Turns& t, i64 position, const double* frequency, int half,
                                         float magnitude) {
  constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
  __builtin_amdgcn_wave_barrier();    // reads of the last position's are done: a wave's are in order
  for (int i = threadIdx.x & 63; i < half; i += 64) {
    const double turns = static_cast<double>(position) * (frequency[i] * kPerTurn);
    const float2 cs = turned_by(static_cast<float>(turns - rint(turns)));
    t.c[i] = cs.x * magnitude;
    t.s[i] = cs.y * magnitude;
  }
  __builtin_amdgcn_wave_barrier();
}

// How rows are cut: whole chunks, chunks that reach back, or single elements; and lanes of a row.
enum Cut { kWhole, kEdge, kRagged };
struct Lanes {
  Cut cut;
  int lanes;
};
inline Lanes lanes_of(int64_t dtype, int dim, int half, int64_t layout) {
  const int n = dtype == TG_F32 ? 4 : 8, rest = dim - 2 * half;
  const auto up = [n](int x) { return (x + n - 1) / n; };
  int units = up(dim);
  Cut cut = dim % n == 0 ? kWhole : dim % 2 == 0 && dim >= n ? kEdge : kRagged;
  if (layout == TG_HALF) {
    units = up(half) + up(rest);
    cut = half % n == 0 && rest % n == 0 ? kWhole
          : (half == 0 || half >= n) && (rest == 0 || rest >= n) ? kEdge
                                                                 : kRagged;
  }
  if (cut == kRagged) return {cut, 64};
  return {cut, units <= 4 ? 4 : units <= 8 ? 8 : units <= 16 ? 16 : units <= 32 ? 32 : 64};
}

// The checks that the norms share; 0 or a status.
inline int check_norm(const char* what, int64_t dtype, int64_t weight_dtype, int64_t tokens,
                      int64_t heads, int64_t kv_heads, int64_t dim, int64_t rotary,
                      int64_t layout, double epsilon) {
  if (dtype < TG_BF16 || dtype > TG_F32) return refuse(-1, what, "unknown dtype", dtype);
  if (weight_dtype != dtype && weight_dtype != TG_F32)
    return refuse(-1, what, "weights must be of the heads' type or float32", weight_dtype);
  if (layout != TG_HALF && layout != TG_INTERLEAVED)
    return refuse(-1, what, "unknown layout", layout);
  if (tokens < 0 || heads < 0 || kv_heads < 0) return refuse(-1, what, "negative size", tokens);
  if (dim < 1 || dim > kMostDim) return refuse(-1, what, "dim must be 1 to 256", dim);
  if (rotary < 0 || rotary > dim || rotary % 2)
    return refuse(-1, what, "rotary must be even and at most dim", rotary);
  if (!(epsilon >= 0) || !(epsilon < 1e30))
    return refuse(-1, what, "epsilon must be at least 0 and finite", 0);
  if (tokens > 0x7FFFFF) return refuse(-2, what, "more than 8388607 tokens in one launch", tokens);
  if (heads > 0x10000 || kv_heads > 0x10000)
    return refuse(-2, what, "more than 65536 heads", heads > kv_heads ? heads : kv_heads);
  return 0;
}

}  // namespace tg
