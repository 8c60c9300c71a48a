// Eviction by weight (launch_paged_evict): which tokens stay is decided for each sequence and kv
// head by one workgroup, then workgroups for slices of each head move what has to.
//
// Of the C candidates between the first and the recent tokens the n heaviest stay.  Weights map to
// whole numbers of the same order, which threads hold in registers, and the n-th largest is found
// digit by digit from the top, by counting.  Ties at it go to the lowest positions.  Moves:
// tokens that stay below `front` are left alone; the others are as many as the holes there, and
// both lists are taken in order.  No place is both a source and a target of those, so they go in
// any order; then the recent tokens go down, chunk by chunk, each read whole before it is
// written.
//
// 256 heads of up to 1088 tokens of 128 cut to 1024 (78 MB): 19.6 us, 4 TB/s.  32 heads of up to
// 16384 cut to 2048: 14.1 us to choose, on as many compute units, and 14.6 to move 60 MB, 4.1 TB/s.  Of
// the 14.1 some 60 instructions a key are 6.4 by their issue alone (256 waves of keys on 4 SIMDs at
// 2.4 GHz); lookups, counts in LDS and the waits between the steps of one workgroup are the rest.  9
// heads of up to 210: 11 us, the chain of lookups, two counts, two rankings and the moves' own
// lookups.
#include "cache.h"

namespace tg {
namespace {

struct Evict {
  void *key_cache, *value_cache;
  float* weights;
  int64_t* lengths_out;
  int32_t* kept;
  Table table;
  i64 kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, w_page, w_slot, w_head;
  int kv_heads, dim, keep, recent, first, move_weights;
  int units;              // of 16 bytes, of a row of a cache
  int slices, slice;      // how it is cut, units of each
  int chunks;             // the kept tokens, for fills
  Div by_heads, by_parts, by_row, by_slice, by_last;    // units of a row, of a slice, of the last
};

// Sequence b's pages, as far as its tokens go.
struct Held {
  const int64_t* list;
  int keys;
};
__device__ __forceinline__ Held held_of(const Evict& a, int b) {
  const Table& t = a.table;
  i64 begin = t.indptr[b], end = t.indptr[b + 1];
  begin = begin < 0 ? 0 : begin > t.n_indices ? t.n_indices : begin;
  end = end < begin ? begin : end > t.n_indices ? t.n_indices : end;
  i64 length = t.lengths[b];
  length = length < 0 ? 0 : length > kMostKeys ? kMostKeys : length;
  const i64 room = (end - begin) * t.page;
  return {t.indices + begin, static_cast<int>(length < room ? length : room)};
}

// A sequence's pages, -1 for those outside the cache: from its list, or the first of them from LDS,
// where a lookup does not wait for memory (1024 heads of 1088 tokens 69 us, 73 by the list; 3 to 8%
// with many heads, nothing with few).
struct Far {
  const int64_t* list;
  i64 pages;
  __device__ __forceinline__ i64 operator()(int nth) const {
    const i64 page = list[nth];
    return page >= 0 && page < pages ? page : -1;
  }
};
struct Near {
  const int32_t* near;
  int count;
  Far far;
  __device__ __forceinline__ i64 operator()(int nth) const {
    return nth < count ? near[nth] : far(nth);
  }
};

// A position's page and slot.
struct Place {
  i64 page;
  int slot;
};
template <typename P>
__device__ __forceinline__ Place place_of(const Evict& a, const P& page_of, int p) {
  const int nth = a.table.by_page(p);
  return {page_of(nth), p - nth * a.table.page};
}

// Whole numbers in the order of the weights: 0 for none, the largest for NaN; -0 is 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t x = __builtin_bit_cast(uint32_t, w + 0.f);
  if (w != w) return 0xFFFFFFFFu;
  return x >> 31 ? ~x : x | 0x80000000u;
}

// Digits of 11 bits for a large workgroup: two passes mostly, three of 8 bits, and weights of one
// magnitude spread over four bins (4 x 8 heads of up to 16384 tokens cut to 2048: 5% faster than by 8
// bits in 8 copies).
template <int THREADS>
struct Digit {
  static constexpr int kBits = THREADS >= 1024 ? 11 : 8, kBins = 1 << kBits;
  static constexpr int kCopies = THREADS >= 1024 ? 2 : 8;
  static constexpr int kCopy = kBins + 1;       // copies start in banks of their own
  static constexpr int kEach = (kBins + THREADS - 1) / THREADS;   // bins of a thread
};
template <int THREADS, int MOVES>
struct Shared {
  uint32_t bins[Digit<THREADS>::kCopies * Digit<THREADS>::kCopy];
  int waves[2][THREADS / 64];
  uint32_t prefix;
  int left, equal;
  uint32_t moves[MOVES];        // where the fills come from, in order
};

// Where a position's weight stands; none: nowhere, and `at` is something that may be read.
struct Spot {
  const float* at;
  bool none;
};
__device__ __forceinline__ Spot spot_at(const Evict& a, i64 page, const float* weights,
                                        uint32_t slot) {
  // (32 bits each, by strides of 64)
  return {page < 0 ? reinterpret_cast<const float*>(a.table.indptr)
                   : weights + static_cast<i64>(static_cast<uint32_t>(page)) * a.w_page +
                         static_cast<i64>(slot) * a.w_slot,
          page < 0};
}
template <typename P>
__device__ __forceinline__ Spot spot_of(const Evict& a, const P& page_of, const float* weights,
                                        int p) {
  const Place at = place_of(a, page_of, p);
  return spot_at(a, at.page, weights, at.slot);
}

// After a digit's counts: in which bin the `left`-th largest is, how many of it are left, and how
// many it holds.  Bins are counted from the largest down, neighbours by one thread.
template <int THREADS, typename S>
__device__ __forceinline__ void find_bin(S& s, uint32_t prefix, int bits, int left) {
  using D = Digit<THREADS>;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int top = D::kBins - 1 - tid * D::kEach;
  int n[D::kEach], mine = 0;
#pragma unroll
  for (int i = 0; i < D::kEach; ++i) {
    n[i] = 0;
    if (top >= i) {
#pragma unroll
      for (int c = 0; c < D::kCopies; ++c) n[i] += s.bins[c * D::kCopy + top - i];
    }
    mine += n[i];
  }
  int sum = upto(mine);
  if (lane == 63) s.waves[0][wave] = sum;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int other = s.waves[0][w];
    sum += w < wave ? other : 0;
  }
  if (sum >= left && sum - mine < left) {
    sum -= mine;
#pragma unroll
    for (int i = 0; i < D::kEach; ++i) {
      if (sum < left && sum + n[i] >= left) {
        s.prefix = prefix << bits | static_cast<uint32_t>(top - i);
        s.left = left - sum;
        s.equal = n[i];
      }
      sum += n[i];
    }
  }
  __syncthreads();
}

template <int THREADS, typename S>
__device__ __forceinline__ void clear_bins(S& s) {
  constexpr int kAll = Digit<THREADS>::kCopies * Digit<THREADS>::kCopy;
#pragma unroll
  for (int i = 0; i < (kAll + THREADS - 1) / THREADS; ++i)
    if (threadIdx.x + i * THREADS < kAll) s.bins[threadIdx.x + i * THREADS] = 0;
  __syncthreads();
}
// Counts a key: the digit of `bits` from `shift` on.
template <int THREADS, typename S>
__device__ __forceinline__ void count_key(S& s, uint32_t key, int shift, int bits) {
  using D = Digit<THREADS>;
  atomicAdd(&s.bins[(threadIdx.x % D::kCopies) * D::kCopy + (key >> shift & ((1u << bits) - 1))], 1u);
}

// Of positions, from the four of the first one on, those that threads have to hold.
__device__ __forceinline__ int span_of(int count, int first) { return count + (first & 3); }

// Of a sequence and kv head that loses tokens: what stays, from keys that threads hold, EACH to a
// thread, by fours of neighbouring positions, which start at a multiple of four: one lookup and one
// load for a four where pages hold whole ones: some 60 instructions for a key, 100 key by key (14.1 us
// of 28.3 in the case above, 19 of 34 key by key).  Returns how many fill holes; `targets`, if any,
// are those.
template <int THREADS, int EACH, typename S, typename P>
__device__ __forceinline__ int choose_held(const Evict& a, const P& page_of, const float* weights,
                                           S& s, int count, int first, int front, int32_t* kept,
                                           uint32_t* targets) {
  constexpr int kWaves = THREADS / 64, kFours = EACH / 4, kRuns = kFours * kWaves;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int last = first + count - 1, base = (first & ~3) + 4 * tid;
  auto at = [&](int q) { return base + 4 * THREADS * q; };
  // the first position of a wave's fours: what none of them needs is passed over together
  const int wave_base = (first & ~3) + 256 * __builtin_amdgcn_readfirstlane(wave);
  auto wave_at = [&](int q) { return wave_base + 4 * THREADS * q; };
  // The keys; 0: none of the candidates, below all of them.
  uint32_t key[EACH];
  auto put = [&](int q, int j, float w, bool none) __attribute__((always_inline)) {
    const uint32_t k = none ? 1u : order_of(w);
    key[4 * q + j] = static_cast<uint32_t>(at(q) + j - first) < static_cast<uint32_t>(count) ? k : 0u;
  };
  constexpr int kAtOnce = kFours < 4 ? kFours : 4;      // loads in flight
  if (a.table.page % 4 == 0) {
    // fours lie within a page; past the last candidate: the last's
    const int page = a.table.page;
    const int pages = a.table.by_page(4 * THREADS), slots = 4 * THREADS - pages * page;
    const uint32_t last_nth = a.table.by_page(last), last_slot = (last & ~3) - last_nth * page;
    uint32_t nth = a.table.by_page(base), slot = base - nth * page;
#pragma unroll
    for (int q0 = 0; q0 < kFours; q0 += kAtOnce) {
      Spot x[kAtOnce];
      float w[kAtOnce][4];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const bool past = at(q0 + q) > last;
        x[q] = spot_at(a, page_of(past ? last_nth : nth), weights, past ? last_slot : slot);
        nth += pages;
        slot += slots;
        const bool turn = slot >= static_cast<uint32_t>(page);
        nth += turn;
        slot -= turn ? page : 0;
      }
      if (a.w_slot == 1) {
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          if (!x[q].none) {
            const auto v = Loose<float, 4>::load(x[q].at);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[q][j] = v[j];
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[q][j] = x[q].at[x[q].none ? 0 : j * a.w_slot];
        }
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) put(q0 + q, j, w[q][j], x[q].none);
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < kFours; ++q) {
      Spot x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = spot_of(a, page_of, weights, min(max(at(q) + j, first), last));
#pragma unroll
      for (int j = 0; j < 4; ++j) put(q, j, *x[j].at, x[j].none);
    }
  }
  // the (front - first)-th largest, digit by digit; done when all that a bin holds stay
  uint32_t prefix = 0;
  int left = front - first, equal = 0, shift = 32;
  do {
    const int above = shift, bits = min(Digit<THREADS>::kBits, shift);
    shift -= bits;
    clear_bins<THREADS>(s);
    // (what is no candidate counts too, below all of them)
#pragma unroll
    for (int q = 0; q < kFours; ++q) {
      if (wave_at(q) > last) continue;
#pragma unroll
      for (int k = 4 * q; k < 4 * q + 4; ++k)
        if (above == 32 || key[k] >> above == prefix) count_key<THREADS>(s, key[k], shift, bits);
    }
    __syncthreads();
    find_bin<THREADS>(s, prefix, bits, left);
    prefix = s.prefix;
    left = s.left;
    equal = s.equal;
  } while (shift && left != equal);
  const uint32_t least = prefix << shift;       // what is above stays, and of what is equal `left`

  // Places among the flagged, run by run: a wave's lanes' fours.
  int* runs = reinterpret_cast<int*>(s.bins);
  static_assert(kRuns <= Digit<THREADS>::kCopies * Digit<THREADS>::kCopy && kFours <= 64, "");
  int before[kFours];     // flagged, before a lane's own four
  auto rank = [&](uint32_t flags) __attribute__((always_inline)) {
    int mine = 0;
#pragma unroll
    for (int q = 0; q < kFours; ++q) {
      int n = 0, all = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t mask = __ballot(flags >> (4 * q + j) & 1);
        n = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), n));
        all += __popcll(mask);
      }
      before[q] = n;
      if (lane == q) mine = all;
    }
    __syncthreads();
    if (lane < kFours) runs[lane * kWaves + wave] = mine;
    __syncthreads();
    if (wave == 0) {
      int sums = 0;
#pragma unroll
      for (int r = lane; r < (kRuns + 63) / 64 * 64; r += 64) {
        const int n = r < kRuns ? runs[r] : 0, sum = upto(n);
        if (r < kRuns) runs[r] = sums + sum - n;
        sums += __builtin_amdgcn_readlane(sum, 63);
      }
      if (lane == 0) s.left = sums;
    }
    __syncthreads();
    const int starts = runs[min(lane, kFours - 1) * kWaves + wave];
#pragma unroll
    for (int q = 0; q < kFours; ++q) before[q] += __builtin_amdgcn_readlane(starts, q);
  };
  auto nth_of = [&](uint32_t flags, int q, int j) __attribute__((always_inline)) {
    return before[q] + __popc(flags >> (4 * q) & ((1u << j) - 1));
  };
  uint32_t stays = 0, real = 0;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    stays |= key[k] >= least ? 1u << k : 0u;
    real |= key[k] ? 1u << k : 0u;
  }
  if (left != equal) {
    uint32_t ties = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) ties |= key[k] == least ? 1u << k : 0u;
    rank(ties);
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if ((ties >> k & 1) && nth_of(ties, k / 4, k % 4) >= left) stays &= ~(1u << k);
  }
  // holes below the front, then as many that stay past it, which fill them
  uint32_t below = 0;
#pragma unroll
  for (int q = 0; q < kFours; ++q) {
    const int n = min(max(front - at(q), 0), 4);
    below |= ((1u << n) - 1) << (4 * q);
  }
  const uint32_t flags = (below & real) ^ stays;
  rank(flags);
  const int holes = s.left / 2;
#pragma unroll
  for (int q = 0; q < kFours; ++q) {
    if (wave_at(q) + 256 <= front) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((flags & ~below) >> (4 * q + j) & 1) s.moves[nth_of(flags, q, j) - holes] = at(q) + j;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kFours; ++q) {
    if (wave_at(q) >= front) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((below & real) >> (4 * q + j) & 1) {
        const int p = at(q) + j, n = nth_of(flags, q, j);
        const bool stay = stays >> (4 * q + j) & 1;
        kept[p] = stay ? p : static_cast<int>(s.moves[n]);
        if (targets && !stay) targets[n] = p;
      }
    }
  }
  return holes;
}

// The same from memory, key by key, for any number of candidates.  Each thread has a run of them
// for the places; moves are listed some at a time.
template <int THREADS, int MOVES, typename S, typename F>
__device__ __forceinline__ void choose_any(S& s, int count, int first, int front, int32_t* kept,
                                        F&& spot) {
  constexpr int kWaves = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto key = [&](int c) {
    const Spot x = spot(first + c);
    const uint32_t k = order_of(*x.at);
    return x.none ? 0u : k;
  };
  uint32_t prefix = 0;
  int left = front - first;
  for (int shift = 32; shift > 0;) {
    const int above = shift, bits = min(Digit<THREADS>::kBits, shift);
    shift -= bits;
    clear_bins<THREADS>(s);
#pragma unroll 8
    for (int c = tid; c < count; c += THREADS) {
      const uint32_t k = key(c);
      if (above == 32 || k >> above == prefix) count_key<THREADS>(s, k, shift, bits);
    }
    __syncthreads();
    find_bin<THREADS>(s, prefix, bits, left);
    prefix = s.prefix;
    left = s.left;
  }
  const int run = (count + THREADS - 1) / THREADS;
  const int c0 = min(static_cast<int64_t>(tid) * run, static_cast<int64_t>(count));
  const int c1 = min(c0 + run, count);
  auto scan = [&](int& x, int& y) {     // sums over the threads before
    const int u = upto(x), v = upto(y);
    if (lane == 63) {
      s.waves[0][wave] = u;
      s.waves[1][wave] = v;
    }
    __syncthreads();
    x = u - x;
    y = v - y;
    for (int w = 0; w < wave; ++w) {
      x += s.waves[0][w];
      y += s.waves[1][w];
    }
    __syncthreads();
  };
  int ties = 0, none = 0;
  for (int c = c0; c < c1; ++c) ties += key(c) == prefix;
  scan(ties, none);
  auto each = [&](auto&& visit) {
    int tie = ties;
    for (int c = c0; c < c1; ++c) {
      const uint32_t k = key(c);
      const bool stays = k > prefix || (k == prefix && tie < left);
      tie += k == prefix;
      visit(first + c, stays);
    }
  };
  int holes = 0, fills = 0;
  each([&](int p, bool stays) {
    holes += p < front && !stays;
    fills += p >= front && stays;
  });
  scan(holes, fills);
  bool more = true;
  for (int base = 0; more; base += MOVES) {
    int nth = fills;
    bool past = false;
    each([&](int p, bool stays) {
      if (p >= front && stays) {
        if (nth >= base && nth < base + MOVES) s.moves[nth - base] = p;
        past |= nth >= base + MOVES;
        ++nth;
      }
    });
    more = __syncthreads_or(past);
    nth = holes;
    each([&](int p, bool stays) {
      if (p < front) {
        if (stays) {
          if (base == 0) kept[p] = p;
        } else {
          if (nth >= base && nth < base + MOVES) kept[p] = static_cast<int>(s.moves[nth - base]);
          ++nth;
        }
      }
    });
    __syncthreads();
  }
}

template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void choose(Evict a) {
  constexpr int kMoves = THREADS * EACH / 2;    // at most: as many leave holes as fill them
  __shared__ Shared<THREADS, kMoves> shared;
  const int tid = threadIdx.x;
  const int b = a.by_heads(blockIdx.x), h = blockIdx.x - b * a.kv_heads;
  const Held s = held_of(a, b);
  const int gone = s.keys > a.keep ? s.keys - a.keep : 0;
  int32_t* kept = a.kept + static_cast<i64>(blockIdx.x) * a.keep;
  if (h == 0 && tid == 0) a.lengths_out[b] = s.keys - gone;
  if (gone == 0) {
    for (int i = tid; i < a.keep; i += THREADS) kept[i] = i < s.keys ? i : -1;
    return;
  }
  const int front = a.keep - a.recent, count = s.keys - a.recent - a.first;
  const Far page_of = {s.list, a.table.pages};
  auto spot = [&](int p) { return spot_of(a, page_of, a.weights + h * a.w_head, p); };
  if (front > a.first) {
    if (span_of(count, a.first) <= THREADS * EACH)
      choose_held<THREADS, EACH>(a, page_of, a.weights + h * a.w_head, shared, count, a.first, front, kept,
                                 nullptr);
    else
      choose_any<THREADS, kMoves>(shared, count, a.first, front, kept, spot);
  }
  for (int i = tid; i < a.keep; i += THREADS)
    if (i < a.first || i >= front) kept[i] = i < front ? i : i + gone;
}

constexpr int kMovers = 256;      // threads

// Units of 16 bytes of a row; the last may be shorter.
template <typename T>
__device__ __forceinline__ typename Chunk<T>::Vec read_unit(const T* p, int n) {
  typename Chunk<T>::Vec v = typename Chunk<T>::Vec(T(0));
  if (n >= Chunk<T>::N) return Chunk<T>::load(p);
#pragma unroll
  for (int i = 0; i < Chunk<T>::N; ++i)
    if (i < n) v[i] = p[i];
  return v;
}
template <typename T>
__device__ __forceinline__ void write_unit(T* p, int n, typename Chunk<T>::Vec v) {
  if (n >= Chunk<T>::N) {
    Chunk<T>::store(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < Chunk<T>::N; ++i)
    if (i < n) p[i] = v[i];
}

constexpr int kWindow = 4, kListed = kWindow * kMovers, kDeep = 8;

// Where rows go and come from, in elements from the head's first.
constexpr i64 kNowhere = INT64_MIN;
struct Moves {
  i64 from[kListed], to[kListed];
  int count, past;
};

// A slice of a head's rows: `units` units of 16 bytes (the last may be shorter), `dim` elements.
template <typename T>
struct Slice {
  T* base;
  i64 by_page, by_slot;
  int dim, units;
  Div by_units;
  __device__ __forceinline__ i64 row(const Evict& a, const int64_t* list, int p) const {
    const Place at = place_of(a, Far{list, a.table.pages}, p);
    return at.page < 0 ? kNowhere : at.page * by_page + at.slot * by_slot;
  }
};

// Of the kept tokens i0 .. i1 those that come from `least` or past it, or (before) from below.  No
// place is both a source and a target.  Returns whether one came from `least` on.
template <typename T>
__device__ __forceinline__ bool fill(const Evict& a, const Held& s, const int32_t* kept,
                                     const Slice<T>& slice, Moves& m, int i0, int i1, int least,
                                     bool before) {
  const int tid = threadIdx.x;
  if (tid == 0) m.count = m.past = 0;
  __syncthreads();
  int from[kWindow];
#pragma unroll
  for (int k = 0; k < kWindow; ++k) {
    const int i = i0 + k * kMovers + tid;
    from[k] = i < i1 ? kept[i] : i;
  }
#pragma unroll
  for (int k = 0; k < kWindow; ++k) {
    const int i = i0 + k * kMovers + tid;
    if (from[k] == i) continue;
    if (from[k] >= least) m.past = 1;
    if ((from[k] < least) != before) continue;
    const i64 x = slice.row(a, s.list, from[k]), y = slice.row(a, s.list, i);
    if (x != kNowhere && y != kNowhere) {
      const int n = atomicAdd(&m.count, 1);
      m.from[n] = x;
      m.to[n] = y;
    }
  }
  __syncthreads();
  const int work = m.count * slice.units;
  const bool past = m.past;
  for (int w0 = tid; w0 < work; w0 += kDeep * kMovers) {    // (some reads, then their writes)
    typename Chunk<T>::Vec v[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int w = w0 + k * kMovers;
      if (w < work) {
        const int n = slice.by_units(w), u = (w - n * slice.units) * Chunk<T>::N;
        v[k] = read_unit(slice.base + m.from[n] + u, slice.dim - u);
      }
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int w = w0 + k * kMovers;
      if (w < work) {
        const int n = slice.by_units(w), u = (w - n * slice.units) * Chunk<T>::N;
        write_unit(slice.base + m.to[n] + u, slice.dim - u, v[k]);
      }
    }
  }
  __syncthreads();
  return past;
}

// The recent tokens go down, chunk by chunk, each read whole before any of it is written: what a
// chunk writes is behind all that later ones read.  Below `keep`, where they go, stand sources of
// fills: those fills come before the first chunk is written, while it is on its way.
template <typename T>
__device__ __forceinline__ void shift_down(const Evict& a, const Held& s, const int32_t* kept,
                                           const Slice<T>& slice, Moves& m, Moves& fills) {
  const int tid = threadIdx.x, front = a.keep - a.recent, gone = s.keys - a.keep;
  const int most = kDeep * kMovers / slice.units;       // rows of a chunk
  const int rows = most < kMovers ? most : kMovers;
  typename Chunk<T>::Vec v[kDeep];
  auto read = [&](int row0) __attribute__((always_inline)) {
    const int n = min(rows, a.recent - row0);
    __syncthreads();
    if (tid < n) {
      const i64 x = slice.row(a, s.list, front + row0 + tid + gone);
      const i64 y = slice.row(a, s.list, front + row0 + tid);
      m.from[tid] = x;
      m.to[tid] = x == kNowhere ? x : y;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int w = i * kMovers + tid;
      if (w < n * slice.units) {
        const int r = slice.by_units(w), u = (w - r * slice.units) * Chunk<T>::N;
        if (m.to[r] != kNowhere) v[i] = read_unit(slice.base + m.from[r] + u, slice.dim - u);
      }
    }
  };
  if (a.recent) read(0);
  for (int i0 = a.first; i0 < front; i0 += kListed)
    if (fill(a, s, kept, slice, fills, i0, min(i0 + kListed, front), a.keep, true)) break;
  for (int row0 = 0; row0 < a.recent; row0 += rows) {
    if (row0) read(row0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // every thread has what it read
    __syncthreads();
    const int n = min(rows, a.recent - row0);
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int w = i * kMovers + tid;
      if (w < n * slice.units) {
        const int r = slice.by_units(w), u = (w - r * slice.units) * Chunk<T>::N;
        if (m.to[r] != kNowhere) write_unit(slice.base + m.to[r] + u, slice.dim - u, v[i]);
      }
    }
  }
}

// Fills are in the order of their sources, so that those from below `keep` come first.  A cache's
// head has one workgroup for each slice of its rows, which moves those and then the recent tokens,
// and `chunks` for the other fills, a range of the kept tokens each.
template <typename T>
__global__ __launch_bounds__(kMovers) void move(Evict a) {
  __shared__ Moves m, fills;
  const int per = 2 * (a.slices + a.chunks) + a.move_weights * (1 + a.chunks);
  const int unit = a.by_parts(blockIdx.x);
  int part = blockIdx.x - unit * per;
  const int b = a.by_heads(unit), h = unit - b * a.kv_heads;
  const Held s = held_of(a, b);
  if (s.keys <= a.keep) return;
  const int32_t* kept = a.kept + static_cast<i64>(unit) * a.keep;
  const int front = a.keep - a.recent;
  auto run = [&](const auto& slice, int chunk) __attribute__((always_inline)) {
    if (chunk < 0) {
      shift_down(a, s, kept, slice, m, fills);
      return;
    }
    const int each = ((front - a.first + a.chunks - 1) / a.chunks + kMovers - 1) & -kMovers;
    const int end = min(front, a.first + (chunk + 1) * each);
    for (int i0 = a.first + chunk * each; i0 < end; i0 += kListed)
      fill(a, s, kept, slice, fills, i0, min(i0 + kListed, end), a.keep, false);
  };
  if (part >= 2 * (a.slices + a.chunks)) {
    part -= 2 * (a.slices + a.chunks);
    Slice<float> w = {a.weights + h * a.w_head, a.w_page, a.w_slot, 1, 1, {}};
    w.by_units.mul = 1;
    w.by_units.shift = 0;
    run(w, part - 1);
    return;
  }
  const bool value = part >= a.slices + a.chunks;
  if (value) part -= a.slices + a.chunks;
  const int chunk = part - a.slices;
  const int first = chunk < 0 ? part * a.slice : 0;     // units
  const int units = chunk < 0 ? min(a.units - first, a.slice) : a.units;
  Slice<T> x;
  x.base = static_cast<T*>(value ? a.value_cache : a.key_cache) +
           h * (value ? a.vc_head : a.kc_head) + first * Chunk<T>::N;
  x.by_page = value ? a.vc_page : a.kc_page;
  x.by_slot = value ? a.vc_slot : a.kc_slot;
  x.dim = min(a.dim - first * Chunk<T>::N, units * Chunk<T>::N);
  x.units = units;
  x.by_units = chunk >= 0 ? a.by_row : units == a.slice ? a.by_slice : a.by_last;
  run(x, chunk);
}

// All of it in one launch, for many heads or few bytes: a workgroup chooses for a head and moves its
// keys, values and weights, the recent tokens' on their way while it chooses.
template <typename T, int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void evict_whole(Evict a) {
  constexpr int kMoves = THREADS * EACH / 2, kRows = 256, kFills = 4, kNear = 512;
  __shared__ Shared<THREADS, kMoves> shared;
  __shared__ uint32_t s_to[kMoves];
  __shared__ i64 s_from[2][kRows], s_target[2][kRows];    // of keys and values
  __shared__ int32_t s_pages[kNear];
  const int tid = threadIdx.x;
  const int b = a.by_heads(blockIdx.x), h = blockIdx.x - b * a.kv_heads;
  const Held s = held_of(a, b);
  const int gone = s.keys > a.keep ? s.keys - a.keep : 0;
  int32_t* kept = a.kept + static_cast<i64>(blockIdx.x) * a.keep;
  if (h == 0 && tid == 0) a.lengths_out[b] = s.keys - gone;
  if (gone == 0) {
    for (int i = tid; i < a.keep; i += THREADS) kept[i] = i < s.keys ? i : -1;
    return;
  }
  const int front = a.keep - a.recent, count = s.keys - a.recent - a.first;
  const Far far = {s.list, a.table.pages};
  const Near page_of = {s_pages, min(static_cast<int>(a.table.by_page(s.keys - 1)) + 1, kNear), far};
  for (int i = tid; i < page_of.count; i += THREADS) s_pages[i] = static_cast<int32_t>(far(i));
  __syncthreads();
  T* const keys = static_cast<T*>(a.key_cache) + h * a.kc_head;
  T* const values = static_cast<T*>(a.value_cache) + h * a.vc_head;
  float* const weights = a.weights + h * a.w_head;
  auto put_row = [&](int n, int from, int to) {
    const Place x = place_of(a, page_of, from), y = place_of(a, page_of, to);
    const bool none = x.page < 0 || y.page < 0;
    s_from[0][n] = none ? kNowhere : x.page * a.kc_page + x.slot * a.kc_slot;
    s_target[0][n] = none ? kNowhere : y.page * a.kc_page + y.slot * a.kc_slot;
    s_from[1][n] = x.page * a.vc_page + x.slot * a.vc_slot;
    s_target[1][n] = y.page * a.vc_page + y.slot * a.vc_slot;
  };
  // units of the recent tokens' rows, of keys and then of values, some rows at a time
  const int most = kDeep * THREADS / (2 * a.units), rows = most < kRows ? most : kRows;
  typename Chunk<T>::Vec v[kDeep];
  auto read = [&](int row0) __attribute__((always_inline)) {
    const int n = min(rows, a.recent - row0);
    __syncthreads();
    if (tid < n) put_row(tid, front + row0 + tid + gone, front + row0 + tid);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      int w = i * THREADS + tid;
      const bool value = w >= n * a.units;
      if (value) w -= n * a.units;
      if (w < n * a.units) {
        const int r = a.by_row(w), u = (w - r * a.units) * Chunk<T>::N;
        if (s_target[0][r] != kNowhere)
          v[i] = read_unit((value ? values : keys) + s_from[value][r] + u, a.dim - u);
      }
    }
  };
  if (a.recent) read(0);
  auto spot = [&](int p) { return spot_of(a, page_of, weights, p); };
  // (the first chunk's targets, which the fills' places go over)
  i64 target[2] = {kNowhere, 0};
  if (tid < kRows && a.recent) {
    target[0] = s_target[0][tid];
    target[1] = s_target[1][tid];
  }
  int fills = 0;
  bool listed = true;
  if (front > a.first) {
    if (span_of(count, a.first) <= THREADS * EACH) {
      fills = choose_held<THREADS, EACH>(a, page_of, weights, shared, count, a.first, front, kept, s_to);
    } else {
      choose_any<THREADS, kMoves>(shared, count, a.first, front, kept, spot);
      listed = false;
      fills = front - a.first;      // any of them may be one
    }
  }
  for (int i = tid; i < a.keep; i += THREADS)
    if (i < a.first || i >= front) kept[i] = i < front ? i : i + gone;
  __syncthreads();
  for (int n0 = 0; n0 < fills; n0 += kRows) {
    const int n = min(kRows, fills - n0);
    if (tid < n) {
      const int to = listed ? s_to[n0 + tid] : a.first + n0 + tid;
      const int from = listed ? shared.moves[n0 + tid] : kept[to];
      put_row(tid, from, to);
      if (from == to) s_target[0][tid] = kNowhere;
      if (a.move_weights && from != to) {
        const Spot x = spot(from), y = spot(to);
        if (!x.none && !y.none) *const_cast<float*>(y.at) = *x.at;
      }
    }
    __syncthreads();
    for (int w0 = tid; w0 < 2 * n * a.units; w0 += kFills * THREADS) {
      typename Chunk<T>::Vec x[kFills];
#pragma unroll
      for (int i = 0; i < kFills; ++i) {
        int w = w0 + i * THREADS;
        const bool value = w >= n * a.units;
        if (value) w -= n * a.units;
        const int r = a.by_row(w), u = (w - r * a.units) * Chunk<T>::N;
        if (w < n * a.units && s_target[0][r] != kNowhere)
          x[i] = read_unit((value ? values : keys) + s_from[value][r] + u, a.dim - u);
      }
#pragma unroll
      for (int i = 0; i < kFills; ++i) {
        int w = w0 + i * THREADS;
        const bool value = w >= n * a.units;
        if (value) w -= n * a.units;
        const int r = a.by_row(w), u = (w - r * a.units) * Chunk<T>::N;
        if (w < n * a.units && s_target[0][r] != kNowhere)
          write_unit((value ? values : keys) + s_target[value][r] + u, a.dim - u, x[i]);
      }
    }
    __syncthreads();
  }
  if (tid < kRows && a.recent) {
    s_target[0][tid] = target[0];
    s_target[1][tid] = target[1];
  }
  for (int row0 = 0; row0 < a.recent; row0 += rows) {
    if (row0) read(row0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // every thread has what it read
    __syncthreads();
    const int n = min(rows, a.recent - row0);
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      int w = i * THREADS + tid;
      const bool value = w >= n * a.units;
      if (value) w -= n * a.units;
      if (w < n * a.units) {
        const int r = a.by_row(w), u = (w - r * a.units) * Chunk<T>::N;
        if (s_target[0][r] != kNowhere)
          write_unit((value ? values : keys) + s_target[value][r] + u, a.dim - u, v[i]);
      }
    }
  }
  if (!a.move_weights) return;
  for (int row0 = 0; row0 < a.recent; row0 += THREADS) {
    const int p = front + row0 + tid;
    const Spot x = spot(min(p, a.keep - 1) + gone), y = spot(min(p, a.keep - 1));
    const float w = *x.at;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (p < a.keep && !x.none && !y.none) *const_cast<float*>(y.at) = w;
  }
}

template <typename T>
const void* whole_of(int threads) {
  return threads == 256   ? reinterpret_cast<const void*>(&evict_whole<T, 256, 16>)
         : threads == 512 ? reinterpret_cast<const void*>(&evict_whole<T, 512, 8>)
                          : reinterpret_cast<const void*>(&evict_whole<T, 1024, 4>);
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" __attribute__((visibility("default"))) int launch_paged_evict(const tg_paged_evict* r,
                                                                         void* stream) {
  const char* what = "launch_paged_evict";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (r->dtype < TG_BF16 || r->dtype > TG_F32) return refuse(-1, what, "unknown dtype", r->dtype);
  if (const int rc =
          check_table(what, r->sequences, r->pages, r->page, r->n_indices, r->max_length))
    return rc;
  if (r->kv_heads < 1 || r->kv_heads > 0x10000)
    return refuse(-1, what, "kv_heads must be 1 to 65536", r->kv_heads);
  if (r->dim < 1 || r->dim > 1024) return refuse(-1, what, "dim must be 1 to 1024", r->dim);
  if (r->keep < 0 || r->recent < 0 || r->first < 0)
    return refuse(-1, what, "negative size", r->keep < 0 ? r->keep : r->recent);
  if (r->keep > (1 << 22)) return refuse(-2, what, "more than 2^22 tokens to keep", r->keep);
  if (r->recent > r->keep || r->first > r->keep - r->recent)
    return refuse(-1, what, "first and recent are more than keep", r->first);
  if (r->move_weights != 0 && r->move_weights != 1)
    return refuse(-1, what, "move_weights must be 0 or 1", r->move_weights);
  const int64_t strides[] = {r->kc_page, r->kc_slot, r->kc_head, r->vc_page, r->vc_slot,
                             r->vc_head, r->w_page,  r->w_slot,  r->w_head};
  if (const int rc = check_strides(what, strides, 9)) return rc;
  if (r->sequences == 0) return 0;
  const Operand kc = {"key_cache", r->key_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->kc_page, r->kc_slot, r->kc_head, 1}};
  const Operand vc = {"value_cache", r->value_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->vc_page, r->vc_slot, r->vc_head, 1}};
  const Operand w = {"weights", r->weights, 3, {r->pages, r->page, r->kv_heads},
                     {r->w_page, r->w_slot, r->w_head}};
  const int bytes = r->dtype == TG_F32 ? 4 : 2;
  const Operand weights = bytes == 4 ? w : in_halves(w);
  for (const Operand* x : {&kc, &vc})
    if (const int rc = once(what, *x)) return rc;
  if (r->move_weights)
    if (const int rc = once(what, w)) return rc;
  if (const int rc = apart(what, vc, kc, bytes)) return rc;
  for (const Operand* x : {&kc, &vc})
    if (const int rc = apart(what, weights, *x, bytes)) return rc;
  const Operand lengths = {"lengths", r->lengths, 1, {r->sequences}, {1}};
  const Operand lengths_out = {"lengths_out", r->lengths_out, 1, {r->sequences}, {1}};
  if (const int rc = apart(what, lengths_out, lengths, 8)) return rc;
  if (!r->indptr || !r->lengths || !r->lengths_out || (r->keep && !r->kept) ||
      (r->n_indices && !r->indices) ||
      (r->pages && (!r->key_cache || !r->value_cache || !r->weights)))
    return refuse(-1, what, "null array", r->sequences);
  Evict a = {};
  a.key_cache = r->key_cache;
  a.value_cache = r->value_cache;
  a.weights = r->weights;
  a.lengths_out = r->lengths_out;
  a.kept = r->kept;
  a.table.indptr = r->indptr;
  a.table.indices = r->indices;
  a.table.lengths = r->lengths;
  a.table.pages = r->pages;
  a.table.n_indices = r->n_indices;
  a.table.sequences = static_cast<int>(r->sequences);
  a.table.page = static_cast<int>(r->page);
  a.table.by_page = Div(a.table.page);
  a.kc_page = r->kc_page;
  a.kc_slot = r->kc_slot;
  a.kc_head = r->kc_head;
  a.vc_page = r->vc_page;
  a.vc_slot = r->vc_slot;
  a.vc_head = r->vc_head;
  a.w_page = r->w_page;
  a.w_slot = r->w_slot;
  a.w_head = r->w_head;
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.dim = static_cast<int>(r->dim);
  a.keep = static_cast<int>(r->keep);
  a.recent = static_cast<int>(r->recent);
  a.first = static_cast<int>(r->first);
  a.move_weights = static_cast<int>(r->move_weights);
  a.by_heads = Div(a.kv_heads);
  const int64_t heads = r->sequences * r->kv_heads;
  a.units = (a.dim * bytes + 15) / 16;
  // rows in slices of 64 bytes at least, and kept tokens in chunks, while there are few workgroups
  int slices = 1;
  while (heads * 2 * slices < 512 && a.units / (2 * slices) >= 4) slices *= 2;
  a.slice = (a.units + slices - 1) / slices;
  a.slices = (a.units + a.slice - 1) / a.slice;
  const int64_t filled = r->max_length > r->keep ? r->keep - r->recent - r->first : 0;
  int64_t chunks = (filled + kMovers - 1) / kMovers;
  if (chunks * heads > 512) chunks = 512 / heads;
  a.chunks = static_cast<int>(chunks > 1 ? chunks : 1);
  a.by_row = Div(a.units);
  a.by_slice = Div(a.slice);
  a.by_last = Div(a.units - (a.slices - 1) * a.slice);
  const int per = 2 * (a.slices + a.chunks) + a.move_weights * (1 + a.chunks);
  a.by_parts = Div(per);
  if (heads * per > kMostGroups) return refuse(-2, what, "2^24 workgroups or more", heads * per);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  void* args[] = {&a};
  const int64_t most = r->max_length - r->recent - (r->first & ~int64_t(3));    // candidates, in fours
  // One launch where a workgroup's threads hold a head's candidates, unless few heads have many
  // recent tokens to move, which slices do side by side.  8 kv heads of 128, up to 1088 tokens cut to 1024
  // with 256 recent: 1 sequence 14.2 us, 15.2 in two launches, 32 20.2 and 29.4, 128 74 and 134; 4000
  // to 1024: 12.6 and 14.2, 15.5 and 23.9; 4128 to 4096 with 1024 recent: 1 sequence 28.8 and 26.3, 8
  // 35.3 and 38.8, 64 138 and 214.
  if (most <= 4096 && (heads >= 64 || r->recent * a.units <= 8192)) {
    // Workgroups that fill a compute unit by themselves while there is one for each, smaller ones side by
    // side for more heads.  By 1024, 512 and 256 threads, up to 949 tokens of 80 cut to 166: 384 heads
    // 24.9, 18.1 and 20.6 us, 848 heads 50, 36 and 30; up to 1088 of 128 cut to 1024: 256 heads 20,
    // 23 and 28, 512 heads 41, 38 and 41, 1024 heads 90, 79 and 69.
    const int threads = heads <= 256 ? 1024 : heads <= 640 ? 512 : 256;
    const void* k = bytes == 4 ? whole_of<uint32_t>(threads) : whole_of<uint16_t>(threads);
    const hipError_t e = launch(k, heads, threads, args, s);
    return e == hipSuccess ? 0 : hip_failed(e, what);
  }
  const int threads = most <= 2048 ? 256 : 1024;
  hipError_t e = launch(most <= 2048    ? reinterpret_cast<const void*>(&choose<256, 8>)
                        : most <= 4096  ? reinterpret_cast<const void*>(&choose<1024, 4>)
                        : most <= 16384 ? reinterpret_cast<const void*>(&choose<1024, 16>)
                                        : reinterpret_cast<const void*>(&choose<1024, 32>),
                        heads, threads, args, s);
  if (e != hipSuccess) return hip_failed(e, what);
  if (r->keep == 0) return 0;
  e = launch(bytes == 4 ? reinterpret_cast<const void*>(&move<uint32_t>)
                        : reinterpret_cast<const void*>(&move<uint16_t>),
             heads * per, kMovers, args, s);
  return e == hipSuccess ? 0 : hip_failed(e, what);
}
