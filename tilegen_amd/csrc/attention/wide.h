// Attention of many query rows to the same keys: a workgroup of four waves holds 128 rows, 32
// a wave, and walks the keys 64 at a time through LDS.
//
// As in the narrow kernel scores are computed transposed, here on 32x32x16 instructions: a lane
// holds, for query row lane % 32, keys 8 i + 4 (lane / 32) + 0..3 of each 32, and the
// probabilities of 16 keys are a B operand of O^T = V^T P^T when the sum over the keys runs in
// that order.  Tiles are double-buffered, and one barrier a tile separates the buffers.  Loads
// run a tile ahead, but only while scores are taken: the transposing reads of values might read
// what the loads write for all that the compiler knows, so it waits for every load before the
// first of them and not at the barrier alone.
//
// A 32x32x16 product takes 32 cycles of a SIMD's matrix core and reads 1 KB of keys or values
// from LDS, so four waves ask for LDS's 128 bytes a cycle, the loads' writes for a quarter more,
// and the softmax of a tile takes as many vector cycles as its products take matrix cycles.  So
// the next tile's scores are computed while this one's probabilities are, instruction by
// instruction (side_by_side), and two workgroups share a CU.  1024 rows of each of 8 kv heads of
// 128 on 32768 keys (137 GFLOP): 187 to 200 us, 690 to 735 TFLOP/s; a plain product of 8192^3
// reaches 1330.  64 rows a wave (half the LDS reads, one wave a SIMD) took 1.8 times as long;
// eight waves and 256 rows a workgroup as long for the prefix and 8% longer beside own pages.
#pragma once

#include <type_traits>

#include "parts.h"

namespace tg {

template <int DP>
struct Wide {
  static constexpr int kRows = 32 * kWaves, kKeys = 64;
  static constexpr int kPitch = DP == 64 ? 128 : DP == 256 ? 512 : 256;   // bytes of an LDS row
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kLoads = kKeys * kChunks / kThreads;   // of each thread, keys and values
  static constexpr int kPass = kThreads / kChunks;            // rows that one load of all covers
  static constexpr int kSpan = kThreads * 16;                 // and their bytes
  static constexpr int kTile = kKeys * kPitch;
  static constexpr int kBuffer = 2 * kTile;               // keys, then values

  // Loads go straight to LDS, 16 bytes a lane side by side, so rows cannot be padded; instead a
  // row's chunks change places, and a lane fetches the chunk that belongs to its place.  Keys
  // are read as one chunk of 8 rows at a time, values as 4 chunks of 4 rows: with these
  // either is spread over all 64 banks.
  static __device__ __forceinline__ int key_place(int row) {
    return kPitch == 128 ? row >> 1 & 7 : row & 15;
  }
  static __device__ __forceinline__ int value_place(int row) {
    return kPitch == 128 ? (row >> 1 & 1) << 2 : (row & 3) << 2;
  }
};

// The order of a whole tile's instructions: after each product the vector instructions that fit
// beside it (32 cycles: one exponential takes 16, others 4) and the LDS reads of a later one.
template <int KS, int DT>
__device__ __forceinline__ void side_by_side() {
  constexpr int kMatrix = 0x008, kVector = 0x002, kExp = 0x400, kRead = 0x100;
  constexpr int kAhead = 4, kScores = 2 * KS, kValues = 4 * DT;
  __builtin_amdgcn_sched_group_barrier(kRead, kAhead, 0);
#pragma unroll
  for (int i = 0; i < kScores / 2 - kAhead / 2; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kVector, 24 / KS, 0);
    __builtin_amdgcn_sched_group_barrier(kExp, 8 / KS, 0);
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kVector, 32 / KS, 0);
    __builtin_amdgcn_sched_group_barrier(kExp, 8 / KS, 0);
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
    __builtin_amdgcn_sched_group_barrier(kVector, 32 / KS, 0);
    __builtin_amdgcn_sched_group_barrier(kExp, 8 / KS, 0);
  }
#pragma unroll
  for (int i = 0; i < kValues / 2; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
    __builtin_amdgcn_sched_group_barrier(kVector, 20 / DT, 0);
    __builtin_amdgcn_sched_group_barrier(kExp, 8 / DT, 0);
  }
#pragma unroll
  for (int i = 0; i < kValues / 2; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
    __builtin_amdgcn_sched_group_barrier(kVector, 12 / DT, 0);
  }
}

template <typename T, int DP, bool OWN>
__device__ __forceinline__ void wide_part(const Attention& a, const Part& p, int kv_head,
                                          char* lds) {
  using W = Wide<DP>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 16, DT = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;

  // queries: the B operand, elements 16 s + 8 half .. of row col
  s16x8 q[KS];
  const int row = p.row0 + wave * 32 + col;
  const bool live = row < p.rows;
  int see;
  {
    const int r = live ? row : p.rows - 1;
    const int j = a.by_group(r), h = kv_head * a.group + r - j * a.group;
    const T* at = static_cast<const T*>(a.q) + (p.token0 + j) * a.q_token + h * a.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * half;
      q[s] = s16x8(0);
      if (live && d < a.dim) q[s] = __builtin_bit_cast(s16x8, C::load(at + d));
    }
    see = live ? min(p.before + p.step * j, p.k1) : 0;
  }
  const int all = min(p.before + p.step * static_cast<int>(a.by_group(p.row0)), p.k1);

  // this thread's place in rows first + kPass i of a tile, and the chunks that belong there
  const int place = tid % W::kChunks, first = tid / W::kChunks;
  const T* kc = static_cast<const T*>(a.k) + kv_head * a.kc_head;
  const T* vc = static_cast<const T*>(a.v) + kv_head * a.vc_head;
  const int tiles = (p.k1 - p.k0 + W::kKeys - 1) / W::kKeys;

  // Where keys are: bytes from the head's first key, or negative where a key has no page.  Where
  // pages hold whole groups of 8 keys (`even`) a lane knows where one group starts, 64 lanes 8
  // tiles of them; a wave's rows of one load stand in one group, so that the address is uniform.
  // Elsewhere a lane knows one key of one tile.  Pages are asked for a tile before they are
  // needed and before that tile's loads, since loads return in order.  Lookups past the end
  // are the last key's.
  auto key_of_lane = [&](int tile) {
    return min(a.even ? p.k0 + (tile >> 3) * 8 * W::kKeys + 8 * lane
                      : p.k0 + tile * W::kKeys + lane,
               p.k1 - 1);
  };
  auto pages_of = [&](int tile) { return p.list[a.by_page(key_of_lane(tile))]; };
  auto offsets_of = [&](int tile, i64 page) -> i64 {
    const int key = key_of_lane(tile) & (a.even ? ~7 : ~0);
    const int slot = key - static_cast<int>(a.by_page(key)) * a.page;
    const i64 at = a.even ? (page * a.kc_page + slot * a.kc_slot) * 2
                          : page << 32 | static_cast<unsigned>(slot);
    return page < 0 || page >= a.pages ? -1 : at;
  };
  // a bit for each key of a tile that has no page
  auto lost = [&](int tile, i64 offsets) -> unsigned long long {
    unsigned long long none = __ballot(offsets < 0);
    if (!a.even || none == 0) return none;
    none = none >> (tile % 8 * 8) & 0xFF;
    unsigned long long keys = 0;
    for (int i = 0; i < 8; ++i)
      if (none >> i & 1) keys |= 0xFFull << (8 * i);
    return keys;
  };
  unsigned in_group[2];     // bytes from a group's first row to this lane's
#pragma unroll
  for (int i = 0; i < 2; ++i)
    in_group[i] = ((first + W::kPass * i) & 7) * static_cast<unsigned>(a.kc_slot) * 2;
  // one tile's keys or values
  auto load = [&](auto which, int tile, i64 offsets) {
    constexpr bool kKeys = decltype(which)::value;
    char* to = lds + (tile & 1) * W::kBuffer + (kKeys ? 0 : W::kTile) + wave * 1024;
    const T* cache = kKeys ? kc : vc;
    auto chunk = [&](int row) {
      return place ^ (kKeys ? W::key_place(row) : W::value_place(row));
    };
    const int key0 = p.k0 + tile * W::kKeys;
    if (a.even && key0 + W::kKeys <= p.k1 && !__any(offsets < 0)) {
      const char* at[W::kLoads];
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i) {
        const int group =
            tile % 8 * 8 + __builtin_amdgcn_readfirstlane((first + W::kPass * i) >> 3);
        const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(offsets), group);
        const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(offsets >> 32), group);
        at[i] = reinterpret_cast<const char*>(cache) + (static_cast<uint64_t>(hi) << 32 | lo);
      }
      if constexpr (W::kPass >= 16) {     // the same chunk, and place in a group, of all rows
        if (chunk(first) * 8 < a.dim)
#pragma unroll
          for (int i = 0; i < W::kLoads; ++i)
            load_to_lds(at[i] + (in_group[0] + chunk(first) * 16), to + W::kSpan * i);
      } else {
#pragma unroll
        for (int i = 0; i < W::kLoads; ++i) {
          const int c = chunk(first + W::kPass * i);
          if (c * 8 < a.dim) load_to_lds(at[i] + (in_group[i & 1] + c * 16), to + W::kSpan * i);
        }
      }
      return;
    }
    const i64 page_stride = kKeys ? a.kc_page : a.vc_page;
    const i64 slot_stride = kKeys ? a.kc_slot : a.vc_slot;
#pragma unroll 1
    for (int i = 0; i < W::kLoads; ++i) {
      const int r = first + W::kPass * i, d = chunk(r) * 8;
      const int key = min(key0 + r, p.k1 - 1);
      const i64 at = __shfl(offsets, a.even ? tile % 8 * 8 + ((key - key0) >> 3) : r);
      if (at >= 0 && key0 + r < p.k1) {
        const T* from = a.even ? cache + at / 2 + (key & 7) * slot_stride
                               : cache + (at >> 32) * page_stride +
                                     static_cast<i64>(static_cast<unsigned>(at)) * slot_stride;
        if (d < a.dim) load_to_lds(from + d, to + W::kSpan * i);
      } else {    // no page, or past the end: hidden below, and zero, since 0 times an infinity
                  // or a NaN would be NaN
        *reinterpret_cast<s16x8*>(to + W::kSpan * i + 16 * lane) = s16x8(0);
      }
    }
  };
  const std::integral_constant<bool, true> keys_of{};
  const std::integral_constant<bool, false> values_of{};

  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x16(0.f);
  float m = -INFINITY, l = 0.f;
  bool huge = false;

  // elements past the head: zero keys, once (their queries are zero, and must not meet a NaN)
#pragma unroll
  for (int i = 0; i < W::kLoads; ++i)
    if ((place ^ W::key_place(first + W::kPass * i)) * 8 >= a.dim)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        *reinterpret_cast<s16x8*>(lds + b * W::kBuffer + W::kSpan * i + 16 * tid) = s16x8(0);

  // scores of the keys at `keys`
  auto score = [&](const char* keys, f32x16* s) {
    s[0] = f32x16(0.f);
    s[1] = f32x16(0.f);
#pragma unroll
    for (int e = 0; e < KS; ++e)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const s16x8 k = *reinterpret_cast<const s16x8*>(
            keys + (32 * t + col) * W::kPitch + ((2 * e + half) ^ W::key_place(col)) * 16);
        s[t] = M::mul32(k, q[e], s[t]);
      }
  };
  // -inf where a row sees fewer keys, and for keys without a page (a bit each); this lane's
  // keys are 32 t + 8 (i / 4) + i % 4 from its first
  auto hide = [&](f32x16* s, int left, unsigned long long without) {
    left -= 4 * half;
    without >>= 4 * half;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned word = static_cast<unsigned>(without >> (32 * t));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = 8 * (i / 4) + i % 4;
        if (32 * t + at >= left || (word >> at & 1)) s[t][i] = -INFINITY;
      }
    }
  };
  auto largest = [&](const f32x16* s) {
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    return top;
  };
  // lets the running maximum follow where a row's scores have left it far behind
  auto follow = [&](float top) {
    top *= a.scale;
    if (__any(passes<T>(top, m))) {
      const Both both = halves(top);
      const float to = fmaxf(base_of<T>(fmaxf(both.a, both.b)), m);
      const float f = m == -INFINITY ? 0.f : exp2f(m - to);
      m = to;
      huge |= __any(fabsf(to) > kHuge && to != -INFINITY);
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
  };
  // probabilities of 32 keys: the B operands of two products
  auto weigh = [&](const f32x16& s, float scale, float base, s16x8* prob) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -base));
      sum += e;
      prob[i / 8][i % 8] = __builtin_bit_cast(short, static_cast<T>(e));
    }
    return sum;
  };
  // V^T, an A operand: lanes name rows 4 half + i/4 of 16 keys and columns 16 (lane/16 % 2) ..
  const int vrow = 4 * half + (lane & 15) / 4;
  auto value = [&](const char* values, int step, int d) {
    const int c = (4 * d + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ W::value_place(vrow);
    const char* at = values + (16 * step + vrow) * W::kPitch + c * 16 + 8 * (lane & 1);
    const s16x4 lo = transposed(at), hi = transposed(at + 8 * W::kPitch);
    return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  // (scale, base) for weigh; past kHuge the products are rounded before
  auto bases = [&](f32x16* s, float* scale, float* base) {
    *base = m == -INFINITY ? 0.f : m;
    *scale = a.scale;
    if (huge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = apart(s[t][i], a.scale, *base);
      *base = 0.f;
      *scale = 1.f;
    }
  };

  // Tiles that all rows see whole.  A tile's scores are taken while the tile before it is weighed:
  // its keys are loaded two tiles ahead, its values one.
  const int whole = (all - p.k0) / W::kKeys > 0 ? (all - p.k0) / W::kKeys : 0;
  if (DP > 128 && whole) {
    // A head this long leaves no registers for a second tile's scores (they and O would change
    // between register files every tile): only the loads run ahead.  1280 rows of one kv head on
    // 32000 keys 93 us, 109 with scores ahead; 40 rows of 8 kv heads 83 and 101.
    i64 where = offsets_of(0, pages_of(0)), page = pages_of(1);
    load(keys_of, 0, where);
    load(values_of, 0, where);
    __syncthreads();
#pragma unroll 1
    for (int tile = 0; tile < whole; ++tile) {
      const unsigned long long without = lost(tile, where);
      if (tile + 1 < whole) {
        if (!a.even || (tile + 1) % 8 == 0) where = offsets_of(tile + 1, page);
        page = pages_of(tile + 2);
        load(keys_of, tile + 1, where);
        load(values_of, tile + 1, where);
      }
      const char* keys = lds + (tile & 1) * W::kBuffer;
      const char* values = keys + W::kTile;
      f32x16 s[2];
      score(keys, s);
      if (without) hide(s, W::kKeys, without);
      follow(largest(s));
      float scale, base;
      bases(s, &scale, &base);
      s16x8 prob[4];
      l += weigh(s[0], scale, base, prob);
      l += weigh(s[1], scale, base, prob + 2);
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = M::mul32(value(values, step, d), prob[step], o[d]);
      __syncthreads();
    }
  } else if (whole) {
    const i64 at0 = offsets_of(0, pages_of(0));
    i64 where = a.even ? at0 : offsets_of(1, pages_of(1));    // of the next tile's keys
    i64 page0 = pages_of(2), page1;
    float top;
    load(keys_of, 0, at0);
    load(values_of, 0, at0);
    if (whole > 1) load(keys_of, 1, where);
    __syncthreads();
    f32x16 s0[2], s1[2];
    score(lds, s0);
    if (const unsigned long long without = lost(0, at0)) hide(s0, W::kKeys, without);
    top = largest(s0);
    __syncthreads();    // tile 2's keys take the place of tile 0's

    // with `now` the tile's scores and `top` a lane's largest: adds it, and leaves the next
    // one's scores in `then`.  `page`: of tile + 2; page_then: of the one after, still on its
    // way (a copy of it would wait for it and for the loads behind it)
    auto add = [&](int tile, f32x16* now, f32x16* then, const i64& page, i64& page_then) {
      const char* keys = lds + ((tile + 1) & 1) * W::kBuffer;
      const char* values = lds + (tile & 1) * W::kBuffer + W::kTile;
      const unsigned long long without = lost(tile + 1, where);
      const i64 here = where;
      if (!a.even || (tile + 2) % 8 == 0) where = offsets_of(tile + 2, page);
      page_then = pages_of(tile + 3);
      if (tile + 1 < whole) load(values_of, tile + 1, here);
      if (tile + 2 < whole) load(keys_of, tile + 2, where);
      follow(top);
      float scale, base;
      bases(now, &scale, &base);
      // Products and vector instructions side by side: the first half's exponentials under the
      // next tile's scores, the second's under the first half's values, the next
      // largest under the rest.
      s16x8 prob[4];
      score(keys, then);
      l += weigh(now[0], scale, base, prob);
      l += weigh(now[1], scale, base, prob + 2);
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = M::mul32(value(values, step, d), prob[step], o[d]);
      top = largest(then);
      asm volatile("" : "+v"(top), "+v"(l));    // here, not where they are used
      side_by_side<KS, DT>();
      if (without) {
        hide(then, W::kKeys, without);
        top = largest(then);
      }
      __syncthreads();
    };
    for (int tile = 0;;) {
      add(tile, s0, s1, page0, page1);
      if (++tile == whole) break;
      add(tile, s1, s0, page1, page0);
      if (++tile == whole) break;
    }
  }

  // Tiles that end inside, or that some rows see in part: one after the other.
#pragma unroll 1
  for (int tile = whole; tile < tiles; ++tile) {
    const i64 at = offsets_of(tile, pages_of(tile));
    load(keys_of, tile, at);
    load(values_of, tile, at);
    __syncthreads();
    const char* keys = lds + (tile & 1) * W::kBuffer;
    const char* values = keys + W::kTile;
    const int left = see - (p.k0 + tile * W::kKeys);
    f32x16 s[2];
    score(keys, s);
    hide(s, left, lost(tile, at));
    follow(largest(s));
    float scale, base;
    bases(s, &scale, &base);
    s16x8 prob[4];
    l += weigh(s[0], scale, base, prob);
    l += weigh(s[1], scale, base, prob + 2);
    bool strange = false;
    if (OWN) {
#pragma unroll 1
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x8 vt = value(values, step, d);
#pragma unroll
          for (int i = 0; i < 8; ++i)   // (nothing was stored past the head)
            strange |= 32 * d + col < a.dim && (vt[i] & M::kExponent) == M::kExponent;
        }
      strange = __any(strange);
    }
    if (!strange) {
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = M::mul32(value(values, step, d), prob[step], o[d]);
    } else {
      // an infinity or NaN among values that not all rows see: key by key, added to the rows
      // that see it alone (0 times either would be NaN in the others)
#pragma unroll 1
      for (int key = 0; key < W::kKeys; ++key) {
        const int step = key / 16, i = key % 16 / 8 * 4 + key % 4;
        const bool holds = key % 8 / 4 == half;
        const s16x8 pr = step == 0 ? prob[0] : step == 1 ? prob[1] : step == 2 ? prob[2] : prob[3];
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x8 vt = value(values, step, d);
          s16x8 one = s16x8(0);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (holds && e == i) one[e] = vt[e];
          const f32x16 part = M::mul32(one, pr, f32x16(0.f));
          if (key < left) o[d] += part;
        }
      }
    }
    __syncthreads();
  }

  const Both both = halves(l);
  l = both.a + both.b;
  if (live) {
    const int j = a.by_group(row), h = kv_head * a.group + row - j * a.group;
    const i64 at = p.slot * (static_cast<i64>(a.tokens) * a.heads) +
                   static_cast<i64>(p.token0 + j) * a.heads + h;
    float* to = a.part + at * a.dim + 4 * half;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (32 * d + 8 * b + 4 * half < a.dim)
          *reinterpret_cast<f32x4*>(to + 32 * d + 8 * b) =
              f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    if (half == 0) a.part_ml[at] = make_float2(m, l);
  }
}

}  // namespace tg
