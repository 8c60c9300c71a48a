// Attention of few query rows to many keys: every wave reads keys and values of its own.
//
// Scores are computed transposed, S^T = K Q^T, on 16x16x32 matrix instructions: a wave's tile
// is 32 keys by NT x 16 query rows.  In the result a lane holds, for one query row (lane % 16),
// the keys 4 (lane / 16) + 0..3 of both halves of the tile.  That is a B operand of
// O^T = V^T P^T as it stands when the sum over the 32 keys runs in the order
// {4 q + i, 16 + 4 q + i}, so that probabilities never leave their lane.  The A operand V^T wants,
// in that order, four keys at a time of one element of the head: the transposing LDS read
// gives just that from values stored as they come.
//
// The running maximum of a row follows the scores only when they pass it by 2^8: until then
// probabilities are up to 256 times too large, sums and products as well, and their quotient
// is the same.  So most tiles need neither the exchange between lanes nor the rescaling.
//
// Memory bounds it: each wave keeps a ring of tiles in LDS that its loads fill without passing
// through registers, whole rows at a time, and waits for the oldest alone.
#pragma once

#include <type_traits>

#include "parts.h"

namespace tg {

template <int DP, int NT>
struct Narrow {
  static constexpr int kWaves = DP == 256 ? 2 : 4;
  static constexpr int kKeys = 32;                                        // of a wave's tile
  static constexpr int kPitch = DP == 64 ? 128 : DP == 256 ? 512 : 256;   // bytes of an LDS row
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kPass = 64 / kChunks;              // rows of one load
  static constexpr int kLoads = kKeys / kPass;            // of keys, and of values
  static constexpr int kTile = kKeys * kPitch;            // keys, then values
  static constexpr int kRing = DP == 64 ? 4 : 2;
  static constexpr int kSum = DP + 4;                     // floats of a row of sums
  static constexpr int kTops = kWaves * 16 * NT * 8;
  static constexpr int kBytes = kWaves * kRing * 2 * kTile + kTops;
  static_assert(kWaves * 16 * NT * kSum * 4 <= kWaves * kRing * 2 * kTile, "sums fit the rings");

  // as in wide.h: places of a row's 16-byte chunks
  static __device__ __forceinline__ int key_place(int row) {
    return kPitch == 128 ? row >> 1 & 7 : row & 15;
  }
  static __device__ __forceinline__ int value_place(int row) {
    return kPitch == 128 ? (row >> 1 & 1) << 2 : (row & 3) << 2;
  }
};

template <typename T, int DP, int NT>
__device__ __forceinline__ void narrow_part(const Attention& a, const Part& p, int kv_head,
                                            char* lds) {
  using W = Narrow<DP, NT>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 32;   // steps of a score's sum
  constexpr int DT = DP / 16;   // 16-row tiles of O^T
  constexpr int kWaves = W::kWaves;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;

  // queries: the B operand, lane's row nt * 16 + col, elements 32 s + 8 quad ..
  s16x8 q[NT][KS];
  int see[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = p.row0 + nt * 16 + col;
    const bool live = row < p.rows;
    const int r = live ? row : p.rows - 1;
    const int j = a.by_group(r), h = kv_head * a.group + r - j * a.group;
    const T* at = static_cast<const T*>(a.q) + (p.token0 + j) * a.q_token + h * a.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 32 * s + 8 * quad;
      q[nt][s] = s16x8(0);
      if (live && d < a.dim) q[nt][s] = __builtin_bit_cast(s16x8, C::load(at + d));
    }
    see[nt] = live ? min(p.before + p.step * j, p.k1) : 0;
  }
  // every live row sees the keys below `all`
  const int all = min(p.before + p.step * static_cast<int>(a.by_group(p.row0)), p.k1);

  f32x4 o[NT][DT];
  float m[NT], l[NT];
  bool huge = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY;
    l[nt] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[nt][d] = f32x4(0.f);
  }

  char* ring = lds + wave * (W::kRing * 2 * W::kTile);
  const T* kc = static_cast<const T*>(a.k) + kv_head * a.kc_head;
  const T* vc = static_cast<const T*>(a.v) + kv_head * a.vc_head;
  // this wave's tiles: wave, wave + kWaves, ... of the part's
  const int total = (p.k1 - p.k0 + W::kKeys - 1) / W::kKeys;
  const int tiles = wave < total ? (total - wave + kWaves - 1) / kWaves : 0;
  auto key_at = [&](int tile) { return p.k0 + W::kKeys * (wave + kWaves * tile); };

  const int place = lane % W::kChunks, first = lane / W::kChunks;   // of rows first + kPass i
  const unsigned in_first = first * static_cast<unsigned>(a.kc_slot) * 2;
  auto key_chunk = [&](int row) { return place ^ W::key_place(row); };
  auto value_chunk = [&](int row) { return place ^ W::value_place(row); };

  // Where pages hold whole groups of 8 keys (`eights`) each group's page is uniform: scalar
  // loads, a tile ahead, and scalar arithmetic (vector loads would have to be waited for, and
  // with them every load of a tile behind them).
  typedef const __attribute__((address_space(4))) int64_t ScalarList;
  ScalarList* scalar_list = (ScalarList*)(uintptr_t)p.list;
  constexpr int kGroups = W::kKeys / 8;
  struct Pages {
    i64 at[kGroups];
  };
  const int last_group = (p.k1 - 1) & ~7;
  auto pages_of = [&](int tile) {
    Pages g;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      g.at[i] = a.eights ? scalar_list[a.by_page(min(key_at(tile) + 8 * i, last_group))] : 0;
    return g;
  };
  // The loads of a tile into its place of the ring, which nothing reads any more; a bit for
  // each key that has no page.
  auto fetch = [&](int tile, const Pages& pages) -> unsigned {
    wait_lds();
    char* to = ring + tile % W::kRing * (2 * W::kTile);
    const int key0 = key_at(tile);
    bool fast = a.eights && key0 + W::kKeys <= p.k1;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) fast &= pages.at[g] >= 0 && pages.at[g] < a.pages;
    if (fast) {
      constexpr int kEach = 8 / W::kPass;     // loads of a group
      i64 at[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int key = key0 + 8 * g;
        const int slot = key - static_cast<int>(a.by_page(key)) * a.page;
        at[g] = (pages.at[g] * a.kc_page + slot * a.kc_slot) * 2;
      }
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i) {
        const int c = key_chunk(first + W::kPass * i);
        if (c * 8 < a.dim)
          fetch_to_lds(reinterpret_cast<const char*>(kc) + at[i / kEach] +
                           i % kEach * W::kPass * a.kc_slot * 2,
                       in_first + c * 16, to + 1024 * i);
      }
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i) {
        const int c = value_chunk(first + W::kPass * i);
        if (c * 8 < a.dim)
          fetch_to_lds(reinterpret_cast<const char*>(vc) + at[i / kEach] +
                           i % kEach * W::kPass * a.kc_slot * 2,
                       in_first + c * 16, to + W::kTile + 1024 * i);
      }
      return 0;
    }
    // Any other tile: lane i (and i + 32) looks key i up; keys past the end stand for the last
    // one (hidden below).
    const int key = min(key0 + (lane & 31), p.k1 - 1);
    const int nth = a.by_page(key), slot = key - nth * a.page;
    const i64 page = p.list[nth];
    const bool none = page < 0 || page >= a.pages;
    const i64 where = none ? -1 : page << 32 | static_cast<unsigned>(slot);
#pragma unroll 1
    for (int i = 0; i < W::kLoads; ++i) {
      const int row = first + W::kPass * i, kd = key_chunk(row) * 8, vd = value_chunk(row) * 8;
      const i64 at = __shfl(where, row), pg = at >> 32, in = static_cast<unsigned>(at);
      if (at >= 0) {
        if (kd < a.dim)
          fetch_to_lds(kc + pg * a.kc_page + in * a.kc_slot + kd, to + 1024 * i);
        if (vd < a.dim)
          fetch_to_lds(vc + pg * a.vc_page + in * a.vc_slot + vd, to + W::kTile + 1024 * i);
      } else {    // no page: zero, since 0 times a NaN would be NaN
        *reinterpret_cast<s16x8*>(to + 1024 * i + 16 * lane) = s16x8(0);
        *reinterpret_cast<s16x8*>(to + W::kTile + 1024 * i + 16 * lane) = s16x8(0);
      }
    }
    wait_loads<0>();      // (their number varies, and the waits below count on it)
    return static_cast<unsigned>(__ballot(none));
  };

  // elements past the head: zero keys, once (their queries are zero, and must not meet a NaN)
#pragma unroll
  for (int i = 0; i < W::kLoads; ++i)
    if (key_chunk(first + W::kPass * i) * 8 >= a.dim)
#pragma unroll
      for (int b = 0; b < W::kRing; ++b)
        *reinterpret_cast<s16x8*>(ring + b * 2 * W::kTile + 1024 * i + 16 * lane) = s16x8(0);

  unsigned gone[W::kRing];    // bit i: key i of the tile at that place has no page
  // one tile, then the loads of the one that takes its place
  auto add = [&](int tile, unsigned without, Pages& pages) -> unsigned {
    const int key0 = key_at(tile);
    const char* keys = ring + tile % W::kRing * (2 * W::kTile);
    const char* values = keys + W::kTile;
    // all but the loads of the tiles behind this one
    if (tile + W::kRing <= tiles)
      wait_loads<(W::kRing - 1) * 2 * W::kLoads>();
    else
      wait_loads<0>();
    f32x4 sc[NT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][t] = f32x4(0.f);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const s16x8 k = *reinterpret_cast<const s16x8*>(
            keys + (16 * t + col) * W::kPitch +
            ((4 * s + quad) ^ W::key_place(16 * t + col)) * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][t] = M::mul16(k, q[nt][s], sc[nt][t]);
      }
    }
    const bool partial = without != 0 || key0 + W::kKeys > all;
    if (partial) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int left = see[nt] - key0 - 4 * quad;
        const unsigned word = without >> (4 * quad);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * t + i >= left || (word >> (16 * t + i) & 1)) sc[nt][t][i] = -INFINITY;
      }
    }
    s16x8 prob[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = fmaxf(fmaxf(fmaxf(sc[nt][0][0], sc[nt][0][1]), fmaxf(sc[nt][0][2], sc[nt][0][3])),
                        fmaxf(fmaxf(sc[nt][1][0], sc[nt][1][1]), fmaxf(sc[nt][1][2], sc[nt][1][3])));
      top *= a.scale;
      if (__any(top > m[nt] + kSlack)) {
        const float now = fmaxf(row_max(top), m[nt]);
        const float f = m[nt] == -INFINITY ? 0.f : exp2f(m[nt] - now);
        m[nt] = now;
        huge |= __any(fabsf(now) > kHuge && now != -INFINITY);
        l[nt] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nt][d] *= f;
      }
      const float base = m[nt] == -INFINITY ? 0.f : m[nt];
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = huge ? apart(sc[nt][t][i], a.scale, base)
                               : __builtin_fmaf(sc[nt][t][i], a.scale, -base);
          const float e = __builtin_amdgcn_exp2f(x);
          sum += e;
          prob[nt][4 * t + i] = __builtin_bit_cast(short, static_cast<T>(e));
        }
      l[nt] += sum;
    }
    // V^T, the A operand: element 16 d + col of keys 4 quad + i and 16 + 4 quad + i
    const int vrow = 4 * quad + (col >> 2);
    auto value = [&](int d) {
      const int c = (2 * d + (col >> 1 & 1)) ^ W::value_place(vrow);
      const char* at = values + vrow * W::kPitch + c * 16 + 8 * (col & 1);
      const s16x4 lo = transposed(at), hi = transposed(at + 16 * W::kPitch);
      return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    bool strange = false;
    if (partial) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const s16x8 vt = value(d);
#pragma unroll
        for (int i = 0; i < 8; ++i)   // (nothing was stored past the head)
          strange |= 16 * d + col < a.dim && (vt[i] & M::kExponent) == M::kExponent;
      }
      strange = __any(strange);
    }
    if (!strange) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const s16x8 vt = value(d);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][d] = M::mul16(vt, prob[nt], o[nt][d]);
      }
    } else {
      // an infinity or NaN among the values of a tile that not all rows see: key by key, added
      // to the rows that see it alone (0 times either would be NaN in the others)
#pragma unroll 1
      for (int key = 0; key < W::kKeys; ++key) {
        const int mine = key % 16 - 4 * quad;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x8 vt = value(d);
          s16x8 one = s16x8(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (key < 16 && mine == i) one[i] = vt[i];
            if (key >= 16 && mine == i) one[4 + i] = vt[4 + i];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const f32x4 part = M::mul16(one, prob[nt], f32x4(0.f));
            if (key0 + key < see[nt]) o[nt][d] += part;
          }
        }
      }
    }
    unsigned none = 0;
    if (tile + W::kRing < tiles) {
      none = fetch(tile + W::kRing, pages);
      pages = pages_of(tile + W::kRing + 1);
    }
    return none;
  };

  if (tiles) {
    Pages pages = pages_of(0);
#pragma unroll
    for (int b = 0; b < W::kRing; ++b) {
      if (b < tiles) gone[b] = fetch(b, pages);
      pages = pages_of(b + 1);
    }
    // the queries have to be there by now, not (for all the compiler knows) in every turn
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < KS; ++s) asm volatile("" ::"v"(q[nt][s]));
    for (int tile = 0;;) {
#pragma unroll
      for (int b = 0; b < W::kRing; ++b) {
        gone[b] = add(tile, gone[b], pages);
        if (++tile == tiles) break;
      }
      if (tile == tiles) break;
    }
  }
  __syncthreads();    // the rings become the sums

  // The waves' sums become one: their common maximum, then O and l scaled to it.
  float* sums = reinterpret_cast<float*>(lds);
  float2* tops = reinterpret_cast<float2*>(lds + W::kBytes - W::kTops);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] = row_sum(l[nt]);
    if (quad == 0) tops[wave * 16 * NT + nt * 16 + col] = make_float2(m[nt], l[nt]);
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w * 16 * NT + nt * 16 + col].x);
    const float f = m[nt] == -INFINITY ? 0.f : exp2f(m[nt] - top);
    float* to = sums + (wave * 16 * NT + nt * 16 + col) * W::kSum + 4 * quad;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(to + 16 * d) = o[nt][d] * f;
  }
  __syncthreads();
  constexpr int kQuads = DP / 4;
  for (int i = threadIdx.x; i < 16 * NT * kQuads; i += 64 * kWaves) {
    const int r = i / kQuads, d = (i - r * kQuads) * 4;
    const int row = p.row0 + r;
    if (row >= p.rows || d >= a.dim) continue;
    f32x4 sum = f32x4(0.f);
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      sum += *reinterpret_cast<const f32x4*>(sums + (w * 16 * NT + r) * W::kSum + d);
      top = fmaxf(top, tops[w * 16 * NT + r].x);
    }
    const int j = a.by_group(row), h = kv_head * a.group + row - j * a.group;
    const i64 at = static_cast<i64>(p.token0 + j) * a.heads + h;
    const i64 rows = static_cast<i64>(a.tokens) * a.heads;
    *reinterpret_cast<f32x4*>(a.part + (p.slot * rows + at) * a.dim + d) = sum;
    if (d == 0) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = tops[w * 16 * NT + r];
        total += ml.x == -INFINITY ? 0.f : ml.y * exp2f(ml.x - top);
      }
      a.part_ml[p.slot * rows + at] = make_float2(top, total);
    }
  }
}

template <typename T, int DP, int NT>
__global__ __launch_bounds__((64 * Narrow<DP, NT>::kWaves)) void narrow_prefix(Attention a) {
  __shared__ __align__(16) char lds[Narrow<DP, NT>::kBytes];
  int tile, kv_head, split;
  if (!prefix_place(a, &tile, &kv_head, &split)) return;
  Part p;
  p.list = a.prefix;
  p.k0 = split * a.prefix_chunk;
  p.k1 = min(p.k0 + a.prefix_chunk, a.prefix_length);
  p.row0 = tile * 16 * NT;
  p.rows = a.tokens * a.group;
  p.token0 = 0;
  p.before = a.prefix_length;
  p.step = 0;
  p.slot = split;
  narrow_part<T, DP, NT>(a, p, kv_head, lds);
}

template <typename T, int DP, int NT>
__global__ __launch_bounds__((64 * Narrow<DP, NT>::kWaves)) void narrow_own(Attention a) {
  __shared__ __align__(16) char lds[Narrow<DP, NT>::kBytes];
  int first, split, head, b;
  if (!own_place(a, &first, &split, &head, &b)) return;
  const Sequence s = sequence(a, b);
  Part p;
  p.list = s.list;
  p.rows = s.count * a.group;
  p.token0 = s.first;
  p.before = s.before + 1;
  p.step = 1;
  p.slot = a.prefix_splits + split;
  p.k0 = split * a.own_chunk;
  for (int tile = first; tile * 16 * NT < p.rows; tile += a.own_tiles) {
    p.row0 = tile * 16 * NT;
    const int last = min(p.row0 + 16 * NT, p.rows) - 1;
    p.k1 = seen(s, a.by_group(last));
    if (split + 1 < a.own_splits) p.k1 = min(p.k1, p.k0 + a.own_chunk);
    if (p.k0 >= p.k1) continue;
    narrow_part<T, DP, NT>(a, p, head, lds);
    __syncthreads();
  }
}

template <int DP, typename T, int NT>
hipError_t launch_narrow_as(const Attention& a, bool prefix, hipStream_t stream) {
  i64 grid;
  const void* f;
  if (prefix) {
    grid = prefix_grid(a);
    f = reinterpret_cast<const void*>(&narrow_prefix<T, DP, NT>);
  } else {
    grid = own_grid(a);
    f = reinterpret_cast<const void*>(&narrow_own<T, DP, NT>);
  }
  Attention copy = a;
  void* args[] = {&copy};
  return hipLaunchKernel(f, dim3(static_cast<unsigned>(grid)), dim3(64 * Narrow<DP, NT>::kWaves), args, 0, stream);
}

template <int DP, typename T>
hipError_t launch_narrow_nt(const Attention& a, int nt, bool prefix, hipStream_t stream) {
  if (nt == 1) return launch_narrow_as<DP, T, 1>(a, prefix, stream);
  return launch_narrow_as<DP, T, 2>(a, prefix, stream);
}

template <int DP>
hipError_t launch_narrow(const Attention& a, int64_t dtype, int nt, bool prefix,
                         hipStream_t stream) {
  return dtype == TG_F16 ? launch_narrow_nt<DP, _Float16>(a, nt, prefix, stream)
                         : launch_narrow_nt<DP, __bf16>(a, nt, prefix, stream);
}

}  // namespace tg
