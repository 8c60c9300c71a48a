// Attention of few query rows to many keys: every wave reads keys and values of its own.
//
// Scores are computed transposed, S^T = K Q^T, on 16x16x32 matrix instructions: a wave's tile
// is 32 keys by 16 query rows.  In the result a lane holds, for one query row (lane % 16),
// the keys 4 (lane / 16) + 0..3 of both halves of the tile.  That is a B operand of
// O^T = V^T P^T as it stands when the sum over the 32 keys runs in the order
// {4 q + i, 16 + 4 q + i}, so that probabilities never leave their lane.  The A operand V^T wants,
// in that order, four keys at a time of one element of the head: the transposing LDS read
// gives just that from values stored as they come.
//
// The running maximum of a row follows the scores only when they pass it by 2^8: until then
// probabilities are up to 256 times too large (in float16 another 128 times, base_of), sums and
// products as well, and their quotient is the same.  So most tiles need neither the exchange
// between lanes nor the rescaling.
//
// Memory bounds it: 16 rows are half a matrix instruction's worth of work for the bytes read.
// Keys go straight to registers (the A operand is 16 bytes of a key a lane), the next tile's
// while this one's values go through LDS, and page numbers are asked for a tile earlier still.
// 128 sequences of 1 to 2048 own keys, 8 kv heads of 128 (540 MB): 135 us, 4.0 TB/s with the
// joining; a plain sum of as much reaches 5.7.  When it took 138, tiles through an LDS ring with
// one wave a workgroup took 145 to 155, loads that bypass the caches 161.
#pragma once

#include "parts.h"

namespace tg {

template <int DP>
struct Narrow {
  static constexpr int kRows = 16, kKeys = 32;            // of a wave's tile
  static constexpr int kRow = DP * 2 + 32;                // bytes of a value's row in LDS
  static constexpr int kValues = kWaves * kKeys * kRow;
  static constexpr int kSum = DP + 4;                     // floats of a row of sums
  static constexpr int kSums = kWaves * kRows * kSum * 4;
  static constexpr int kTops = kWaves * kRows * 8;
  static constexpr int kBytes = (kValues > kSums ? kValues : kSums) + kTops;
};

// BOTH: the prefix's keys and a sequence's own, and the rows' results instead of a part's sums.
template <typename T, int DP, bool BOTH>
__device__ __forceinline__ void narrow_part(const Attention& a, const Part& p, int kv_head,
                                            char* lds) {
  using W = Narrow<DP>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 32;   // steps of a score's sum
  constexpr int DT = DP / 16;   // 16-row tiles of O^T
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, quad = lane >> 4;

  // queries: the B operand, lane's row col, elements 32 s + 8 quad ..
  s16x8 q[KS];
  int see;
  {
    const int row = p.row0 + col;
    const bool live = row < p.rows;
    const int r = live ? row : p.rows - 1;
    const int j = a.by_group(r), h = kv_head * a.group + r - j * a.group;
    const T* at = static_cast<const T*>(a.q) + (p.token0 + j) * a.q_token + h * a.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 32 * s + 8 * quad;
      q[s] = s16x8(0);
      if (live && d < a.dim) q[s] = __builtin_bit_cast(s16x8, C::load(at + d));
    }
    see = live ? min(p.before + p.step * j, p.k1) : 0;
    if (BOTH && live) see = max(see, p.own_from);
  }
  // every live row sees the keys below `all`
  int all = min(p.before + p.step * static_cast<int>(a.by_group(p.row0)), p.k1);
  if (BOTH) all = max(all, p.own_from);

  f32x4 o[DT];
  float m = -INFINITY, l = 0.f;
  bool huge = false;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4(0.f);

  char* values = lds + wave * 32 * W::kRow;
  const T* kc = static_cast<const T*>(a.k) + kv_head * a.kc_head;
  const T* vc = static_cast<const T*>(a.v) + kv_head * a.vc_head;
  const int tiles = (p.k1 - p.k0 + 31) / 32;

  // keys k0 + 32 tile + {0, 16} + col: their pages, asked for one tile before their loads;
  // keys past the end stand for the last one (hidden below)
  i64 pg[2];
  int slot[2];
  auto find = [&](int tile) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = min(p.k0 + 32 * tile + 16 * t + col, p.k1 - 1);
      const bool own = BOTH && key >= p.own_from;
      const int in = own ? key - p.own_from : key;
      const int nth = a.by_page(in);
      slot[t] = in - nth * a.page;
      pg[t] = (own ? p.own_list : p.list)[nth];
    }
  };
  s16x8 k[2][KS], v[2][KS];
  bool bad[2];
  auto load = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      bad[t] = pg[t] < 0 || pg[t] >= a.pages;
      const i64 page = bad[t] ? 0 : pg[t];
      const T* ka = kc + page * a.kc_page + slot[t] * a.kc_slot + 8 * quad;
      const T* va = vc + page * a.vc_page + slot[t] * a.vc_slot + 8 * quad;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (32 * s + 8 * quad < a.dim) {
          k[t][s] = __builtin_bit_cast(s16x8, C::load(ka + 32 * s));
          v[t][s] = __builtin_bit_cast(s16x8, C::load(va + 32 * s));
        } else {
          k[t][s] = s16x8(0);
          v[t][s] = s16x8(0);
        }
      }
    }
  };

  if (wave < tiles) {
    find(wave);
    load();
    find(wave + kWaves);
  }
  for (int tile = wave; tile < tiles; tile += kWaves) {
    const int key0 = p.k0 + 32 * tile;
    // bit i: key 16 t + i of the tile has no page
    unsigned gone[2] = {0u, 0u};
    bool strange = false;
    const bool any_bad = __any(bad[0] || bad[1]);
    const bool partial = any_bad || key0 + 32 > all;
    if (partial) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        gone[t] = static_cast<unsigned>(__ballot(bad[t])) & 0xFFFFu;
        if (bad[t]) {
#pragma unroll
          for (int s = 0; s < KS; ++s) v[t][s] = s16x8(0);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            strange |= (v[t][s][i] & M::kExponent) == M::kExponent;
      }
      strange = __any(strange);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        *reinterpret_cast<s16x8*>(values + (16 * t + col) * W::kRow + 64 * s + 16 * quad) =
            v[t][s];
    f32x4 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4(0.f);
#pragma unroll
      for (int s = 0; s < KS; ++s) sc[t] = M::mul16(k[t][s], q[s], sc[t]);
    }
    if (tile + kWaves < tiles) {
      load();
      find(tile + 2 * kWaves);
    }

    if (partial) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = 4 * quad + i;
          if (key0 + 16 * t + at >= see || (gone[t] >> at & 1)) sc[t][i] = -INFINITY;
        }
    }
    float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                      fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    top *= a.scale;
    if (__any(passes<T>(top, m))) {
      const float now = fmaxf(base_of<T>(row_max(top)), m);
      const float f = m == -INFINITY ? 0.f : exp2f(m - now);
      m = now;
      huge |= __any(fabsf(now) > kHuge && now != -INFINITY);
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;
    s16x8 prob;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = huge ? apart(sc[t][i], a.scale, base)
                             : __builtin_fmaf(sc[t][i], a.scale, -base);
        const float e = __builtin_amdgcn_exp2f(x);
        l += e;
        prob[4 * t + i] = __builtin_bit_cast(short, static_cast<T>(e));
      }
    __builtin_amdgcn_wave_barrier();
    const char* from = values + (4 * quad + (col >> 2)) * W::kRow + (col & 3) * 8;
    if (!strange) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const s16x4 lo = transposed(from + 32 * d);
        const s16x4 hi = transposed(from + 32 * d + 16 * W::kRow);
        const s16x8 vt = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        o[d] = M::mul16(vt, prob, o[d]);
      }
    } else {
      // an infinity or NaN among the values of a tile that not all rows see: key by key, added
      // to the rows that see it alone (0 times either would be NaN in the others)
#pragma unroll 1
      for (int key = 0; key < 32; ++key) {
        const int mine = key < 16 ? key - 4 * quad : key - 16 - 4 * quad;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x4 lo = transposed(from + 32 * d);
          const s16x4 hi = transposed(from + 32 * d + 16 * W::kRow);
          s16x8 vt = s16x8(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (key < 16 && mine == i) vt[i] = lo[i];
            if (key >= 16 && mine == i) vt[4 + i] = hi[i];
          }
          const f32x4 one = M::mul16(vt, prob, f32x4(0.f));
          if (key0 + key < see) o[d] += one;
        }
      }
    }
  }

  // The waves' sums become one: their common maximum, then O and l scaled to it.
  float* sums = reinterpret_cast<float*>(lds);
  float2* tops = reinterpret_cast<float2*>(lds + W::kBytes - W::kTops);
  l = row_sum(l);
  if (quad == 0) tops[wave * 16 + col] = make_float2(m, l);
  __syncthreads();
  {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w * 16 + col].x);
    const float f = m == -INFINITY ? 0.f : exp2f(m - top);
    float* to = sums + (wave * 16 + col) * W::kSum + 4 * quad;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(to + 16 * d) = o[d] * f;
  }
  __syncthreads();
  constexpr int kQuads = DP / 4;
  for (int i = threadIdx.x; i < 16 * kQuads; i += 64 * kWaves) {
    const int r = i / kQuads, d = (i - r * kQuads) * 4;
    const int row = p.row0 + r;
    if (row >= p.rows || d >= a.dim) continue;
    f32x4 sum = f32x4(0.f);
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      sum += *reinterpret_cast<const f32x4*>(sums + (w * 16 + r) * W::kSum + d);
      top = fmaxf(top, tops[w * 16 + r].x);
    }
    const int j = a.by_group(row), h = kv_head * a.group + row - j * a.group;
    const i64 at = static_cast<i64>(p.token0 + j) * a.heads + h;
    if (BOTH || d == 0) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = tops[w * 16 + r];
        // without a maximum the sum is 0, or NaN from scores that are
        total += ml.x == -INFINITY ? ml.y : ml.y * exp2f(ml.x - top);
      }
    }
    if (BOTH) {
      T* out = static_cast<T*>(a.out) + (p.token0 + j) * a.o_token + h * a.o_head + d;
      const float f = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(total == 0.f ? 0.f : sum[e] * f);
      if (d == 0 && a.lse) a.lse[at] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
    } else {
      const i64 rows = static_cast<i64>(a.tokens) * a.heads;
      *reinterpret_cast<f32x4*>(a.part + (p.slot * rows + at) * a.dim + d) = sum;
      if (d == 0) a.part_ml[p.slot * rows + at] = make_float2(top, total);
    }
  }
}

}  // namespace tg
