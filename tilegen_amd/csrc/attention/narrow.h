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
#pragma once

#include "parts.h"

namespace tg {

constexpr int kWaves = 4;

template <int DP, int NT>
struct NarrowLds {
  static constexpr int kRow = DP * 2 + 32;               // bytes of a value's row
  static constexpr int kValues = kWaves * 32 * kRow;
  static constexpr int kSum = DP + 4;                    // floats of a row of sums
  static constexpr int kSums = kWaves * 16 * NT * kSum * 4;
  static constexpr int kBytes = (kValues > kSums ? kValues : kSums) + kWaves * 16 * NT * 8;
};

template <typename T, int DP, bool FULL, int NT>
__device__ __forceinline__ void narrow_part(const Attention& a, const Part& p, int kv_head,
                                            char* lds) {
  using L = NarrowLds<DP, NT>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 32;   // steps of a score's sum
  constexpr int DT = DP / 16;   // 16-row tiles of O^T
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
      if (live && (FULL || d < a.dim)) q[nt][s] = __builtin_bit_cast(s16x8, C::load(at + d));
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

  char* values = lds + wave * 32 * L::kRow;
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
      const int nth = a.by_page(key);
      slot[t] = key - nth * a.page;
      pg[t] = p.list[nth];
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
        if (FULL || 32 * s + 8 * quad < a.dim) {
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
        *reinterpret_cast<s16x8*>(values + (16 * t + col) * L::kRow + 64 * s + 16 * quad) =
            v[t][s];
    f32x4 sc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[nt][t] = f32x4(0.f);
#pragma unroll
        for (int s = 0; s < KS; ++s) sc[nt][t] = M::mul16(k[t][s], q[nt][s], sc[nt][t]);
      }
    if (tile + kWaves < tiles) {
      load();
      find(tile + 2 * kWaves);
    }

    if (partial) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 4 * quad + i;
            if (key0 + 16 * t + at >= see[nt] || (gone[t] >> at & 1)) sc[nt][t][i] = -INFINITY;
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
    __builtin_amdgcn_wave_barrier();
    const char* from = values + (4 * quad + (col >> 2)) * L::kRow + (col & 3) * 8;
    if (!strange) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const s16x4 lo = transposed(from + 32 * d);
        const s16x4 hi = transposed(from + 32 * d + 16 * L::kRow);
        const s16x8 vt = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][d] = M::mul16(vt, prob[nt], o[nt][d]);
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
          const s16x4 hi = transposed(from + 32 * d + 16 * L::kRow);
          s16x8 vt = s16x8(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (key < 16 && mine == i) vt[i] = lo[i];
            if (key >= 16 && mine == i) vt[4 + i] = hi[i];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const f32x4 one = M::mul16(vt, prob[nt], f32x4(0.f));
            if (key0 + key < see[nt]) o[nt][d] += one;
          }
        }
      }
    }
  }

  // The four waves' sums become one: their common maximum, then O and l scaled to it.
  float* sums = reinterpret_cast<float*>(lds);
  float2* tops = reinterpret_cast<float2*>(lds + L::kBytes - kWaves * 16 * NT * 8);
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
    float* to = sums + (wave * 16 * NT + nt * 16 + col) * L::kSum + 4 * quad;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(to + 16 * d) = o[nt][d] * f;
  }
  __syncthreads();
  constexpr int kQuads = DP / 4;
  for (int i = threadIdx.x; i < 16 * NT * kQuads; i += 64 * kWaves) {
    const int r = i / kQuads, d = (i - r * kQuads) * 4;
    const int row = p.row0 + r;
    if (row >= p.rows || (!FULL && d >= a.dim)) continue;
    f32x4 sum = f32x4(0.f);
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      sum += *reinterpret_cast<const f32x4*>(sums + (w * 16 * NT + r) * L::kSum + d);
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

template <typename T, int DP, bool FULL, int NT>
__global__ __launch_bounds__(64 * kWaves) void narrow_prefix(Attention a) {
  __shared__ __align__(16) char lds[NarrowLds<DP, NT>::kBytes];
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
  narrow_part<T, DP, FULL, NT>(a, p, kv_head, lds);
}

template <typename T, int DP, bool FULL, int NT>
__global__ __launch_bounds__(64 * kWaves) void narrow_own(Attention a) {
  __shared__ __align__(16) char lds[NarrowLds<DP, NT>::kBytes];
  int first, split, head, b;
  own_place<64 * kWaves>(a, &first, &split, &head, &b);
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
    narrow_part<T, DP, FULL, NT>(a, p, head, lds);
    __syncthreads();
  }
}

template <int DP, typename T, bool FULL, int NT>
hipError_t launch_narrow_as(const Attention& a, bool prefix, hipStream_t stream) {
  i64 grid;
  const void* f;
  if (prefix) {
    grid = prefix_grid(a);
    f = reinterpret_cast<const void*>(&narrow_prefix<T, DP, FULL, NT>);
  } else {
    grid = own_grid(a);
    f = reinterpret_cast<const void*>(&narrow_own<T, DP, FULL, NT>);
  }
  Attention copy = a;
  void* args[] = {&copy};
  return hipLaunchKernel(f, dim3(static_cast<unsigned>(grid)), dim3(64 * kWaves), args, 0, stream);
}

template <int DP, typename T, bool FULL>
hipError_t launch_narrow_nt(const Attention& a, int nt, bool prefix, hipStream_t stream) {
  if (nt == 1) return launch_narrow_as<DP, T, FULL, 1>(a, prefix, stream);
  return launch_narrow_as<DP, T, FULL, 2>(a, prefix, stream);
}

template <int DP>
hipError_t launch_narrow(const Attention& a, int64_t dtype, int nt, bool prefix,
                         hipStream_t stream) {
  const bool full = a.dim == DP;
  if (dtype == TG_F16)
    return full ? launch_narrow_nt<DP, _Float16, true>(a, nt, prefix, stream)
                : launch_narrow_nt<DP, _Float16, false>(a, nt, prefix, stream);
  return full ? launch_narrow_nt<DP, __bf16, true>(a, nt, prefix, stream)
              : launch_narrow_nt<DP, __bf16, false>(a, nt, prefix, stream);
}

}  // namespace tg
