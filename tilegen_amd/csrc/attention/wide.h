// Attention of many query rows to the same keys: a workgroup of four waves holds 128 rows, 32
// a wave, and walks the keys 64 at a time through LDS.
//
// As in the narrow kernel scores are computed transposed, here on 32x32x16 instructions: a lane
// holds, for query row lane % 32, keys 8 i + 4 (lane / 32) + 0..3 of each 32, and the
// probabilities of 16 keys are a B operand of O^T = V^T P^T when the sum over the keys runs in that
// order.  Tiles are double-buffered: the next one's loads are in flight while this one is
// multiplied, and one barrier a tile separates the buffers.
//
// A 32x32x16 product takes 32 cycles of a SIMD's matrix core and reads 1 KB of keys or values from
// LDS, so four waves ask for LDS's 128 bytes a cycle and the softmax of a tile takes as
// many vector cycles as its products take matrix cycles: two workgroups a CU overlap them.
#pragma once

#include "parts.h"

namespace tg {

template <int DP>
struct Wide {
  static constexpr int kRows = 128, kKeys = 64;
  static constexpr int kSlots = DP == 96 ? 16 : DP / 8;     // 16-byte chunks of a row, padded
  static constexpr int kLoads = kKeys * kSlots / 256;       // of each thread, keys and values
  static constexpr int kPass = 256 / kSlots;                // rows that one load of all covers
  // LDS rows.  Keys are read 16 bytes of 8 rows at a time: 16 bytes more than a power of two
  // spread them over all banks.  Values are read as 64 bytes of 4 rows: 64 bytes more.
  static constexpr int kKeyRow = DP * 2 + 16;
  static constexpr int kValueRow = DP == 96 ? 192 : DP * 2 + 64;
  static constexpr int kBuffer = kKeys * (kKeyRow + kValueRow);
  static constexpr int kPerCu = DP == 256 ? 1 : 2;
};

// Addresses of a tile's rows.  EVEN: pages hold whole groups of 16 keys, so that a wave's rows of
// one load stand on one page: its number and offset are uniform.
template <typename T, int DP, bool EVEN, bool OWN>
__device__ __forceinline__ void wide_part(const Attention& a, const Part& p, int kv_head,
                                          char* lds) {
  using W = Wide<DP>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 16, DT = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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

  // this thread's chunk of rows first + kPass i of a tile
  const int chunk = tid % W::kSlots, first = tid / W::kSlots;
  const bool mine = chunk * 8 < a.dim;
  const T* kc = static_cast<const T*>(a.k) + kv_head * a.kc_head + chunk * 8;
  const T* vc = static_cast<const T*>(a.v) + kv_head * a.vc_head + chunk * 8;
  const int tiles = (p.k1 - p.k0 + W::kKeys - 1) / W::kKeys;

  i64 pg[W::kLoads];
  int slot[W::kLoads];
  unsigned long long gone;      // keys of the tile in the registers that have no page
  auto find = [&](int tile) {
    const int key0 = p.k0 + tile * W::kKeys;
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) {
      if (EVEN) {
        const int group = __builtin_amdgcn_readfirstlane((first + W::kPass * i) & ~15);
        const int key = min(key0 + group, (p.k1 - 1) & ~15);
        const int nth = a.by_page(key);
        slot[i] = key - nth * a.page + min((first + W::kPass * i) & 15, p.k1 - 1 - key);
        pg[i] = p.list[nth];
      } else {
        const int key = min(key0 + first + W::kPass * i, p.k1 - 1);
        const int nth = a.by_page(key);
        slot[i] = key - nth * a.page;
        pg[i] = p.list[nth];
      }
    }
  };
  s16x8 k[W::kLoads], v[W::kLoads];
  auto load = [&]() {
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) {
      i64 page = pg[i];
      if (page < 0 || page >= a.pages) {
        page = 0;
        bad |= 1u << i;
      }
      if (mine) {
        k[i] = __builtin_bit_cast(s16x8, C::load(kc + page * a.kc_page + slot[i] * a.kc_slot));
        v[i] = __builtin_bit_cast(s16x8, C::load(vc + page * a.vc_page + slot[i] * a.vc_slot));
      }
    }
    return bad;
  };
  auto store = [&](int buffer, unsigned bad) {
    char* to = lds + buffer * W::kBuffer;
    if (bad) {
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i)
        if (bad >> i & 1) v[i] = s16x8(0);
    }
    if (mine) {
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i) {
        const int r = first + W::kPass * i;
        *reinterpret_cast<s16x8*>(to + r * W::kKeyRow + chunk * 16) = k[i];
        *reinterpret_cast<s16x8*>(to + W::kKeys * W::kKeyRow + r * W::kValueRow + chunk * 16) = v[i];
      }
    }
  };
  // which keys of a tile have no page: lane = key
  auto lost = [&](int tile) {
    const int key = min(p.k0 + tile * W::kKeys + lane, p.k1 - 1);
    const i64 page = p.list[a.by_page(key)];
    return __ballot(page < 0 || page >= a.pages);
  };

  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x16(0.f);
  float m = -INFINITY, l = 0.f;
  bool huge = false;

  // elements past the head: zero keys, once (their queries are zero, and must not meet a NaN)
  if (!mine && chunk * 8 < DP) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < W::kLoads; ++i)
        *reinterpret_cast<s16x8*>(lds + b * W::kBuffer + (first + W::kPass * i) * W::kKeyRow +
                                  chunk * 16) = s16x8(0);
  }
  find(0);
  unsigned bad = load();
  find(1);
  store(0, bad);
  gone = lost(0);
  __syncthreads();

  for (int tile = 0; tile < tiles; ++tile) {
    const int key0 = p.k0 + tile * W::kKeys;
    const char* keys = lds + (tile & 1) * W::kBuffer;
    const char* values = keys + W::kKeys * W::kKeyRow;
    const bool more = tile + 1 < tiles;
    const unsigned long long without = gone;
    if (more) {
      bad = load();
      find(tile + 2);
      gone = lost(tile + 1);
    }
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x16(0.f);
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        const s16x8 ka = *reinterpret_cast<const s16x8*>(keys + (32 * t + col) * W::kKeyRow +
                                                         32 * e + 16 * half);
        s[t] = M::mul32(ka, q[e], s[t]);
      }
    }
    const bool partial = without != 0 || key0 + W::kKeys > all;
    if (partial) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 32 * t + 8 * (i / 4) + 4 * half + i % 4;
          if (key0 + at >= see || (without >> at & 1)) s[t][i] = -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    top *= a.scale;
    if (__any(top > m + kSlack)) {
      const Both both = halves(top);
      const float now = fmaxf(fmaxf(both.a, both.b), m);
      const float f = m == -INFINITY ? 0.f : exp2f(m - now);
      m = now;
      huge |= __any(fabsf(now) > kHuge && now != -INFINITY);
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;
    s16x8 prob[4];
    float sum = 0.f;
    if (!huge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], a.scale, -base));
          sum += e;
          prob[2 * t + i / 8][i % 8] = __builtin_bit_cast(short, static_cast<T>(e));
        }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(apart(s[t][i], a.scale, base));
          sum += e;
          prob[2 * t + i / 8][i % 8] = __builtin_bit_cast(short, static_cast<T>(e));
        }
    }
    l += sum;

    // V^T, an A operand: lanes name rows 4 half + i/4 of 16 keys and columns 16 (lane/16 % 2) ..
    const char* from = values + (4 * half + (lane & 15) / 4) * W::kValueRow +
                       32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto value = [&](int step, int d) {
      const char* at = from + 16 * step * W::kValueRow + 64 * d;
      const s16x4 lo = transposed(at), hi = transposed(at + 8 * W::kValueRow);
      return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    bool strange = false;
    if (OWN && partial) {
#pragma unroll 1
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x8 vt = value(step, d);
#pragma unroll
          for (int i = 0; i < 8; ++i) strange |= (vt[i] & M::kExponent) == M::kExponent;
        }
      strange = __any(strange);
    }
    if (!OWN || !strange) {
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = M::mul32(value(step, d), prob[step], o[d]);
    } else {
      // an infinity or NaN among the values of a tile that not all rows see: key by key, added
      // to the rows that see it alone (0 times either would be NaN in the others)
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
          const int i = (key / 8) * 4 + key % 4;
          const bool holds = key % 8 / 4 == half;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const s16x8 vt = value(step, d);
            s16x8 one = s16x8(0);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (holds && e == i) one[e] = vt[e];
            const f32x16 part = M::mul32(one, prob[step], f32x16(0.f));
            if (key0 + 16 * step + key < see) o[d] += part;
          }
        }
    }
    if (more) store((tile + 1) & 1, bad);
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

template <typename T, int DP, bool EVEN>
__global__ __launch_bounds__(256, Wide<DP>::kPerCu) void wide_prefix(Attention a) {
  __shared__ __align__(16) char lds[2 * Wide<DP>::kBuffer];
  const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
  const int tile = i % a.prefix_tiles, unit = i / a.prefix_tiles * 8 + x;
  if (unit >= a.kv_heads * a.prefix_splits) return;
  const int split = unit / a.kv_heads;
  Part p;
  p.list = a.prefix;
  p.k0 = split * a.prefix_chunk;
  p.k1 = min(p.k0 + a.prefix_chunk, a.prefix_length);
  p.row0 = tile * Wide<DP>::kRows;
  p.rows = a.tokens * a.group;
  p.token0 = 0;
  p.before = a.prefix_length;
  p.step = 0;
  p.slot = split;
  wide_part<T, DP, EVEN, false>(a, p, unit - split * a.kv_heads, lds);
}

template <typename T, int DP, bool EVEN>
__global__ __launch_bounds__(256, Wide<DP>::kPerCu) void wide_own(Attention a) {
  __shared__ __align__(16) char lds[2 * Wide<DP>::kBuffer];
  int i = blockIdx.x;
  const int head = i % a.kv_heads;
  i /= a.kv_heads;
  const int split = i % a.own_splits;
  i /= a.own_splits;
  const int first = i % a.own_tiles;
  const Sequence s = sequence(a, i / a.own_tiles);
  Part p;
  p.list = s.list;
  p.rows = s.count * a.group;
  p.token0 = s.first;
  p.before = s.before + 1;
  p.step = 1;
  p.slot = a.prefix_splits + split;
  p.k0 = split * a.own_chunk;
  for (int tile = first; tile * Wide<DP>::kRows < p.rows; tile += a.own_tiles) {
    p.row0 = tile * Wide<DP>::kRows;
    const int last = min(p.row0 + Wide<DP>::kRows, p.rows) - 1;
    p.k1 = seen(s, a.by_group(last));
    if (split + 1 < a.own_splits) p.k1 = min(p.k1, p.k0 + a.own_chunk);
    if (p.k0 >= p.k1) continue;
    wide_part<T, DP, EVEN, true>(a, p, head, lds);
    __syncthreads();
  }
}

template <int DP, typename T, bool EVEN>
hipError_t launch_wide_as(const Attention& a, bool prefix, hipStream_t stream) {
  i64 grid;
  const void* f;
  if (prefix) {
    grid = (static_cast<i64>(a.kv_heads) * a.prefix_splits + 7) / 8 * 8 * a.prefix_tiles;
    f = reinterpret_cast<const void*>(&wide_prefix<T, DP, EVEN>);
  } else {
    grid = static_cast<i64>(a.kv_heads) * a.own_splits * a.own_tiles * a.sequences;
    f = reinterpret_cast<const void*>(&wide_own<T, DP, EVEN>);
  }
  Attention copy = a;
  void* args[] = {&copy};
  return hipLaunchKernel(f, dim3(static_cast<unsigned>(grid)), dim3(256), args, 0, stream);
}

template <int DP>
hipError_t launch_wide(const Attention& a, int64_t dtype, bool prefix, hipStream_t stream) {
  const bool even = a.page % 16 == 0;
  if (dtype == TG_F16)
    return even ? launch_wide_as<DP, _Float16, true>(a, prefix, stream)
                : launch_wide_as<DP, _Float16, false>(a, prefix, stream);
  return even ? launch_wide_as<DP, __bf16, true>(a, prefix, stream)
              : launch_wide_as<DP, __bf16, false>(a, prefix, stream);
}

}  // namespace tg
