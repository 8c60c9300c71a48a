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
  static constexpr int kPitch = DP == 64 ? 128 : DP == 256 ? 512 : 256;   // bytes of an LDS row
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kLoads = kKeys * kChunks / 256;    // of each thread, keys and values
  static constexpr int kPass = 256 / kChunks;             // rows that one load of all covers
  static constexpr int kTile = kKeys * kPitch;
  static constexpr int kBuffer = 2 * kTile;               // keys, then values
  static constexpr int kPerCu = DP == 256 ? 1 : 2;

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

// 16 bytes of every active lane to LDS at `to` + 16 * lane, without a register between.
__device__ __forceinline__ void load_to_lds(const void* from, char* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) unsigned*)from,
      (__attribute__((address_space(3))) unsigned*)to, 16, 0, 0);
}

// EVEN: pages hold whole groups of 16 keys, so that a wave's rows of one load stand on one page
// and its number is uniform.
template <typename T, int DP, bool EVEN, bool OWN>
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

  // The pages of a tile's keys, lane = key: asked for two tiles ahead and before the tile's own
  // loads, since loads return in order.  Keys past the end stand for the last one (hidden).
  auto pages_of = [&](int tile) {
    return p.list[a.by_page(min(p.k0 + tile * W::kKeys + lane, p.k1 - 1))];
  };
  unsigned key_at[2], value_at[2];    // EVEN: bytes from a group's first row to this lane's place
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = first + W::kPass * i;
    key_at[i] = (r & 15) * static_cast<unsigned>(a.kc_slot) * 2 + (place ^ W::key_place(r)) * 16;
    value_at[i] =
        (r & 15) * static_cast<unsigned>(a.vc_slot) * 2 + (place ^ W::value_place(r)) * 16;
  }
  auto load = [&](int tile, i64 pages) {
    char* to = lds + (tile & 1) * W::kBuffer + wave * 1024;
    const int key0 = p.k0 + tile * W::kKeys;
    const bool tail = key0 + W::kKeys > p.k1;
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) {
      const int r = first + W::kPass * i;
      const int kd = (place ^ W::key_place(r)) * 8, vd = (place ^ W::value_place(r)) * 8;
      i64 page;
      const char *ka, *va;
      if (EVEN) {
        const int group = __builtin_amdgcn_readfirstlane(r & ~15);
        page = static_cast<i64>(
            static_cast<uint64_t>(
                static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(pages >> 32), group)))
                << 32 |
            static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(pages), group)));
        const int key = min(key0 + group, (p.k1 - 1) & ~15);
        const int slot = key - static_cast<int>(a.by_page(key)) * a.page;
        unsigned kat = key_at[i & 1], vat = value_at[i & 1];
        if (tail) {
          const unsigned in = min(r & 15, p.k1 - 1 - key);
          kat = in * static_cast<unsigned>(a.kc_slot) * 2 + kd * 2;
          vat = in * static_cast<unsigned>(a.vc_slot) * 2 + vd * 2;
        }
        ka = reinterpret_cast<const char*>(kc + page * a.kc_page + slot * a.kc_slot) + kat;
        va = reinterpret_cast<const char*>(vc + page * a.vc_page + slot * a.vc_slot) + vat;
      } else {
        page = __shfl(pages, r);
        const int key = min(key0 + r, p.k1 - 1);
        const int slot = key - static_cast<int>(a.by_page(key)) * a.page;
        ka = reinterpret_cast<const char*>(kc + page * a.kc_page + slot * a.kc_slot + kd);
        va = reinterpret_cast<const char*>(vc + page * a.vc_page + slot * a.vc_slot + vd);
      }
      if (page >= 0 && page < a.pages) {
        if (kd < a.dim) load_to_lds(ka, to + 4096 * i);
        if (vd < a.dim) load_to_lds(va, to + W::kTile + 4096 * i);
      } else {    // no page: hidden below, and zero, since 0 times a NaN would be NaN
        *reinterpret_cast<s16x8*>(to + 4096 * i + 16 * lane) = s16x8(0);
        *reinterpret_cast<s16x8*>(to + W::kTile + 4096 * i + 16 * lane) = s16x8(0);
      }
    }
  };

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
        *reinterpret_cast<s16x8*>(lds + b * W::kBuffer + 4096 * i + 16 * tid) = s16x8(0);
  i64 pages = pages_of(0), next = pages_of(1);
  load(0, pages);
  __syncthreads();

  for (int tile = 0; tile < tiles; ++tile) {
    const int key0 = p.k0 + tile * W::kKeys;
    const char* keys = lds + (tile & 1) * W::kBuffer;
    const char* values = keys + W::kTile;
    const bool more = tile + 1 < tiles;
    // keys that have no page
    const unsigned long long without = __ballot(pages < 0 || pages >= a.pages);
    pages = next;
    if (more) {
      next = pages_of(tile + 2);
      load(tile + 1, pages);
    }
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x16(0.f);
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        const s16x8 ka = *reinterpret_cast<const s16x8*>(
            keys + (32 * t + col) * W::kPitch + ((2 * e + half) ^ W::key_place(col)) * 16);
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
    const int vrow = 4 * half + (lane & 15) / 4;
    auto value = [&](int step, int d) {
      const int chunk = (4 * d + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ W::value_place(vrow);
      const char* at = values + (16 * step + vrow) * W::kPitch + chunk * 16 + 8 * (lane & 1);
      const s16x4 lo = transposed(at), hi = transposed(at + 8 * W::kPitch);
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
          for (int i = 0; i < 8; ++i)   // (nothing was stored past the head)
            strange |= 32 * d + col < a.dim && (vt[i] & M::kExponent) == M::kExponent;
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
#pragma unroll 1
      for (int key = 0; key < W::kKeys; ++key) {
        const int step = key / 16, i = key % 16 / 8 * 4 + key % 4;
        const bool holds = key % 8 / 4 == half;
        const s16x8 pr = step == 0 ? prob[0] : step == 1 ? prob[1] : step == 2 ? prob[2] : prob[3];
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x8 vt = value(step, d);
          s16x8 one = s16x8(0);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (holds && e == i) one[e] = vt[e];
          const f32x16 part = M::mul32(one, pr, f32x16(0.f));
          if (key0 + key < see) o[d] += part;
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
  const bool even = a.page % 16 == 0 && a.kc_slot >= 0 && a.kc_slot < (1 << 24) &&
                    a.vc_slot >= 0 && a.vc_slot < (1 << 24);
  if (dtype == TG_F16)
    return even ? launch_wide_as<DP, _Float16, true>(a, prefix, stream)
                : launch_wide_as<DP, _Float16, false>(a, prefix, stream);
  return even ? launch_wide_as<DP, __bf16, true>(a, prefix, stream)
              : launch_wide_as<DP, __bf16, false>(a, prefix, stream);
}

}  // namespace tg
