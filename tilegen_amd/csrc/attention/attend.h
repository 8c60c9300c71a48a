// The kernel that computes attention's parts: some workgroups take parts of the prefix, the
// others parts of the sequences' own pages, in one launch, so that neither waits for the
// other's last workgroup and the one's products run beside the other's loads.
#pragma once

#include "narrow.h"
#include "wide.h"

namespace tg {

// PREFIX, OWN: rows of a workgroup, 16 (narrow) or 128 (wide).
template <int DP, int PREFIX, int OWN>
struct Attend {
  static constexpr bool kWide = PREFIX > 16;
  static constexpr int kNarrowBytes = Narrow<DP>::kBytes;
  static constexpr int kWideBytes = 2 * Wide<DP>::kBuffer;
  static constexpr int kBytes = !kWide                        ? kNarrowBytes
                                : OWN > 16                    ? kWideBytes
                                : kNarrowBytes > kWideBytes ? kNarrowBytes
                                                            : kWideBytes;
  // of a CU: registers for two waves a SIMD (256 each), where a head leaves room for them
  static constexpr int kPerCu = DP == 256 ? 1 : 2;
};

template <typename T, int DP, int ROWS, bool OWN>
__device__ __forceinline__ void part(const Attention& a, const Part& p, int kv_head, char* lds) {
  if constexpr (ROWS == 16)
    narrow_part<T, DP, false>(a, p, kv_head, lds);
  else
    wide_part<T, DP, OWN>(a, p, kv_head, lds);
}

// Workgroup i goes to XCD i % 8, so they are dealt in eights, the prefix's first: its parts are
// alike and long.
template <typename T, int DP, int PREFIX, int OWN>
__global__ __launch_bounds__(64 * kWaves, (Attend<DP, PREFIX, OWN>::kPerCu)) void attend(
    Attention a) {
  __shared__ __align__(16) char lds[Attend<DP, PREFIX, OWN>::kBytes];
  const int xcd = blockIdx.x & 7, eight = blockIdx.x >> 3;
  Part p;
  if (eight < a.prefix_eights) {
    int tile, kv_head, split;
    if (!prefix_place(a, xcd, eight, &tile, &kv_head, &split)) return;
    p.list = a.prefix;
    p.k0 = split * a.prefix_chunk;
    p.k1 = min(p.k0 + a.prefix_chunk, a.prefix_length);
    p.row0 = tile * PREFIX;
    p.rows = a.tokens * a.group;
    p.token0 = 0;
    p.before = a.prefix_length;
    p.step = 0;
    p.slot = split;
    part<T, DP, PREFIX, false>(a, p, kv_head, lds);
    return;
  }
  int first, split, kv_head, b;
  if (!own_place(a, (eight - a.prefix_eights) * 8 + xcd, &first, &split, &kv_head, &b))
    return;
  const Sequence s = sequence(a, b);
  p.list = s.list;
  p.rows = s.count * a.group;
  p.token0 = s.first;
  p.before = s.before + 1;
  p.step = 1;
  p.slot = a.prefix_splits + split;
  p.k0 = split * a.own_chunk;
  for (int tile = first; tile * OWN < p.rows; tile += a.own_tiles) {
    p.row0 = tile * OWN;
    const int last = min(p.row0 + OWN, p.rows) - 1;
    p.k1 = seen(s, a.by_group(last));
    if (split + 1 < a.own_splits) p.k1 = min(p.k1, p.k0 + a.own_chunk);
    if (p.k0 >= p.k1) continue;
    part<T, DP, OWN, true>(a, p, kv_head, lds);
    __syncthreads();
  }
}

template <typename T, int DP, int PREFIX, int OWN>
hipError_t launch(const Attention& a, hipStream_t stream) {
  Attention copy = a;
  void* args[] = {&copy};
  return hipLaunchKernel(reinterpret_cast<const void*>(&attend<T, DP, PREFIX, OWN>),
                         dim3(static_cast<unsigned>(a.prefix_eights + a.own_eights) * 8),
                         dim3(64 * kWaves), args, 0, stream);
}

// A small call in one launch: a workgroup takes all keys of 16 of a sequence's rows (own_tiles
// such tiles, and in turns those past them) for one kv head, the prefix's among them, and writes
// their results.  The last kv_heads workgroups write those of tokens that belong to no sequence.
template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves, (DP == 256 ? 1 : 2)) void attend_whole(Attention a) {
  __shared__ __align__(16) char lds[Narrow<DP>::kBytes];
  const int unit = blockIdx.x / a.kv_heads, kv_head = blockIdx.x - unit * a.kv_heads;
  const int b = unit / a.own_tiles, tile = unit - b * a.own_tiles;
  auto nothing = [&](int from, int to) {    // rows that see no key
    for (int row = from + threadIdx.x / 64; row < to; row += kWaves) {
      const int t = a.by_group(row), h = kv_head * a.group + row - t * a.group;
      T* out = static_cast<T*>(a.out) + t * a.o_token + h * a.o_head;
      for (int d = threadIdx.x & 63; d < a.dim; d += 64) out[d] = T(0);
      if (a.lse && threadIdx.x % 64 == 0) a.lse[static_cast<i64>(t) * a.heads + h] = -INFINITY;
    }
  };
  if (b >= a.sequences) {
    i64 begin = a.ends ? a.ends[0] : 0, end = a.ends ? a.ends[a.sequences] : a.tokens;
    begin = begin < 0 ? 0 : begin > a.tokens ? a.tokens : begin;
    end = end < begin ? begin : end > a.tokens ? a.tokens : end;
    nothing(0, static_cast<int>(begin) * a.group);
    nothing(static_cast<int>(end) * a.group, a.tokens * a.group);
    return;
  }
  const Sequence s = sequence(a, b);
  Part p;
  p.list = a.prefix;
  p.own_list = s.list;
  p.own_from = a.prefix_length;
  p.k0 = 0;
  p.rows = s.count * a.group;
  p.token0 = s.first;
  p.before = a.prefix_length + s.before + 1;
  p.step = 1;
  for (p.row0 = tile * 16; p.row0 < p.rows; p.row0 += a.own_tiles * 16) {
    const int last = min(p.row0 + 16, p.rows) - 1;
    p.k1 = a.prefix_length + (a.pages ? seen(s, a.by_group(last)) : 0);
    if (p.k1 == 0) {
      nothing(s.first * a.group + p.row0, s.first * a.group + last + 1);
      continue;
    }
    narrow_part<T, DP, true>(a, p, kv_head, lds);
    __syncthreads();
  }
}

template <typename T, int DP>
hipError_t launch_whole(const Attention& a, hipStream_t stream) {
  Attention copy = a;
  void* args[] = {&copy};
  return hipLaunchKernel(reinterpret_cast<const void*>(&attend_whole<T, DP>),
                         dim3(static_cast<unsigned>((a.sequences * a.own_tiles + 1) * a.kv_heads)),
                         dim3(64 * kWaves), args, 0, stream);
}

template <typename T, int DP>
hipError_t launch_parts(const Attention& a, int prefix_rows, int own_rows, hipStream_t stream) {
  if (prefix_rows == 16) return launch<T, DP, 16, 16>(a, stream);
  return own_rows == 16 ? launch<T, DP, 128, 16>(a, stream) : launch<T, DP, 128, 128>(a, stream);
}

}  // namespace tg
