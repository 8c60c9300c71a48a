// What the kernels of attention's parts share: matrix instructions of both types, exchanges
// between the lanes of a row, and what a part is.
#pragma once

#include "prefix_attention.h"

namespace tg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Matrix;

template <>
struct Matrix<__bf16> {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mul16(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a),
                                                   __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mul32(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a),
                                                   __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static constexpr short kExponent = 0x7F80;
  static constexpr float kLift = 0.f;
};

template <>
struct Matrix<_Float16> {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mul16(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a),
                                                  __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mul32(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a),
                                                  __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static constexpr short kExponent = 0x7C00;
  static constexpr float kLift = 7.f;
};

// A value of the other half of the wave, and of the other half of each half, beside one's own:
// the pair holds both, in either order.
struct Both {
  float a, b;
};
__device__ __forceinline__ Both halves(float v) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const unsigned a = r[0], b = r[1];
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ Both quarters(float v) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const unsigned a = r[0], b = r[1];
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}

// The larger, and the sum, of a value over the four lanes that hold one row of a 16x16 tile.
__device__ __forceinline__ float row_max(float v) {
  const Both h = halves(v);
  const Both q = quarters(fmaxf(h.a, h.b));
  return fmaxf(q.a, q.b);
}
__device__ __forceinline__ float row_sum(float v) {
  const Both h = halves(v);
  const Both q = quarters(h.a + h.b);
  return q.a + q.b;
}

constexpr float kSlack = 8.f;   // log2 of how far scores may pass the running maximum
// Scores times scale less the maximum is one fused operation, exact in the product where the
// maximum has been rounded.  Past this the rounding, 2^-24 of it, is no longer small against
// one, and the product is rounded too.
constexpr float kHuge = 16777216.f;
__device__ __forceinline__ float apart(float s, float scale, float base) {
#pragma clang fp contract(off)
  const float x = s * scale;
  return x - base;
}

// What a row's probabilities are taken against: its largest score, 2^kLift down, so that the
// largest probability is 2^kLift, and 2^(kLift + kSlack) before the maximum follows, 2^15 in
// float16.  The factor is in sums and products alike.  It keeps probabilities down to 2^-32 of
// the largest apart from 0 where float16 by itself ends at 2^-25: on long prefixes what is below
// counts (131071 keys 18 nats under one have 0.2% of the weight).  Past kHuge differences are
// whole and the lift would be rounded.
template <typename T>
__device__ __forceinline__ float base_of(float top) {
  return fabsf(top) > kHuge ? top : top - Matrix<T>::kLift;
}
// Whether the maximum has to follow `top`.  Past 2^27 neighbouring scores are 16 apart, and a sum
// would round up to the next one and leave a probability of 2^16: bfloat16 holds it, float16 does
// not and compares the difference, which is exact for neighbours (in bfloat16 that costs heads of
// 256 up to 4%, 262 us for 253: 2 prompts of up to 2048 tokens, 16 heads).
template <typename T>
__device__ __forceinline__ bool passes(float top, float base) {
  if constexpr (Matrix<T>::kLift > 0.f) return top - base > kSlack + Matrix<T>::kLift;
  return top > base + kSlack;
}

constexpr int kWaves = 4;       // of a workgroup

// Rows and keys of one workgroup's part.
struct Part {
  const int64_t* list;  // pages
  int k0, k1;           // keys, k0 < k1, all of them on the list
  int row0, rows;       // its first row and the end of all rows (row = token * group + head)
  int token0;
  int before, step;     // the row of token j sees min(k1, before + step j) keys
  int slot;
  // of narrow parts that take the prefix and a sequence's own pages (`list`: the prefix's) in one:
  // keys from own_from on stand on own_list, and every row sees those before
  const int64_t* own_list;
  int own_from;
};

// 16 bytes of every active lane to LDS at `to` + 16 * lane, without a register between.
__device__ __forceinline__ void load_to_lds(const void* from, char* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) unsigned*)from,
      (__attribute__((address_space(3))) unsigned*)to, 16, 0, 0);
}

// The prefix's workgroups: those that read the same keys (the row tiles of a kv head and a key
// range) follow one another, and every XCD takes an eighth of all in that order, so that they
// share an L2 and all XCDs have as much to do.  `i` counts the workgroups of one XCD.
__device__ __forceinline__ bool prefix_place(const Attention& a, int xcd, int i, int* tile,
                                             int* kv_head, int* split) {
  const int n = a.prefix_tiles * a.kv_heads * a.prefix_splits, each = (n + 7) / 8;
  const int at = xcd * each + i;
  if (i >= each || at >= n) return false;
  const int unit = at / a.prefix_tiles;
  *tile = at - unit * a.prefix_tiles;
  *split = unit / a.kv_heads;
  *kv_head = unit - *split * a.kv_heads;
  return true;
}

// The own pages' workgroups: the kv heads of a sequence's row tile and key range side by side.
// (All heads of it on one XCD instead measured 5% slower.)
//
// With `sorted`, at most as many sequences as a workgroup has threads stand in the order of their
// lengths, the longest first: long parts that start last would leave most of the chip idle
// behind them.  Each thread ranks one sequence.
__device__ __forceinline__ bool own_place(const Attention& a, int i, int* tile, int* split,
                                          int* kv_head, int* b) {
  int unit = i / a.kv_heads;
  *kv_head = i - unit * a.kv_heads;
  *split = unit % a.own_splits;
  unit /= a.own_splits;
  *tile = unit % a.own_tiles;
  *b = unit / a.own_tiles;
  if (*b >= a.sequences) return false;
  if (a.sorted) {
    __shared__ __align__(16) int lengths[64 * kWaves];
    __shared__ int found;
    const int tid = threadIdx.x;
    const int64_t length = tid < a.sequences ? a.lengths[tid] : -1;
    const int mine = length < 0 ? -1 : length > INT32_MAX ? INT32_MAX : static_cast<int>(length);
    lengths[tid] = mine;
    __syncthreads();
    int before = 0;
#pragma unroll 4
    for (int i = 0; i < a.sequences; i += 4) {
      const int4 other = *reinterpret_cast<const int4*>(lengths + i);
      before += other.x > mine || (other.x == mine && i < tid);
      before += other.y > mine || (other.y == mine && i + 1 < tid);
      before += other.z > mine || (other.z == mine && i + 2 < tid);
      before += other.w > mine || (other.w == mine && i + 3 < tid);
    }
    if (tid < a.sequences && before == *b) found = tid;
    __syncthreads();
    *b = __builtin_amdgcn_readfirstlane(found);
  }
  return true;
}

// The four keys of V^T that the transposing LDS read gives a lane: 16 lanes name 4 rows of 16
// values (8 bytes each) and lane i of them receives column i of the four rows.
__device__ __forceinline__ s16x4 transposed(const char* at) {
  typedef __attribute__((address_space(3))) s16x4 Lds4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4*)at);
}

}  // namespace tg
