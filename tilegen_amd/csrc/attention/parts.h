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

// Rows and keys of one workgroup's part.
struct Part {
  const int64_t* list;  // pages
  int k0, k1;           // keys, k0 < k1, all of them on the list
  int row0, rows;       // its first row and the end of all rows (row = token * group + head)
  int token0;
  int before, step;     // the row of token j sees min(k1, before + step j) keys
  int slot;
};

// 16 bytes of every active lane to LDS at `to` + 16 * lane, without a register between.
__device__ __forceinline__ void load_to_lds(const void* from, char* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) unsigned*)from,
      (__attribute__((address_space(3))) unsigned*)to, 16, 0, 0);
}

// The same, from a uniform address and 32-bit offsets or from any address, written out: the
// compiler knows nothing of it and inserts no wait, so that a wave can read one tile from LDS
// while another is on its way.  (It returns no register; the waits are the caller's, wait_loads.)
__device__ __forceinline__ unsigned lds_address(char* to) {
  return static_cast<unsigned>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)to));
}
__device__ __forceinline__ void fetch_to_lds(const char* from, unsigned offset, char* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                   lds_address(to)),
               "v"(offset), "s"(from)
               : "memory", "m0");
}
__device__ __forceinline__ void fetch_to_lds(const void* from, char* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                   lds_address(to)),
               "v"(from)
               : "memory", "m0");
}

// Waits until at most N of this wave's loads are on their way (they return in order), or until
// its LDS reads are done; neither lets the compiler move memory accesses past it.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The prefix's workgroups: those that read the same keys (the row tiles of a kv head and a key
// range) follow one another, and every XCD takes an eighth of all in that order (workgroup i
// goes to XCD i % 8), so that they share an L2 and all XCDs have as much to do.
__host__ __device__ inline i64 prefix_count(const Attention& a) {
  return static_cast<i64>(a.prefix_tiles) * a.kv_heads * a.prefix_splits;
}
inline i64 prefix_grid(const Attention& a) { return (prefix_count(a) + 7) / 8 * 8; }
__device__ __forceinline__ bool prefix_place(const Attention& a, int* tile, int* kv_head,
                                             int* split) {
  const int n = static_cast<int>(prefix_count(a));
  const int i = static_cast<int>(blockIdx.x & 7) * ((n + 7) / 8) + (blockIdx.x >> 3);
  if (static_cast<int>(blockIdx.x >> 3) >= (n + 7) / 8 || i >= n) return false;
  const int unit = i / a.prefix_tiles;
  *tile = i - unit * a.prefix_tiles;
  *split = unit / a.kv_heads;
  *kv_head = unit - *split * a.kv_heads;
  return true;
}

// The own pages' workgroups: a sequence's row tile and key range go to an XCD in turn, all kv
// heads of it to the same one.  (A head to each XCD would have every XCD read 256 bytes of each
// key's 2 KB, say, which stand in few channels of its L2.)
inline i64 own_grid(const Attention& a) {
  const i64 units = static_cast<i64>(a.own_splits) * a.own_tiles * a.sequences;
  return (units + 7) / 8 * 8 * a.kv_heads;
}
__device__ __forceinline__ bool own_place(const Attention& a, int* tile, int* split, int* kv_head,
                                          int* b) {
  const int i = blockIdx.x >> 3, group = i / a.kv_heads;
  int unit = group * 8 + (blockIdx.x & 7);
  *kv_head = i - group * a.kv_heads;
  *split = unit % a.own_splits;
  unit /= a.own_splits;
  *tile = unit % a.own_tiles;
  *b = unit / a.own_tiles;
  return *b < a.sequences;
}

// The four keys of V^T that the transposing LDS read gives a lane: 16 lanes name 4 rows of 16
// values (8 bytes each) and lane i of them receives column i of the four rows.
__device__ __forceinline__ s16x4 transposed(const char* at) {
  typedef __attribute__((address_space(3))) s16x4 Lds4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4*)at);
}

}  // namespace tg
