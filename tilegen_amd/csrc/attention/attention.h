// What the kernels of libtgattn share: element types, 16-byte accesses, division by a number
// known at launch, and the search for a token's sequence.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>

#include "tgrt.h"
#include "tilegen_attention.h"

namespace tg {

using i64 = long long;

// 16 bytes that lie on a boundary of the element type alone: one global_load_dwordx4 all the
// same (gfx950 loads global memory from any byte address).
template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(N)));
  struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    Vec v;
  };
  static __device__ __forceinline__ Vec load(const T* p) {
    return reinterpret_cast<const Loose*>(p)->v;
  }
  static __device__ __forceinline__ void store(T* p, Vec v) {
    reinterpret_cast<Loose*>(p)->v = v;
  }
};

// floor(n / d) for 0 <= n < 2^31 by one high multiplication.
struct Div {
  uint32_t mul, shift;
  Div() = default;
  explicit Div(uint32_t d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return (__umulhi(mul, n) + n) >> shift;
  }
};

// The sequence of token t: how many of ends[1 .. sequences] are at most t (equal ends are
// empty sequences); `sequences`, which is none, for a token before ends[0] as for one past the
// last.  A whole wave asks for one token; each round looks at 64 places.
__device__ __forceinline__ int sequence_of(const int64_t* __restrict__ ends, int sequences,
                                           i64 t) {
  const int lane = threadIdx.x & 63;
  const bool before = t < ends[0];
  int lo = 0, hi = sequences;  // the answer is in lo .. hi
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + (lane + 1) * step;  // ends[at] <= t: the answer is at least `at`
    const bool past = at <= hi && ends[at] <= t;
    const int n = __popcll(__ballot(past));
    lo += n * step;
    hi = min(hi, lo + step - 1);
  }
  return before ? sequences : lo;
}

// Host side: one message format for refusals and HIP errors.
inline int refuse(int code, const char* what, const char* why, long long value) {
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: %s (%lld)", what, why, value);
  return tg_fail(code, msg);
}

inline int hip_failed(hipError_t e, const char* what) {
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: %s (hipError %d)", what, hipGetErrorString(e),
                static_cast<int>(e));
  return tg_fail(static_cast<int>(e), msg);
}

}  // namespace tg
